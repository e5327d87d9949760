"""A training run of a small token model between whose embedding and head lie shift layers:

    python -m deepshift_amd.train_tokens --steps 50 --tokens 4096 --vocabulary 8192 --width 512

The model predicts the next token of a synthetic stream (every token is a fixed function of the two before it, with noise) from
the embeddings of the last two: ``training.ScaledEmbedding``, a stack of ``LinearShift`` layers on their float path (or
``LinearShiftQ``), and ``training.LinearCrossEntropy``; the gradients, which straight-through estimators pass to shifts and
signs unscaled, are clipped by their global norm.  Prints the loss and the norm as it goes, then tokens per second.
"""
import argparse
import time

import torch
import torch.nn as nn

from . import modules, modules_q, training


class TokenModel(nn.Module):
    """Embeddings of two tokens side by side, ``depth`` shift layers with ReLU, a linear head with its loss."""

    def __init__(self, vocabulary, width, depth, shift_type="PS", weight_bits=5, padding_idx=None):
        super().__init__()
        layer = modules.LinearShift if shift_type == "PS" else modules_q.LinearShiftQ
        self.embedding = training.ScaledEmbedding(vocabulary, width // 2, scale=(width // 2) ** 0.5, padding_idx=padding_idx)
        self.layers = nn.ModuleList([layer(width, width, weight_bits=weight_bits) for _ in range(depth)])
        self.norms = nn.ModuleList([nn.LayerNorm(width) for _ in range(depth)])
        self.head = training.LinearCrossEntropy(width, vocabulary)

    def hidden(self, tokens):
        """``tokens`` [N, 2] -> [N, width]."""
        x = self.embedding(tokens).flatten(1)
        for norm, layer in zip(self.norms, self.layers):
            x = x + torch.relu(layer(norm(x)))
        return x

    def forward(self, tokens, target):
        return self.head(self.hidden(tokens), target)


def batch(tokens, vocabulary, device, generator, noise=0.1, ignored=0.05):
    """Pairs of tokens and what follows them; a few targets are not to be counted."""
    pair = torch.randint(0, vocabulary, (tokens, 2), generator=generator, device=device)
    pair = torch.minimum(pair, torch.randint(0, vocabulary, (tokens, 2), generator=generator, device=device))
    target = (pair[:, 0] // 3 + pair[:, 1] // 5) % vocabulary
    shuffled = torch.randint(0, vocabulary, (tokens,), generator=generator, device=device)
    draw = torch.rand(tokens, generator=generator, device=device)
    target = torch.where(draw < noise, shuffled, target)
    return pair, torch.where(draw > 1 - ignored, torch.full_like(target, -100), target)


def train_step(model, optimizer, pair, target, max_norm):
    """One step; returns the loss and the gradients' norm before clipping, both on the device."""
    optimizer.zero_grad(set_to_none=True)
    loss = model(pair, target)
    loss.backward()
    norm = training.clip_grad_norm_(model.parameters(), max_norm)
    optimizer.step()
    return loss.detach(), norm


def main(argv=None):
    parser = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    parser.add_argument("--steps", type=int, default=50)
    parser.add_argument("--tokens", type=int, default=4096, help="tokens a step")
    parser.add_argument("--vocabulary", type=int, default=8192)
    parser.add_argument("--width", type=int, default=512)
    parser.add_argument("--depth", type=int, default=2)
    parser.add_argument("--shift-type", choices=("PS", "Q"), default="PS")
    parser.add_argument("--weight-bits", type=int, default=5)
    parser.add_argument("--lr", type=float, default=2e-3)
    parser.add_argument("--max-norm", type=float, default=1.0)
    parser.add_argument("--seed", type=int, default=0)
    args = parser.parse_args(argv)
    if args.width % 2 or min(args.steps, args.tokens, args.vocabulary, args.width) < 1:
        parser.error("width has to be even, and all sizes positive")
    if not torch.cuda.is_available():
        parser.error("training needs a GPU")
    device = torch.device("cuda", torch.cuda.current_device())
    torch.manual_seed(args.seed)
    generator = torch.Generator(device=device).manual_seed(args.seed)
    with device:
        model = TokenModel(args.vocabulary, args.width, args.depth, args.shift_type, args.weight_bits)
    optimizer = torch.optim.Adam(model.parameters(), lr=args.lr)
    first = loss = None
    start = time.perf_counter()
    for step in range(args.steps):
        pair, target = batch(args.tokens, args.vocabulary, device, generator)
        loss, norm = train_step(model, optimizer, pair, target, args.max_norm)
        first = loss if first is None else first
        if step % 10 == 0 or step == args.steps - 1:
            print("step %4d  loss %.4f  norm %.3f" % (step, loss.item(), norm.item()), flush=True)
    torch.cuda.synchronize()
    took = time.perf_counter() - start
    print("%.0f tokens/s" % (args.steps * args.tokens / took))
    return first.item(), loss.item()


if __name__ == "__main__":
    main()
