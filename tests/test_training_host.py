"""CPU: what deepshift_amd.training refuses or decides before anything is launched, and its entry points' status codes."""
import pytest
import torch

from deepshift_amd import _lib, training


def test_cpu_tensors_are_refused():
    ids = torch.zeros(3, dtype=torch.int64)
    x, w = torch.zeros(3, 4), torch.zeros(5, 4)
    with pytest.raises(ValueError, match="GPU"):
        training.embedding(ids, w)
    with pytest.raises(ValueError, match="GPU"):
        training.embedding_grad(ids, x, 5)
    with pytest.raises(ValueError, match="GPU"):
        training.linear_cross_entropy_grad(x, w, ids)
    with pytest.raises(ValueError, match="GPU"):
        training.clip_gradients_([x], 1.0)
    with pytest.raises(TypeError):
        training.gradient_norm([ids])
    with pytest.raises(ValueError, match="reduction"):
        training.LinearCrossEntropy(4, 5, reduction="batch")
    with pytest.raises(ValueError, match="padding_idx"):
        training.ScaledEmbedding(5, 4, padding_idx=5)


def test_native_entry_points_refuse():
    native = _lib.native()
    x = torch.zeros(3)
    for args in ((), (1, 2, 3), (x, x, 1.0, 0, 0)):
        with pytest.raises(TypeError):
            native.embed(*args)
    for args in ((), (x, None, 1.0, 1, 0, 0), ([x, 1], None, 1.0, 1, 0, 0), ([1], None, 1.0, 1, 0, 0), ([x], x, 1.0, 1, 0, 0)):
        with pytest.raises((TypeError, ValueError)):
            native.clip(*args)
    with pytest.raises(ValueError, match="no gradients"):
        native.clip([], None, 1.0, 1, 0, 0)
    with pytest.raises(ValueError, match="1 tensors in out for 2"):
        native.clip([x, x], [x], 1.0, 1, 0, 0)


def test_modules_hold_what_their_counterparts_hold():
    e = training.ScaledEmbedding(7, 3, scale=4.0, padding_idx=-1)
    assert e.weight.shape == (7, 3) and e.padding_idx == 6 and (e.weight[6] == 0).all()
    head = training.LinearCrossEntropy(3, 7)
    plain = torch.nn.Linear(3, 7)
    plain.load_state_dict(head.state_dict())
    x = torch.randn(2, 3)
    assert torch.equal(head.logits(x), plain(x))
    assert training.LinearCrossEntropy(3, 7, bias=False).bias is None


def test_workspaces_grow_with_what_they_hold():
    L = _lib.lib()
    assert L.ds_clip_workspace_bytes(-1) == 0 and L.ds_clip_workspace_bytes(1) > 0
    assert L.ds_clip_workspace_bytes(1000) > L.ds_clip_workspace_bytes(1)
    assert L.ds_embed_grad_workspace_bytes(-1, 4) == 0
    assert L.ds_embed_grad_workspace_bytes(1000, 512) >= 1000 * 16
    args = (4096, 64, 4096, 64, 100, 64, 1000)
    assert L.ds_vocab_workspace_bytes(*args, 9, 1) == 0
    assert L.ds_vocab_workspace_bytes(*args, _lib.DS_BF16, 2) >= 100 * 1000 * 2     # the probabilities of one piece
    assert L.ds_vocab_workspace_bytes(*args, _lib.DS_F32, 2) >= 100 * 1000 * 6
    # a piece is bounded: the logits of a large batch over a large vocabulary are never all there
    large = L.ds_vocab_workspace_bytes(4096, 64, 4096, 64, 1 << 20, 64, 1 << 18, _lib.DS_BF16, 2)
    assert large < (1 << 20) * (1 << 18) * 2 // 64


@pytest.mark.parametrize("fault", ["type", "target", "reduction", "rows", "vocabulary", "workspace", "size"])
def test_status_codes_of_the_loss(fault):
    L = _lib.lib()
    p = 4096
    T, D, V, ld, kind, tb, red, rows, ws, nbytes = 4, 8, 5, 8, 0, 8, 2, p, p, 1 << 30
    want = -1
    if fault == "type":
        kind = 3
    elif fault == "target":
        tb = 2
    elif fault == "reduction":
        red = 3
    elif fault == "rows":
        ld = 7
    elif fault == "vocabulary":
        V = 0
    elif fault == "workspace":
        nbytes, want = 1, -4
    else:
        V, want = 1 << 31, -5
    assert L.ds_vocab_loss(p, ld, p, ld, None, p, tb, -100, T, D, V, kind, red, rows, p, p, ws, nbytes, None) == want


@pytest.mark.parametrize("T, V, D", [(4, 1 << 31, 8), (1 << 31, 4, 8), (4, 1 << 20, 1 << 40), (4, 1 << 30, 1 << 30)])
def test_an_embeddings_gradient_has_to_fit(T, V, D):
    assert _lib.lib().ds_embed_grad(4096, 8, 4096, D, 4096, T, V, D, -1, 1.0, 0, 4096, 1 << 62, None) == -5


def test_status_codes_of_clipping():
    L = _lib.lib()
    t = (_lib.Tensor * 1)((4096, 4096, 10, 0, 0))
    assert L.ds_clip(t, -1, 1.0, 1, 4096, 4096, 1 << 20, None) == -1
    assert L.ds_clip(t, 1, -1.0, 1, 4096, 4096, 1 << 20, None) == -1
    assert L.ds_clip(t, 1, 1.0, 0, None, 4096, 1 << 20, None) == -1
    assert L.ds_clip(t, 1, 1.0, 1, 4096, 4096, 8, None) == -4
    t[0].src_type = 5
    assert L.ds_clip(t, 1, 1.0, 1, 4096, 4096, 1 << 20, None) == -1
    t[0] = (4098, 4096, 10, 0, 0)
    assert L.ds_clip(t, 1, 1.0, 1, 4096, 4096, 1 << 20, None) == -1
