"""CPU: what deepshift_amd.train_tokens.SequenceModel refuses."""
import pytest
import torch

from deepshift_amd import train_tokens


def test_generation_needs_a_token_to_go_on_from():
    model = train_tokens.SequenceModel(20, 8, 1)
    with pytest.raises(ValueError, match="tokens must be"):
        model.generate(torch.zeros(2, 0, dtype=torch.long), 3)
    with pytest.raises(ValueError, match="GPU"):
        model.generate(torch.zeros(2, 3, dtype=torch.long), 1)
