"""Sizes at which the embedding gradient's indexes end."""
import pytest
import torch

from dlvk_b200.ops import nn as NN


@pytest.mark.gpu
def test_more_tokens_than_ints_have_places_for_are_refused():
    """The last block of the sums counts up to 256 chunks of 64 places past the end: from 2^31 -
    16384 tokens on those places would pass 2^31.  (Expanded tensors: a refused call reads nothing.)"""
    dy = torch.zeros(1, 1, device="cuda")
    for n in (2 ** 31 - 32768, 2 ** 31 - 2000, 2 ** 31 + 5):
        ids = torch.zeros(1, dtype=torch.int32, device="cuda").expand(n)
        with pytest.raises(RuntimeError, match="tokens"):
            NN.embedding_grad(ids, dy.expand(n, 1), 8)
    with pytest.raises(RuntimeError, match="words"):
        NN.embedding_grad(torch.zeros(1, dtype=torch.int32, device="cuda"), dy, 2 ** 31)
