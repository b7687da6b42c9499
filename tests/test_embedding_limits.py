"""Sizes at which the embedding gradient's indexes end, and words at the borders of
its sort's blocks (limits as in test_embedding_sorted.py)."""
import pytest
import torch

from dlvk_b200.ops import nn as NN
from test_embedding_sorted import check_grad


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


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
@pytest.mark.parametrize("words", [1, 2, 7, 15, 16, 17, 31, 63, 127, 128, 129, 1000, 1023, 1024, 1025, 4097, 131071,
                                   131072, 131073, 151936, 300001])
def test_words_at_the_borders_of_blocks(words, kind):
    """Every power of 2 and its neighbours, the last words, ids just outside and far outside on
    either side, in several thousand tokens of which half are the commonest eight words."""
    g = torch.Generator().manual_seed(words)
    edge = [2 ** k + d for k in range(31) for d in (-1, 0, 1)] + [words + d for d in range(-3, 300, 7)]
    edge = torch.tensor(edge + [-v - 1 for v in edge] + [2 ** 31 - 1, -2 ** 31])
    edge = edge[edge.abs() < 2 ** 31]
    ids = torch.cat([edge.repeat(5), torch.randint(0, words, (2000,), generator=g),
                     torch.randint(0, min(words, 8), (3000,), generator=g)])
    ids = ids[torch.randperm(ids.numel(), generator=g)]
    if kind == torch.int64:  # what no int holds, whose lower half is a word
        ids[::17] = ids[::17].clamp(0, words - 1) + 2 ** 32
    dy = torch.randn(ids.numel(), 8, generator=g).cuda()
    ids = ids.to(kind).cuda()
    first = check_grad(ids, dy, words, padding=words // 2)
    assert torch.equal(first, NN.embedding_grad(ids, dy, words, padding_idx=words // 2))
