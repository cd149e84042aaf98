"""CPU checks of what the embedding, the log probabilities and the clipping refuse, and of what
the model leaves to modules of the user's own."""
import pytest
import torch

from prime_moment_attention import _lib, embedding_lookup, token_logprobs

BIG = (1 << 32) + 5  # 5 in the 32 bits of a C int


def test_sizes_beyond_the_entry_points_are_refused():
    """By views that take no memory: none of them may be cut to 32 bits on the way."""
    one, ids = torch.zeros(1, 1), torch.zeros(3, dtype=torch.int64)
    for C in (BIG, (1 << 20) + 1):
        with pytest.raises(ValueError, match="columns"):
            embedding_lookup(ids, one.expand(2, C))
        with pytest.raises(ValueError, match="columns"):
            _lib.embedding(ids, one.expand(2, C), 1.0, one.expand(3, C))
        with pytest.raises(ValueError, match="columns"):
            _lib.embedding_backward(torch.zeros(0, dtype=torch.uint8), one.expand(3, C), 1.0, one.expand(2, C))
    for n, vocab in ((BIG, 1), (1 << 31, 1), (1, BIG), (1, (1 << 24) + 1)):
        x, t = one.expand(n, vocab), ids[:1].expand(n)
        with pytest.raises(ValueError, match="rows"):
            token_logprobs(x, t)
        with pytest.raises(ValueError, match="rows"):
            _lib.token_logprobs(x, t, -100, one, None, None, 0, None, None)
        with pytest.raises(ValueError, match="rows"):
            _lib.token_logprobs_backward(x, t, -100, one, None, one, None, x)
    with pytest.raises(RuntimeError, match="HIP device"):  # the largest sizes go on to the next check
        token_logprobs(one.expand(1, 1 << 24), ids[:1])
    with pytest.raises(RuntimeError, match="HIP device"):
        embedding_lookup(ids, one.expand(2, 1 << 20))
