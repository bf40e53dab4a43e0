"""Attention over the paged 8-bit K/V cache where its parts meet: segments of one tile, moves of
the maximum that no vote announces. Needs a B200."""
import pytest
import torch

from test_paged_gpu import _b200, call, check_attend, paged_problem  # noqa: F401 (fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hq,hkv,dim,q_len,window", [(8, 2, 64, 1, None), (16, 1, 128, 1, 60), (32, 1, 128, 1, 200),
                                                    (16, 2, 256, 1, 130), (8, 2, 128, 4, 150)])
def test_short_segments_repeat_bit_for_bit(hq, hkv, dim, q_len, window):
    """Requests of one or two tiles, many to a CTA (the row sums of a segment follow at once upon the
    move of its maxima), and window edges in each tile (moves without a vote): held to the oracle,
    and the same bits in every one of 60 runs."""
    lens = [q_len + (37 * i) % 290 for i in range(200)]
    p = paged_problem(lens, hq, hkv, dim, 32, "bf16", [q_len] * len(lens), seed=dim + hq, spread=4.0)
    want, want_lse = call(p, window_left=window, return_lse=True)
    for _ in range(60):
        o, lse = call(p, window_left=window, return_lse=True)
        assert torch.equal(o, want) and torch.equal(lse, want_lse)
    few = list(range(0, 200, 17))
    p = paged_problem([lens[i] for i in few], hq, hkv, dim, 32, "bf16", [q_len] * len(few), seed=dim, spread=4.0)
    check_attend(p, window=window)
