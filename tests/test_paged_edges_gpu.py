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


def step_with_rows_behind(spare, decode, before=0, dim=128):
    """A step as kv_cache_plan leaves it: q has `spare` rows behind the last request (and `before` in front)."""
    q_lens = [1] * 48 if decode else [512, 300, 1]
    lens = [500 + 40 * i for i in range(48)] if decode else [2000, 300, 900]
    p = paged_problem(lens, 32, 8, dim, 32, "bf16", q_lens, seed=spare, spare_rows=before)
    used = sum(q_lens)
    p["q"] = torch.cat([p["q"], torch.randn(spare, 32, dim, dtype=torch.float32).bfloat16()])
    p["cu"] = [before + c for c in p["cu"]]
    return p, before, before + used


@pytest.mark.parametrize("decode", [True, False])
@pytest.mark.parametrize("before,spare", [(0, 1), (0, 700), (3, 0), (1000, 333), (0, 4096)])
def test_rows_outside_the_requests_are_zero(decode, before, spare):
    p, first, last = step_with_rows_behind(spare, decode, before)
    total = p["q"].shape[0]
    torch.full((4, total, 32, 128), 3.0, dtype=torch.bfloat16, device="cuda")  # what a new tensor may find in its place
    o, lse = call(p, return_lse=True)
    assert not o[:first].any() and not o[last:].any()
    assert not lse[:, :first].any() and not lse[:, last:].any()
    inner = dict(p, q=p["q"][first:last], cu=[c - first for c in p["cu"]])
    want, want_lse = call(inner, return_lse=True)
    assert torch.equal(o[first:last], want) and torch.equal(lse[:, first:last], want_lse)


@pytest.mark.parametrize("decode", [True, False])
def test_rows_behind_the_requests_cost_what_their_bytes_do(decode):
    """Padded steps are the ordinary ones (the host knows an upper bound of the new tokens only). The limit is
    20 us and their bytes at 2 TB/s; one warp that cleared them all took 4096 rows some milliseconds."""
    from apex_attn import custom_attention_paged_forward

    def microseconds(spare):
        p, _, _ = step_with_rows_behind(spare, decode)
        (kc, ks), (vc, vs) = p["gpu"]
        q, table, lens, cu = p["q"].cuda(), *(torch.tensor(p[n], dtype=torch.int32, device="cuda")
                                              for n in ("table", "lens", "cu"))
        best = float("inf")
        for _ in range(12):
            start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            torch.cuda._sleep(1000000)  # the host runs ahead
            start.record()
            custom_attention_paged_forward(q, kc, vc, ks, vs, table, lens, cu, p["max_q"])
            end.record()
            torch.cuda.synchronize()
            best = min(best, start.elapsed_time(end) * 1e3)
        return best

    alone = microseconds(0)
    for spare in (64, 512, 4096):
        limit = alone + 20 + spare * 32 * 128 * 2 / 2e6
        took = microseconds(spare)
        print(f"{spare} rows behind: {took:.1f} us, {alone:.1f} without")
        assert took <= limit, f"{spare} rows behind the requests: {took:.0f} us, {alone:.0f} without them"
