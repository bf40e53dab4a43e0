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


def test_captured_behind_copies_fills_and_other_streams():
    """The kernels may start before the work in front of them ends where that is a kernel; behind a copy, a fill or
    a join of streams they have to wait for it as a whole."""
    from apex_attn import custom_attention_paged_forward
    p = paged_problem([700, 33, 2100], 16, 4, 128, 32, "bf16", [1, 1, 1], seed=3)
    (kc, ks), (vc, vs) = p["gpu"]
    table, lens = (torch.tensor(p[n], dtype=torch.int32, device="cuda") for n in ("table", "lens"))
    new_q, new_lens = p["q"].cuda(), lens.clone()
    q, held = torch.zeros_like(new_q), torch.zeros_like(lens)
    step = lambda x, n: custom_attention_paged_forward(x, kc, vc, ks, vs, table, n)
    want, none = step(new_q, lens), torch.zeros_like(new_q)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        q.copy_(new_q)
        held.copy_(new_lens)
        first = step(q, held)
        held.zero_()
        second = step(q, held)
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            held.copy_(new_lens)
        main.wait_stream(side)
        third = step(q, held)
    for _ in range(20):
        for x in (q, first, second, third):
            x.fill_(5.0)
        held.fill_(1)
        graph.replay()
        assert torch.equal(first, want) and torch.equal(second, none) and torch.equal(third, want)


@pytest.mark.parametrize("blocks,max_new", [(6, 300), (20, 150)])
def test_a_step_whose_requests_do_not_all_fit(blocks, max_new):
    """The stack, or the slot array, is short: the offsets of the new tokens may pass the end of q. Placed requests
    get what they get alone, the others leave every block as it is, and nothing behind q is touched."""
    from apex_attn import custom_attention_paged_forward, kv_cache_append, kv_cache_plan
    new, block, dim = [40, 64, 100, 16, 90], 16, 64
    g = torch.Generator(device="cuda").manual_seed(blocks)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    cache = lambda: [torch.zeros(blocks, 2, block, dim, device="cuda").to(torch.float8_e4m3fn) for _ in range(2)] + [
        torch.zeros(blocks, 2, device="cuda") for _ in range(2)]
    q = torch.randn(max_new, 4, dim, generator=g, device="cuda").bfloat16()
    k = torch.randn(max_new, 2, dim, generator=g, device="cuda").bfloat16()
    c = cache()
    table = torch.full((5, 8), -1, dtype=torch.int32, device="cuda")
    free = torch.arange(blocks, dtype=torch.int32, device="cuda")
    plan = kv_cache_plan(table, ints([0] * 5), ints(new), free, ints([blocks]), block, max_new)
    kv_cache_append(k, k, *c, plan.slots)
    guarded = torch.full((max_new + 64, 4, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    o = custom_attention_paged_forward(q, *c, table, plan.seq_lens, plan.cu_seqlens, max(new), out=guarded[:max_new])
    torch.cuda.synchronize()
    placed, cu = plan.placed.tolist(), plan.cu_seqlens.tolist()
    assert 0 < sum(placed) < 5 and cu == [0, 40, 104, 204, 220, 310]
    assert (guarded[max_new:] == 7).all()
    for b in range(5):
        if not placed[b]:
            assert plan.seq_lens[b] == 0 and (table[b] == -1).all()
            continue
        alone, one, n = cache(), torch.full((1, 8), -1, dtype=torch.int32, device="cuda"), new[b]
        mine = kv_cache_plan(one, ints([0]), ints([n]), free, ints([blocks]), block, n)
        rows = slice(cu[b], cu[b] + n)
        kv_cache_append(k[rows], k[rows], *alone, mine.slots)
        want = custom_attention_paged_forward(q[rows], *alone, one, mine.seq_lens, mine.cu_seqlens, n)
        assert (o[rows].float() - want.float()).abs().max() <= 2.0 ** -6  # |o| < 4: two roundings to bf16
