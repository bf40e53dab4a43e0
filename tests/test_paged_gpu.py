"""The paged 8-bit K/V cache operators against the float64 oracle. Needs a B200.

Bookkeeping and cache writes are exact. Attention is held, element by element, to the bound
that oracle.paged_oracle.attend derives from the kernels' documented roundings, plus half a
step of the output type.
"""
import os
import random

import pytest
import torch

from oracle import paged_oracle as ref

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.fixture(scope="module", autouse=True)
def _b200():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    if torch.cuda.get_device_capability() != (10, 0):
        pytest.skip("needs sm_100")
    import apex_attn
    assert os.path.exists(apex_attn.library_path())
    yield
    assert apex_attn.device_status() == 0


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def cumulated(values):
    out = [0]
    for v in values:
        out.append(out[-1] + v)
    return out


# ------------------------------------------------------------------- bookkeeping --
def plan_inputs(batch, block, width, seed, spare, new_max, pool=None):
    rng = random.Random(seed)
    lens = [rng.choice([0, 1, block - 1, block, rng.randrange(width * block // 2 + 1)]) for _ in range(batch)]
    new = [rng.choice([0, 1, 1, rng.randint(1, new_max)]) for _ in range(batch)]
    ids = list(range(sum(-(-n // block) for n in lens) + spare))
    rng.shuffle(ids)
    table = [[-7] * width for _ in range(batch)]
    for b, n in enumerate(lens):
        for j in range(-(-n // block)):
            table[b][j] = ids.pop()
    count = len(ids)
    free = ids + [-9] * sum(-(-n // block) for n in lens)
    return table, lens, new, free or [-9], count


PLAN_CASES = [
    # batch, block, width, spare blocks, new_max, slack of max_new_tokens
    (1, 16, 4, 10, 1, 0),
    (3, 16, 40, 60, 200, 5),
    (64, 32, 20, 64, 1, 0),
    (257, 64, 10, 500, 90, 100),
    (300, 128, 6, 120, 300, 0),     # the stack runs short
    (40, 16, 8, 400, 100, 3),       # table rows too short for some
    (1000, 16, 30, 3000, 40, 1),
    (2500, 32, 12, 9000, 30, 77),
    (8192, 128, 3, 9000, 4, 9),
]


@pytest.mark.parametrize("batch,block,width,spare,new_max,slack", PLAN_CASES)
def test_plan_matches_oracle(batch, block, width, spare, new_max, slack):
    from apex_attn import kv_cache_plan
    table, lens, new, free, count = plan_inputs(batch, block, width, batch + block, spare, new_max)
    max_new = max(1, sum(new) + slack)
    t, f = ints(table), ints(free)
    got = kv_cache_plan(t, ints(lens), ints(new), f, ints([count]), block, max_new)
    want_table = [list(r) for r in table]
    slots, cu, out_lens, out_count, placed = ref.plan(want_table, lens, new, free, count, block, max_new)
    assert got.cu_seqlens.tolist() == cu
    assert got.placed.tolist() == placed
    assert got.seq_lens.tolist() == out_lens
    assert got.free_count.tolist() == [out_count]
    assert t.tolist() == want_table
    assert got.slots.tolist() == slots
    assert f.tolist() == free


def test_plan_without_room_for_slots_places_no_part_of_a_request():
    from apex_attn import kv_cache_plan
    table = ints([[-1] * 4 for _ in range(3)])
    got = kv_cache_plan(table, ints([0, 0, 0]), ints([10, 20, 3]), ints(list(range(9))), ints([9]), 16, 25)
    assert got.placed.tolist() == [1, 0, 0]
    assert got.seq_lens.tolist() == [10, 0, 0]
    assert got.free_count.tolist() == [8]
    assert got.slots.tolist() == [8 * 16 + i for i in range(10)] + [-1] * 15


def test_plan_clamps_negative_lengths_and_counts():
    from apex_attn import kv_cache_plan
    table = ints([[5, -1], [-1, -1]])
    got = kv_cache_plan(table, ints([3, -4]), ints([-2, 1]), ints([8, 9]), ints([77]), 16, 4)
    assert got.cu_seqlens.tolist() == [0, 0, 1]
    assert got.seq_lens.tolist() == [3, 1]
    assert got.slots.tolist() == [9 * 16, -1, -1, -1]
    assert got.free_count.tolist() == [1]


@pytest.mark.parametrize("batch,block,width,spare,new_max,slack", PLAN_CASES)
def test_release_matches_oracle(batch, block, width, spare, new_max, slack):
    from apex_attn import kv_cache_release
    table, lens, _, free, count = plan_inputs(batch, block, width, 3 * batch + block, spare, new_max)
    rng = random.Random(batch)
    done = [rng.choice([0, 0, 1, -3]) for _ in range(batch)]
    f = ints(free)
    got_lens, got_count = kv_cache_release(ints(table), ints(lens), ints(done), f, ints([count]), block)
    want = list(free)
    out_lens, out_count = ref.release(table, lens, done, want, count, block)
    assert got_lens.tolist() == out_lens
    assert got_count.tolist() == [out_count]
    assert f.tolist() == want


def test_table_rows_of_a_wider_table():
    """A row stride above the width: neighbours in the same storage stay as they are."""
    from apex_attn import kv_cache_plan
    wide = ints([[-5] * 9 for _ in range(4)])
    kv_cache_plan(wide[:, 2:5], ints([0] * 4), ints([17] * 4), ints(list(range(20))), ints([20]), 16, 80)
    want = [[-5, -5, 19 - 2 * b, 18 - 2 * b] + [-5] * 5 for b in range(4)]
    assert wide.tolist() == want


# ------------------------------------------------------------------------ append --
def new_cache(blocks, heads, block, dim, token_major, seed, fill_nan=False):
    g = torch.Generator().manual_seed(seed)
    shape = (blocks, block, heads, dim) if token_major else (blocks, heads, block, dim)
    codes = torch.randn(shape, generator=g).mul(90).clamp(-448, 448).to(E4M3)
    if fill_nan:
        codes = torch.full(shape, float("nan")).to(E4M3)
    codes = codes.cuda()
    scale = torch.exp2(torch.randint(-9, -4, (blocks, heads), generator=g).float()).cuda()
    return codes.transpose(1, 2) if token_major else codes, scale


def as_values(codes):
    return codes.float().double().cpu()


def check_append(k, v, k_cache, v_cache, k_scale, v_scale, slots, block):
    from apex_attn import kv_cache_append
    want = [(as_values(c), s.double().cpu()) for c, s in ((k_cache, k_scale), (v_cache, v_scale))]
    host = slots.tolist()[:k.shape[0]]
    for x, (codes, scale) in zip((k, v), want):
        ref.append(x.cpu(), codes, scale, host, block)
    kv_cache_append(k, v, k_cache, v_cache, k_scale, v_scale, slots)
    torch.cuda.synchronize()
    for c, s, (codes, scale) in ((k_cache, k_scale, want[0]), (v_cache, v_scale, want[1])):
        assert torch.equal(s.double().cpu(), scale)
        got = as_values(c)
        assert torch.equal(torch.isnan(got), torch.isnan(codes))
        assert torch.equal(got.nan_to_num(), codes.nan_to_num())


APPEND_CASES = [
    # (start, length) of each request's new tokens, block, heads, dim, dtype, token_major
    ([(0, 1)], 16, 1, 64, "bf16", False),
    ([(5, 1), (16, 1), (31, 1), (0, 1)], 16, 2, 128, "fp16", False),
    ([(3, 40), (0, 128), (127, 2)], 64, 2, 256, "bf16", True),
    ([(9, 200), (0, 7), (15, 1)], 16, 8, 128, "bf16", True),
    ([(100, 300)], 128, 1, 64, "fp16", True),
    ([(i, 1) for i in range(130)], 32, 4, 128, "bf16", False),
    ([(7 * i, 150 + i) for i in range(30)], 32, 4, 64, "fp16", False),
]


@pytest.mark.parametrize("runs,block,heads,dim,dtype,token_major", APPEND_CASES)
@pytest.mark.parametrize("amp", [0.01, 1.0, 300.0])
def test_append_matches_oracle(runs, block, heads, dim, dtype, token_major, amp):
    g = torch.Generator().manual_seed(len(runs) + dim)
    counts = [-(-(s + n) // block) for s, n in runs]
    ids = torch.randperm(sum(counts) + 2, generator=g).tolist()
    table, at = [], 0
    for c in counts:
        table.append(ids[at:at + c])
        at += c
    slots = [table[b][t // block] * block + t % block for b, (s, n) in enumerate(runs) for t in range(s, s + n)]
    total = len(slots)
    k, v = ((torch.randn(total, heads, dim, generator=g) * amp * torch.exp2(
        torch.randint(-3, 4, (total, 1, 1), generator=g).float())).to(DTYPES[dtype]).cuda() for _ in range(2))
    kc, ks = new_cache(len(ids), heads, block, dim, token_major, 1)
    vc, vs = new_cache(len(ids), heads, block, dim, token_major, 2)
    check_append(k, v, kc, vc, ks, vs, torch.tensor(slots, device="cuda"), block)


def test_append_skips_slots_outside_the_cache():
    k = torch.randn(6, 2, 64, device="cuda").bfloat16()
    kc, ks = new_cache(4, 2, 16, 64, False, 3)
    vc, vs = new_cache(4, 2, 16, 64, False, 4)
    slots = torch.tensor([-1, 5, 6, 64, 10 ** 15, -(10 ** 15), 3, 4], device="cuda")
    check_append(k, -k, kc, vc, ks, vs, slots, 16)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_append_extreme_values(dtype):
    """Zeros, the type's subnormals and largest values, values on either side of a change of
    scale, NaN and infinities; each beside an old scale that is larger and one that is smaller."""
    t = DTYPES[dtype]
    info = torch.finfo(t)
    rows = [[0.0], [info.smallest_normal / 64, info.smallest_normal / 8], [info.max, -info.max], [7.0], [7.03125],
            [448.0, -3.5], [float("nan"), 2.0], [float("inf"), -float("inf"), 0.5], [float("nan")], [-1e-3],
            [2.0 ** -9 * 1.5, 448.0], [2.0 ** -10, 448.0]]
    x = torch.zeros(len(rows), 1, 64, dtype=torch.float64)
    for i, r in enumerate(rows):
        for j, value in enumerate(r):
            x[i, 0, j * 5::len(r) * 5] = value
    x = x.to(t).cuda()
    for start in (0, 3):
        for exponent in (-60, -3, 3):
            kc, _ = new_cache(len(rows), 1, 16, 64, False, 5)
            vc, _ = new_cache(len(rows), 1, 16, 64, True, 6)
            ks = torch.full((len(rows), 1), 2.0 ** exponent, device="cuda")
            slots = torch.arange(len(rows), device="cuda") * 16 + start
            check_append(x, -x, kc, vc, ks, ks.clone(), slots, 16)


def test_append_to_blocks_scaled_elsewhere():
    """An old scale that is no power of two: kept while it is large enough."""
    x = (torch.randn(8, 3, 128, device="cuda") * torch.tensor([0.1, 1, 2, 3, 4, 5, 6, 7], device="cuda")[:, None, None])
    x = x.bfloat16()
    kc, ks = new_cache(8, 3, 32, 128, False, 7)
    vc, vs = new_cache(8, 3, 32, 128, False, 8)
    ks.copy_(torch.rand(8, 3, device="cuda") * 0.02 + 0.003)
    vs.copy_(torch.rand(8, 3, device="cuda") * 0.02 + 0.003)
    from apex_attn import kv_cache_append
    before = kc.float(), ks.clone()
    slots = torch.arange(8, device="cuda") * 32 + 9
    kv_cache_append(x, x, kc, vc, ks, vs, slots)
    top = x.float().abs().amax(-1)
    m, e = torch.frexp(top)
    want = torch.ldexp(torch.ones_like(top), e - torch.where(m <= 0.875, 9, 8))
    after = torch.maximum(before[1], want)
    assert torch.equal(ks, after)
    assert torch.equal(kc[:, :, 9].float(), (x.float() / after[..., None]).clamp(-448, 448).to(E4M3).float())
    kept = (before[0][:, :, :9] * (before[1] / after)[..., None, None]).to(E4M3).float()
    assert torch.equal(kc[:, :, :9].float(), kept)
    assert torch.equal(kc[:, :, 10:].float(), before[0][:, :, 10:])


def test_append_strided_inputs():
    """K and V as views of one projection's output, and as views that need a copy."""
    g = torch.Generator().manual_seed(9)
    qkv = torch.randn(50, 12, 64, generator=g).bfloat16().cuda()
    slots = torch.arange(50, device="cuda") + 7
    for k, v in ((qkv[:, 8:10], qkv[:, 10:12]), (qkv.flip(0)[:, 3:5], qkv.transpose(1, 2).contiguous().transpose(1, 2)[:, :2])):
        kc, ks = new_cache(5, 2, 16, 64, False, 10)
        vc, vs = new_cache(5, 2, 16, 64, True, 11)
        check_append(k, v, kc, vc, ks, vs, slots, 16)


# --------------------------------------------------------------------- attention --
def paged_problem(lens, heads_q, heads_kv, dim, block, dtype, q_lens, token_major=False, seed=0, spread=1.0,
                  general_scales=False, spare_rows=0):
    """Blocks in a random order; everything that no request owns (spare blocks, rows behind the
    last token, unused table entries' blocks) is NaN."""
    g = torch.Generator().manual_seed(seed)
    counts = [-(-n // block) for n in lens]
    ids = torch.randperm(sum(counts) + 3, generator=g).tolist()
    width = max(max(counts), 1) + 1
    table, at = [], 0
    nan_block = ids[-1]
    for c in counts:
        table.append(ids[at:at + c] + [nan_block] * (width - c))
        at += c
    caches = []
    for _ in range(2):
        codes = (torch.randn(len(ids), heads_kv, block, dim, generator=g) * 90).clamp(-448, 448)
        codes[ids[at:]] = float("nan")
        for b, n in enumerate(lens):
            if n % block:
                codes[table[b][counts[b] - 1], :, n % block:] = float("nan")
        scale = torch.exp2(torch.randint(-8, -5, (len(ids), heads_kv), generator=g).float())
        if general_scales:
            scale = scale * (torch.rand(len(ids), heads_kv, generator=g) + 0.5)
        scale[ids[at:]] = float("nan")
        caches.append((codes.to(E4M3), scale))
    total = sum(q_lens) + spare_rows
    q = (torch.randn(total, heads_q, dim, generator=g) * spread).to(DTYPES[dtype])
    on_gpu = []
    for codes, scale in caches:
        c = codes.cuda()
        on_gpu.append((c.transpose(1, 2).contiguous().transpose(1, 2) if token_major else c, scale.cuda()))
    return {"q": q, "caches": caches, "gpu": on_gpu, "table": table, "lens": lens, "cu": cumulated(q_lens),
            "block": block, "max_q": max(q_lens)}


def call(p, decode=False, table_on_gpu=None, **kw):
    from apex_attn import custom_attention_paged_forward
    (kc, ks), (vc, vs) = p["gpu"]
    return custom_attention_paged_forward(p["q"].cuda(), kc, vc, ks, vs, ints(table_on_gpu or p["table"]),
                                          ints(p["lens"]),
                                          None if decode else ints(p["cu"]), p["max_q"], **kw)


def check_attend(p, decode=False, causal=True, window=None, sm_scale=None, table_on_gpu=None):
    o, lse = call(p, decode, table_on_gpu, causal=causal, window_left=window, sm_scale=sm_scale, return_lse=True)
    torch.cuda.synchronize()
    (kc, ks), (vc, vs) = p["caches"]
    ro, rl, ob, lb = ref.attend(p["q"], kc.double().nan_to_num(), vc.double().nan_to_num(), ks.double().nan_to_num(),
                                vs.double().nan_to_num(), p["table"], p["lens"], p["cu"], p["block"], causal, window,
                                sm_scale)
    o, lse = o.double().cpu(), lse.double().cpu()
    n = p["cu"][-1]
    assert torch.isfinite(o).all()
    eps = torch.finfo(p["q"].dtype).eps / 2
    err = (o - ro).abs() - (ob + eps * (ro.abs() + ob))
    worst = ((o - ro).abs() / (ob + eps * ro.abs() + 1e-30)).max().item()
    tiny = torch.finfo(p["q"].dtype).smallest_normal * eps * 2  # half a step of the output's subnormals
    assert (err <= tiny).all(), f"o is off by {worst:.2f} of its bound"
    seen = torch.isfinite(rl[:, :n])
    assert torch.equal(torch.isfinite(lse[:, :n]), seen)
    assert (lse[:, :n][~seen] == -torch.inf).all()
    lerr = ((lse - rl).abs() / (lb + 1e-30))[:, :n][seen]
    assert not seen.any() or lerr.max() <= 1, f"lse is off by {lerr.max().item():.2f} of its bound"
    assert not o[n:].any() and not lse[:, n:].any()
    return o


DECODE = [
    # lens, heads_q, heads_kv, dim, block, dtype, token_major
    ([1], 1, 1, 64, 16, "bf16", False),
    ([2, 1, 16, 17], 4, 1, 128, 16, "fp16", False),
    ([129, 0, 128, 127], 8, 2, 128, 32, "bf16", True),
    ([1000], 16, 4, 64, 16, "bf16", False),
    ([700, 3, 511], 10, 2, 256, 64, "fp16", True),
    ([333, 64, 65], 6, 6, 64, 64, "fp16", False),
    ([257] * 5, 32, 1, 128, 128, "bf16", True),
    ([90, 4000], 40, 2, 64, 32, "bf16", False),
    ([1500, 20], 48, 1, 256, 16, "bf16", False),
    ([600, 6], 130, 1, 128, 16, "fp16", False),
]


@pytest.mark.parametrize("lens,hq,hkv,dim,block,dtype,token_major", DECODE)
def test_single_token(lens, hq, hkv, dim, block, dtype, token_major):
    check_attend(paged_problem(lens, hq, hkv, dim, block, dtype, [1] * len(lens), token_major, seed=dim + hq),
                 decode=True)


CHUNKS = [
    # lens, q_lens, heads_q, heads_kv, dim, block, dtype, causal, window
    ([130, 5, 40], [3, 5, 1], 4, 2, 128, 16, "bf16", True, None),
    ([130, 5, 40], [3, 5, 1], 4, 2, 128, 16, "bf16", False, None),
    ([300, 17], [40, 17], 8, 1, 64, 32, "fp16", True, None),
    ([300, 200], [40, 140], 5, 1, 64, 32, "bf16", True, 20),
    ([520, 9, 256], [129, 9, 64], 4, 4, 256, 64, "bf16", True, None),
    ([520, 129, 256], [70, 129, 64], 8, 4, 128, 128, "fp16", True, 0),
    ([260, 0, 31], [4, 3, 40], 8, 2, 128, 16, "bf16", True, None),   # no cache; more tokens than the cache
    ([260, 0, 31], [4, 3, 40], 8, 2, 128, 16, "bf16", False, None),
    ([700, 400], [6, 2], 12, 2, 256, 16, "fp16", True, 130),
    ([385, 900], [0, 33], 16, 2, 64, 16, "bf16", True, 300),         # a request without query tokens
    ([257], [257], 3, 3, 128, 32, "fp16", True, None),
]


@pytest.mark.parametrize("lens,q_lens,hq,hkv,dim,block,dtype,causal,window", CHUNKS)
def test_several_tokens(lens, q_lens, hq, hkv, dim, block, dtype, causal, window):
    check_attend(paged_problem(lens, hq, hkv, dim, block, dtype, q_lens, seed=sum(q_lens) + dim), causal=causal,
                 window=window)


@pytest.mark.parametrize("window", [0, 1, 15, 127, 128, 1000])
def test_single_token_window(window):
    check_attend(paged_problem([900, 130, 12], 8, 2, 128, 16, "bf16", [1, 1, 1], seed=window), decode=True,
                 window=window)


@pytest.mark.parametrize("spread", [1e-3, 8.0, 60.0])
def test_flat_and_peaked_rows(spread):
    check_attend(paged_problem([1200, 77], 8, 2, 64, 32, "bf16", [1, 1], seed=1, spread=spread), decode=True)
    check_attend(paged_problem([500, 77], 8, 2, 128, 32, "fp16", [40, 3], seed=2, spread=min(spread, 20.0)))


def test_scales_of_any_value_and_scale_argument():
    check_attend(paged_problem([300, 90], 8, 2, 128, 16, "bf16", [1, 1], seed=3, general_scales=True), decode=True,
                 sm_scale=0.3)


def test_scores_that_rise_along_the_cache():
    """Each block's scores exceed all before it: the running maximum moves on every tile."""
    p = paged_problem([2000], 4, 1, 64, 16, "bf16", [1], seed=4)
    (kc, ks), (vc, vs) = p["caches"]
    q = torch.zeros_like(p["q"])
    q[..., 0] = 4.0
    p["q"] = q
    for i, blk in enumerate(p["table"][0][:125]):
        values = kc[blk].float()
        values[..., 0] = 100.0 + 2.0 * i
        kc[blk] = values.to(E4M3)
        ks[blk] = 0.25
    p["gpu"] = [(c.cuda(), s.cuda()) for c, s in p["caches"]]
    check_attend(p, decode=True)


def test_rows_outside_the_requests():
    p = paged_problem([100, 50], 4, 2, 64, 16, "bf16", [2, 3], seed=5, spare_rows=9)
    check_attend(p)
    out = torch.full(p["q"].shape, 7.0, dtype=p["q"].dtype, device="cuda")
    got = call(p, out=out)
    assert got is out
    assert (out[5:] == 7).all()
    assert torch.equal(out[:5], call(p)[:5])


def test_blocks_that_no_row_sees_are_not_read():
    """Under a window the blocks before it may have been handed to others: here they are NaN."""
    p = paged_problem([600, 300], 8, 2, 128, 16, "bf16", [1, 1], seed=6)
    want = call(p, decode=True, window_left=100)
    nan = p["table"][0][-1]
    for b, n in enumerate(p["lens"]):
        for j in range((n - 1 - 100) // 16):
            p["table"][b][j] = nan
    assert torch.equal(call(p, decode=True, window_left=100), want)


@pytest.mark.parametrize("bad", [-1, 10 ** 9, 7])
def test_table_entries_outside_the_cache_read_as_zeros(bad):
    """Held to the oracle on a cache whose second block is zero. (Not bit for bit to the kernel on
    that cache: the V scale of a block enters the maximum that its row's weights are rounded
    against, and a block that is not there has none.)"""
    p = paged_problem([64], 4, 2, 64, 16, "bf16", [1], seed=7)
    for c, _ in p["caches"]:
        c[p["table"][0][1]] = 0
    check_attend(p, decode=True, table_on_gpu=[[p["table"][0][0], bad] + p["table"][0][2:]])


def test_same_result_with_and_without_offsets_and_on_another_stream():
    p = paged_problem([300, 40, 900], 16, 4, 128, 32, "bf16", [1, 1, 1], seed=8)
    want = call(p, decode=True)
    assert torch.equal(call(p), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [call(p, decode=True) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_views_of_q():
    p = paged_problem([90, 33], 4, 2, 64, 16, "bf16", [3, 2], seed=9)
    want = call(p)
    wide = torch.zeros(5, 9, 64, dtype=torch.bfloat16)
    wide[:, 2:6] = p["q"]
    p["q"] = wide.cuda()[:, 2:6]
    assert torch.equal(call(p), want)


# -------------------------------------------------------------- a run of them all --
@pytest.mark.parametrize("block,dim,dtype", [(16, 64, "bf16"), (32, 128, "fp16"), (64, 256, "bf16")])
def test_serving_steps(block, dim, dtype):
    """Prompts, single tokens, drafts, finished requests whose blocks go to others: each step is
    release, plan, append, attend, against the oracle holding the same state."""
    from apex_attn import custom_attention_paged_forward, kv_cache_append, kv_cache_plan, kv_cache_release
    batch, hq, hkv, width, blocks = 4, 4, 2, 6, 18
    g = torch.Generator().manual_seed(block)
    kc, ks = new_cache(blocks, hkv, block, dim, block == 32, 1, fill_nan=True)
    vc, vs = new_cache(blocks, hkv, block, dim, False, 2, fill_nan=True)
    want = [[as_values(c).nan_to_num(), s.double().cpu()] for c, s in ((kc, ks), (vc, vs))]
    table = [[0] * width for _ in range(batch)]
    free = list(range(blocks))
    t, f = ints(table), ints(free)
    lens, count = ints([0] * batch), ints([blocks])
    host_lens, host_count = [0] * batch, blocks
    steps = [([0, 0, 0, 0], [block + 3, 1, 2 * block, 0]), ([0, 0, 0, 0], [1, 1, 1, 5]),
             ([0, 0, 0, 0], [3, 0, 4, 2]), ([0, 1, 1, 0], [1, block, 0, 1]), ([1, 0, 0, 0], [2 * block + 1, 1, 1, 1]),
             ([0, 0, 0, 0], [1, 6, block, 1])]
    for done, new in steps:
        lens, count = kv_cache_release(t, lens, ints(done), f, count, block)
        host_lens, host_count = ref.release(table, host_lens, done, free, host_count, block)
        max_new = sum(new) + 3
        plan = kv_cache_plan(t, lens, ints(new), f, count, block, max_new)
        slots, cu, host_lens, host_count, placed = ref.plan(table, host_lens, new, free, host_count, block, max_new)
        assert all(placed) and plan.placed.tolist() == placed
        lens, count = plan.seq_lens, plan.free_count
        k, v = ((torch.randn(max_new, hkv, dim, generator=g) * 3).to(DTYPES[dtype]) for _ in range(2))
        q = torch.randn(max_new, hq, dim, generator=g).to(DTYPES[dtype])
        kv_cache_append(k.cuda(), v.cuda(), kc, vc, ks, vs, plan.slots)
        for x, (codes, scale) in zip((k, v), want):
            ref.append(x, codes, scale, slots, block)
        o = custom_attention_paged_forward(q.cuda(), kc, vc, ks, vs, t, lens, plan.cu_seqlens, max(new))
        ro, _, ob, _ = ref.attend(q, want[0][0], want[1][0], want[0][1], want[1][1], table, host_lens, cu, block)
        eps = torch.finfo(q.dtype).eps / 2
        assert ((o.double().cpu() - ro).abs() <= ob + eps * (ro.abs() + ob)).all()
        assert t.tolist() == table and lens.tolist() == host_lens and count.tolist() == [host_count]


def test_a_captured_step_replays_with_new_lengths():
    """plan, append and attend in one graph, replayed while the requests grow; a second graph
    of the same calls replays in between."""
    from apex_attn import custom_attention_paged_forward, kv_cache_append, kv_cache_plan
    batch, hq, hkv, dim, block, width, blocks = 3, 8, 2, 128, 16, 20, 40
    g = torch.Generator(device="cuda").manual_seed(3)
    kc, ks = new_cache(blocks, hkv, block, dim, False, 1)
    vc, vs = new_cache(blocks, hkv, block, dim, False, 2)
    state = {"table": torch.zeros(batch, width, dtype=torch.int32, device="cuda"),
             "lens": ints([0] * batch), "new": ints([1] * batch), "count": ints([blocks]),
             "free": torch.arange(blocks, dtype=torch.int32, device="cuda")}
    q = torch.randn(batch, hq, dim, generator=g, device="cuda").bfloat16()
    k = torch.randn(batch, hkv, dim, generator=g, device="cuda").bfloat16()

    def step(cache):
        plan = kv_cache_plan(state["table"], state["lens"], state["new"], state["free"], state["count"], block, batch)
        kv_cache_append(k, k, *cache, plan.slots)
        o = custom_attention_paged_forward(q, *cache, state["table"], plan.seq_lens, return_lse=True)
        return plan, o

    caches = [(kc, vc, ks, vs), tuple(x.clone() for x in (kc, vc, ks, vs))]
    step(caches[0])
    state["table"].zero_()
    graphs, outs = [], []
    torch.cuda.synchronize()
    for c in caches:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(c))
        graphs.append(graph)
    for i in range(40):
        k.normal_(generator=g)
        q.normal_(generator=g)
        for graph in graphs:
            graph.replay()
        plan, (o, lse) = outs[0]
        other, (o2, lse2) = outs[1]
        if i % 13 == 0:
            torch.cuda.synchronize()
            want, wl = custom_attention_paged_forward(q, *caches[0], state["table"], plan.seq_lens, return_lse=True)
            assert plan.seq_lens.tolist() == [i + 1] * batch
            assert torch.equal(o, want) and torch.equal(lse, wl)
            assert torch.equal(o2, want) and torch.equal(lse2, wl)
        state["lens"].copy_(plan.seq_lens)
        state["count"].copy_(plan.free_count)
