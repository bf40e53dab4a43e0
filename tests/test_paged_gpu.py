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


@pytest.mark.parametrize("hq,hkv,dim,q_len,window", [(4, 2, 128, 5, None), (8, 2, 64, 7, 3), (16, 2, 128, 30, None),
                                                    (16, 2, 64, 200, 40), (16, 2, 256, 30, None), (4, 2, 256, 4, None),
                                                    (40, 2, 128, 150, None)])
@pytest.mark.parametrize("which", ["k", "v"])
def test_nan_reaches_only_the_rows_that_see_it(hq, hkv, dim, q_len, window, which):
    """A cached token that holds NaN: rows before it (and, under a window, behind) keep their values, the
    others get NaN. Both layouts of the products, tokens at tile edges among them."""
    lens = [q_len + 253, q_len + 1]
    p = paged_problem(lens, hq, hkv, dim, 16, "bf16", [q_len, q_len], seed=dim + q_len)
    want_o, want_lse, ob, lb = ref.attend(p["q"], *(c.double().nan_to_num() for c, _ in p["caches"]),
                                          *(s.double().nan_to_num() for _, s in p["caches"]), p["table"], lens, p["cu"],
                                          16, True, window)
    bad = [lens[0] - q_len // 2 - 1, lens[1] - 1]  # token positions
    column = 5
    for b, pos in enumerate(bad):
        codes = p["gpu"][0 if which == "k" else 1][0]
        codes[p["table"][b][pos // 16], :, pos % 16, column] = float("nan")
    o, lse = call(p, window_left=window, return_lse=True)
    o, lse = o.double().cpu(), lse.double().cpu()
    for b, pos in enumerate(bad):
        for i in range(q_len):
            r, place = p["cu"][b] + i, lens[b] - q_len + i
            sees = pos <= place and (window is None or pos >= place - window)
            if sees:
                assert torch.isnan(o[r, :, column]).all()
                assert which == "v" or torch.isnan(lse[:, r]).all()
            else:
                eps = torch.finfo(torch.bfloat16).eps / 2
                assert ((o[r] - want_o[r]).abs() <= ob[r] + eps * (want_o[r].abs() + ob[r])).all()
                assert ((lse[:, r] - want_lse[:, r]).abs() <= lb[:, r]).all()


@pytest.mark.parametrize("batch", [129, 300, 1000])
def test_large_batches(batch):
    rng = random.Random(batch)
    lens = [rng.choice([0, 1, rng.randint(1, 300)]) for _ in range(batch)]
    check_attend(paged_problem(lens, 4, 1, 64, 16, "bf16", [1] * batch, seed=batch), decode=True)


def test_ragged_queries_in_a_large_batch():
    rng = random.Random(7)
    lens = [rng.randint(1, 200) for _ in range(150)]
    q_lens = [rng.choice([0, 1, 1, 2, 40]) for _ in lens]
    check_attend(paged_problem(lens, 8, 2, 64, 32, "fp16", q_lens, seed=7, spare_rows=3))


def test_heads_of_their_own_and_one_head_for_all():
    check_attend(paged_problem([200, 64], 32, 32, 64, 16, "bf16", [1, 1], seed=1), decode=True)
    check_attend(paged_problem([300, 129], 16, 16, 128, 32, "fp16", [9, 3], seed=2))
    check_attend(paged_problem([513], 200, 1, 64, 16, "bf16", [3], seed=3))


def test_scales_of_zero_and_of_far_apart_blocks():
    p = paged_problem([300, 70], 8, 2, 128, 16, "bf16", [1, 1], seed=4)
    for c, s in p["caches"]:
        s.copy_(s * torch.exp2(torch.randint(-12, 13, s.shape, generator=torch.Generator().manual_seed(1)).float()))
    k_scale, v_scale = p["caches"][0][1], p["caches"][1][1]
    k_scale.clamp_(max=0.05)
    k_scale[p["table"][0][2]] = 0.0
    v_scale[p["table"][0][3]] = 0.0
    v_scale[p["table"][1][0]] = 0.0
    p["gpu"] = [(c.cuda(), s.cuda()) for c, s in p["caches"]]
    check_attend(p, decode=True)


def test_a_context_of_zeros():
    """All V scales zero: o is zero (scales below 2^-100 count as 2^-100), the logsumexp is right."""
    p = paged_problem([400], 8, 2, 64, 16, "bf16", [1], seed=5)
    p["gpu"][1][1].zero_()
    p["caches"][1][1].zero_()
    o, lse = call(p, decode=True, return_lse=True)
    assert o.float().abs().max() < 1e-25
    _, want, _, bound = ref.attend(p["q"], *(c.double().nan_to_num() for c, _ in p["caches"]),
                                   *(s.double().nan_to_num() for _, s in p["caches"]), p["table"], p["lens"], p["cu"], 16)
    assert ((lse.double().cpu() - want).abs() <= bound).all()


def test_infinite_and_nan_queries():
    p = paged_problem([100, 200], 4, 2, 64, 16, "fp16", [1, 1], seed=6)
    want = call(p, decode=True)
    p["q"][0, 1, 3] = float("inf")
    p["q"][1, 2, 0] = float("nan")
    got = call(p, decode=True)
    hurt = torch.zeros(2, 4, dtype=torch.bool, device="cuda")
    hurt[0, 1] = hurt[1, 2] = True
    assert torch.isnan(got[hurt]).all()
    assert torch.isfinite(got[~hurt]).all()
    assert torch.allclose(got[~hurt].float(), want[~hurt].float(), atol=2e-2)


def test_two_calls_at_once():
    """Two streams, two workspaces: each result is the one that the call gives alone."""
    problems = [paged_problem([3000, 500], 16, 2, 128, 16, "bf16", [1, 1], seed=8),
                paged_problem([900, 800, 40], 16, 2, 128, 32, "bf16", [60, 70, 40], seed=9)]
    want = [call(p) for p in problems]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in problems]
    got = [[], []]
    for _ in range(20):
        for i, (p, s) in enumerate(zip(problems, streams)):
            with torch.cuda.stream(s):
                got[i].append(call(p))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_offsets_that_overlap_or_fall_stay_in_bounds():
    """cu_seqlens_q and lengths that no program should give: rows may be wrong, guards stay."""
    p = paged_problem([100, 60, 30], 4, 2, 64, 16, "bf16", [2, 3, 2], seed=10)
    out = torch.full((20, 4, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    for cu in ([0, 7, 7, 7], [5, 2, 9, -4], [0, 2 ** 30, 3, 7], [7, 0, 7, 0]):
        for lens in ([100, 60, 30], [10 ** 9, -5, 112]):
            p["cu"], p["lens"] = cu, lens
            call(p, out=out[:7])
    torch.cuda.synchronize()
    assert (out[7:] == 7).all()


def test_caches_beyond_four_gigabytes():
    """Offsets past 32 bits in append and attend: blocks at the far end of two 5 GB caches."""
    from apex_attn import custom_attention_paged_forward, kv_cache_append
    blocks, heads, block, dim = 20480, 8, 128, 256
    kc, vc = (torch.empty(blocks, heads, block, dim, dtype=E4M3, device="cuda") for _ in range(2))
    ks, vs = (torch.ones(blocks, heads, device="cuda") for _ in range(2))
    g = torch.Generator().manual_seed(11)
    k, v = (torch.randn(200, heads, dim, generator=g).bfloat16() for _ in range(2))
    q = torch.randn(1, heads, dim, generator=g).bfloat16()
    ids = [blocks - 1, blocks - 2]
    slots = [ids[t // block] * block + t % block for t in range(200)]
    kv_cache_append(k.cuda(), v.cuda(), kc, vc, ks, vs, torch.tensor(slots, device="cuda"))
    o = custom_attention_paged_forward(q.cuda(), kc, vc, ks, vs, ints([ids]), ints([200]))
    small = [[torch.zeros(2, heads, block, dim, dtype=torch.float64), torch.ones(2, heads, dtype=torch.float64)]
             for _ in range(2)]
    for x, (codes, scale) in zip((k, v), small):
        ref.append(x, codes, scale, [t for t in range(200)], block)
    assert torch.equal(as_values(kc[ids])[:, :, :72], small[0][0][:, :, :72])
    ro, _, ob, _ = ref.attend(q, small[0][0], small[1][0], small[0][1], small[1][1], [[0, 1]], [200], [0, 1], block)
    eps = torch.finfo(torch.bfloat16).eps / 2
    assert ((o.double().cpu() - ro).abs() <= ob + eps * (ro.abs() + ob)).all()
    del kc, vc
    torch.cuda.empty_cache()


# ---------------------------------------------------------------------- refusals --
def test_python_refusals():
    import apex_attn
    p = paged_problem([40, 20], 4, 2, 64, 16, "bf16", [1, 1], seed=12)
    (kc, ks), (vc, vs) = p["gpu"]
    q, table, lens = p["q"].cuda(), ints(p["table"]), ints(p["lens"])
    good = dict(q=q, k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs, block_table=table, seq_lens=lens)
    run = apex_attn.custom_attention_paged_forward
    run(**good)
    for change, error in [
        (dict(q=q[0]), ValueError), (dict(q=q.float()), TypeError), (dict(q=q.cpu()), ValueError),
        (dict(q=q[:, :3]), ValueError), (dict(q=q[:, :, :32]), ValueError),
        (dict(k_cache=kc[:, :1]), ValueError), (dict(k_cache=kc.float(), v_cache=vc.float()), TypeError),
        (dict(k_cache=kc[..., :32], v_cache=vc[..., :32]), KeyError),
        (dict(k_cache=kc[:, :, :8], v_cache=vc[:, :, :8]), ValueError),
        (dict(k_cache=kc.transpose(2, 3).contiguous().transpose(2, 3)), ValueError),
        (dict(k_scale=ks.double()), ValueError), (dict(v_scale=vs[:1]), ValueError), (dict(k_scale=ks.cpu()), ValueError),
        (dict(block_table=table.long()), ValueError), (dict(block_table=table[0]), ValueError),
        (dict(block_table=table.cpu()), ValueError), (dict(block_table=table[:, :0]), ValueError),
        (dict(seq_lens=lens.long()), ValueError), (dict(seq_lens=lens[:1]), ValueError),
        (dict(cu_seqlens_q=ints([0, 1, 2])), ValueError), (dict(cu_seqlens_q=ints([0, 1]), max_seqlen_q=1), ValueError),
        (dict(max_seqlen_q=3), ValueError), (dict(q=q[:1]), ValueError), (dict(window_left=-1), ValueError),
        (dict(window_left=4, causal=False), ValueError), (dict(out=q[:, :2]), ValueError), (dict(out=q.float()), ValueError),
        (dict(sm_scale=0.0), RuntimeError), (dict(sm_scale=float("nan")), RuntimeError)]:
        with pytest.raises(error):
            run(**{**good, **change})
    assert run(**{**good, "q": q[:0], "cu_seqlens_q": ints([0, 0, 0]), "max_seqlen_q": 1}).shape == (0, 4, 64)

    k = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device="cuda")
    slots = torch.arange(3, device="cuda")
    good = dict(k=k, v=k, k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs, slots=slots)
    for change, error in [
        (dict(k=k[:2]), ValueError), (dict(v=k.half()), TypeError), (dict(k=k.float(), v=k.float()), TypeError),
        (dict(k=k[:, :1], v=k[:, :1]), ValueError), (dict(slots=slots.int()), ValueError), (dict(slots=slots[:2]), ValueError),
        (dict(slots=slots.cpu()), ValueError), (dict(v_cache=vc.cpu()), ValueError)]:
        with pytest.raises(error):
            apex_attn.kv_cache_append(**{**good, **change})
    apex_attn.kv_cache_append(**{**good, "k": k[:0], "v": k[:0]})

    free, count = ints(range(9)), ints([9])
    for change in [dict(block_size=20), dict(max_new_tokens=0), dict(new_lens=ints([1])), dict(free_count=ints([1, 2])),
                   dict(free_blocks=free.long()), dict(block_table=table.cpu()), dict(seq_lens=lens.cpu())]:
        with pytest.raises(ValueError):
            apex_attn.kv_cache_plan(**{**dict(block_table=table, seq_lens=lens, new_lens=lens, free_blocks=free,
                                              free_count=count, block_size=16, max_new_tokens=5), **change})
    with pytest.raises(ValueError):
        apex_attn.kv_cache_release(table, lens, lens[:1], free, count, 16)


def test_release_keeps_to_the_stack():
    """A stack without room for all returned blocks keeps what fits."""
    from apex_attn import kv_cache_release
    free = ints([9, -1, -1])
    lens, count = kv_cache_release(ints([[1, 2, 3], [4, 5, 6]]), ints([33, 16]), ints([1, 1]), free, ints([1]), 16)
    assert lens.tolist() == [0, 0] and count.tolist() == [3] and free.tolist() == [9, 1, 2]


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


def test_native_and_python_ways_agree():
    """Every call of a step through the native module and through Python: the same results."""
    import apex_attn.paged as paged
    if not (paged._calls or paged._load_calls()):
        pytest.skip("_calls is not built")
    native = paged._calls
    used = []
    results = []
    for way in (native, False):
        paged._calls = way
        try:
            table, free = ints([[0] * 8 for _ in range(3)]), ints(list(range(20)))
            kc, ks = new_cache(20, 2, 16, 64, True, 1)
            vc, vs = new_cache(20, 2, 16, 64, False, 2)
            g = torch.Generator(device="cuda").manual_seed(5)
            q = torch.randn(40, 8, 64, generator=g, device="cuda").half()
            lens, count = paged.kv_cache_release(table, ints([0, 0, 0]), ints([0, 1, 0]), free, ints([20]), 16)
            plan = paged.kv_cache_plan(table, lens, ints([20, 3, 17]), free, count, 16, 40)
            assert isinstance(plan, paged.KVCachePlan)
            paged.kv_cache_append(q[:, :2], q[:, 2:4], kc, vc, ks, vs, plan.slots)
            out = torch.zeros_like(q)
            got = [paged.custom_attention_paged_forward(q, kc, vc, ks, vs, table, plan.seq_lens, plan.cu_seqlens, 20,
                                                        return_lse=True, window_left=7, sm_scale=0.2),
                   paged.custom_attention_paged_forward(q, kc, vc, ks, vs, table, plan.seq_lens, plan.cu_seqlens, 20,
                                                        causal=False, out=out),
                   paged.custom_attention_paged_forward(q[:3], kc, vc, ks, vs, table, plan.seq_lens)]
            assert got[1] is out
            results.append([*plan, table, lens, kc.float(), vc.float(), ks, vs, *got[0], *got[1:]])
            used.append(paged._calls)
        finally:
            paged._calls = native
    for a, b in zip(*results):
        assert a.shape == b.shape and a.dtype == b.dtype and a.stride() == b.stride()
        assert torch.equal(a, b)
    assert native.attend(q.float(), kc, vc, ks, vs, table, plan.seq_lens, None, None, True, None, False, None, None) is None


# ------------------------------------------------------------ calls at the edges --
@pytest.mark.parametrize("hq,hkv,dim,q_len,window", [(4, 2, 128, 5, None), (8, 2, 64, 7, 3), (16, 2, 64, 200, 40),
                                                    (40, 2, 128, 150, None), (4, 2, 256, 4, None)])
@pytest.mark.parametrize("which", [0, 1])
def test_a_scale_of_nan_reaches_only_the_rows_that_see_its_block(hq, hkv, dim, q_len, window, which):
    lens = [q_len + 253, q_len + 1]
    p = paged_problem(lens, hq, hkv, dim, 16, "bf16", [q_len, q_len], seed=dim + q_len)
    want_o, want_lse, ob, lb = ref.attend(p["q"], *(c.double().nan_to_num() for c, _ in p["caches"]),
                                          *(s.double().nan_to_num() for _, s in p["caches"]), p["table"], lens, p["cu"],
                                          16, True, window)
    blocks = [(lens[0] - q_len // 2 - 1) // 16, (lens[1] - 1) // 16]
    for b, j in enumerate(blocks):
        p["gpu"][which][1][p["table"][b][j]] = float("nan")
    o, lse = call(p, window_left=window, return_lse=True)
    o, lse = o.double().cpu(), lse.double().cpu()
    some = [0, 0]
    for b, j in enumerate(blocks):
        for i in range(q_len):
            r, place = p["cu"][b] + i, lens[b] - q_len + i
            sees = 16 * j <= place and (window is None or 16 * j + 15 >= place - window)
            some[sees] += 1
            if sees:
                assert torch.isnan(o[r]).all() and torch.isnan(lse[:, r]).all()
            else:
                eps = torch.finfo(torch.bfloat16).eps / 2
                assert ((o[r] - want_o[r]).abs() <= ob[r] + eps * (want_o[r].abs() + ob[r])).all()
                assert ((lse[:, r] - want_lse[:, r]).abs() <= lb[:, r]).all()
    assert some[1]


@pytest.mark.parametrize("hq,hkv,dim,q_len", [(16, 2, 64, 1), (16, 1, 128, 1), (32, 1, 128, 1), (16, 2, 256, 1),
                                              (16, 2, 64, 5), (16, 2, 128, 20)])
def test_what_nobody_sees_changes_no_bit(hq, hkv, dim, q_len):
    """Old codes behind a request's last token, small, of the largest magnitude and NaN. (They must not
    even move a row's running maximum, which its weights are rounded against.)"""
    lens = [150, 135, 260, 131, 300, 145]
    p = paged_problem(lens, hq, hkv, dim, 64, "bf16", [q_len] * len(lens), seed=dim, spread=3.0)
    results = []
    for value in (0.0, 448.0, -448.0, float("nan")):
        for (codes, _), _ in zip(p["gpu"], p["caches"]):
            for b, n in enumerate(lens):
                codes[p["table"][b][n // 64], :, n % 64:] = value
        results.append(call(p, return_lse=True))
    for o, lse in results[1:]:
        assert torch.equal(o, results[0][0]) and torch.equal(lse, results[0][1])


def test_limits_that_reach_past_everything():
    """A window or a bound on the rows above what 31 bits hold is the same as none."""
    p = paged_problem([90, 33], 4, 2, 64, 16, "bf16", [3, 2], seed=9)
    want = call(p)
    assert torch.equal(call(p, window_left=2 ** 40), want)
    p["max_q"] = 2 ** 40
    assert torch.equal(call(p), want)
    from apex_attn import kv_cache_plan
    one = ints([1])
    with pytest.raises(ValueError):
        kv_cache_plan(ints([[0, 1]]), one, one, ints([2, 3]), one, 16, 2 ** 40)


def test_lse_outside_the_requests_is_zero_with_a_given_out():
    p = paged_problem([100, 50], 4, 2, 64, 16, "bf16", [2, 3], seed=5, spare_rows=9)
    torch.full((4, 14), 3.0, device="cuda")  # what a new tensor may find in its place
    out = torch.full(p["q"].shape, 7.0, dtype=p["q"].dtype, device="cuda")
    o, lse = call(p, out=out, return_lse=True)
    assert (o[5:] == 7).all() and not lse[:, 5:].any()
    assert torch.equal(lse, call(p, return_lse=True)[1])


def test_outputs_and_caches_that_overlap_themselves_are_refused():
    import apex_attn
    p = paged_problem([40, 20], 4, 2, 64, 16, "bf16", [1, 1], seed=12)
    with pytest.raises(ValueError):
        call(p, out=torch.zeros(1, 4, 64, dtype=torch.bfloat16, device="cuda").expand(2, 4, 64))
    heads_first = torch.zeros(4, 2, 64, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    assert torch.equal(call(p, out=heads_first), call(p))
    (kc, ks), (vc, vs) = p["gpu"]
    k = torch.zeros(1, 2, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError):
        apex_attn.kv_cache_append(k, k, kc[:1].expand_as(kc), vc, ks, vs, torch.zeros(1, dtype=torch.int64, device="cuda"))


def test_outputs_that_are_the_next_call_s_queries():
    """A chain of calls, each reading what the one before wrote, on one stream and captured: every call
    may start while the last is still running, and waits for it before it reads."""
    p = paged_problem([700, 33, 2100], 16, 4, 128, 32, "bf16", [1, 1, 1], seed=21)
    step = lambda x: call({**p, "q": x}, decode=True)
    want = [p["q"].cuda()]
    for _ in range(6):
        want.append(step(want[-1]))
        torch.cuda.synchronize()
    x = p["q"].cuda()
    for _ in range(6):
        x = step(x)
    assert torch.equal(x, want[-1])

    from apex_attn import custom_attention_paged_forward
    (kc, ks), (vc, vs) = p["gpu"]
    table, lens, q = ints(p["table"]), ints(p["lens"]), p["q"].cuda()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = q
        for _ in range(6):
            y = custom_attention_paged_forward(y, kc, vc, ks, vs, table, lens)
    for _ in range(3):
        y.fill_(float("nan"))
        graph.replay()
        assert torch.equal(y, want[-1])
