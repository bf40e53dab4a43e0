"""Refusals of the paged 8-bit K/V cache operators, and their oracle against plain formulas;
needs no GPU."""
import ctypes

import pytest
import torch

from apex_attn import _lib
from oracle import paged_oracle as ref

FAKE = 0x10000  # 16-byte aligned, never dereferenced: validation fails first
BAD, DIM, DTYPE, LAYOUT, SCALE, NODEV, LARGE = (
    _lib.ERR_INVALID_ARGUMENT, _lib.ERR_UNSUPPORTED_HEAD_DIM, _lib.ERR_UNSUPPORTED_DTYPE, _lib.ERR_BAD_LAYOUT,
    _lib.ERR_BAD_SCALE, _lib.ERR_NO_DEVICE, _lib.ERR_TOO_LARGE)


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


# ------------------------------------------------------------------------- C ABI --
def plan_args(**kw):
    base = dict(block_table=FAKE, seq_lens=FAKE, new_lens=FAKE, finished=FAKE, free_blocks=FAKE, free_count=FAKE,
                slots=FAKE, cu_seqlens=FAKE, seq_lens_out=FAKE + 64, free_count_out=FAKE + 128, placed=FAKE,
                table_stride=4, batch=2, table_width=4, free_capacity=8, block_size=16, max_new_tokens=5)
    return _lib.KVPlanArgs(**{**base, **kw})


PLAN_BAD = [({n: None}, BAD) for n in ("block_table", "seq_lens", "free_blocks", "free_count", "seq_lens_out",
                                       "free_count_out")] + [
    ({"batch": 0}, BAD), ({"batch": -1}, BAD), ({"table_width": 0}, BAD), ({"free_capacity": 0}, BAD),
    ({"block_size": 8}, BAD), ({"block_size": 48}, BAD), ({"block_size": 256}, BAD), ({"block_size": 0}, BAD),
    ({"batch": 8193}, LARGE), ({"table_width": 1 << 28, "table_stride": 1 << 28}, LARGE),
    ({"free_capacity": (1 << 30) + 1}, LARGE), ({"table_stride": 3}, LAYOUT), ({"block_table": FAKE + 2}, LAYOUT),
    ({"seq_lens_out": FAKE}, BAD), ({"free_count_out": FAKE}, BAD)]


@pytest.mark.parametrize("kw,code", PLAN_BAD + [
    ({"new_lens": None}, BAD), ({"slots": None}, BAD), ({"cu_seqlens": None}, BAD), ({"placed": None}, BAD),
    ({"max_new_tokens": 0}, BAD), ({"max_new_tokens": (1 << 30) + 1}, LARGE), ({"slots": FAKE + 4}, LAYOUT)])
def test_plan_refuses(lib, kw, code):
    assert lib.apex_attn_kv_plan(ctypes.byref(plan_args(**kw)), None) == code


@pytest.mark.parametrize("kw,code", PLAN_BAD + [({"finished": None}, BAD)])
def test_release_refuses(lib, kw, code):
    assert lib.apex_attn_kv_release(ctypes.byref(plan_args(**kw)), None) == code


def append_args(strides=(256, 64, 256, 64, 2048, 1024, 64, 2048, 1024, 64), **kw):
    base = dict(k=FAKE, v=FAKE, k_cache=FAKE, v_cache=FAKE, k_scale=FAKE, v_scale=FAKE, slots=FAKE, total=3,
                heads_kv=2, head_dim=64, dtype=0, num_blocks=4, block_size=16,
                strides=(ctypes.c_longlong * 10)(*strides))
    return _lib.KVAppendArgs(**{**base, **kw})


def with_stride(i, value, base=(256, 64, 256, 64, 2048, 1024, 64, 2048, 1024, 64)):
    s = list(base)
    s[i] = value
    return (ctypes.c_longlong * 10)(*s)


@pytest.mark.parametrize("kw,code", [({n: None}, BAD) for n in ("k", "v", "k_cache", "v_cache", "k_scale", "v_scale",
                                                               "slots")] + [
    ({"total": 0}, BAD), ({"heads_kv": 0}, BAD), ({"num_blocks": 0}, BAD), ({"block_size": 20}, BAD),
    ({"head_dim": 96}, DIM), ({"head_dim": 0}, DIM), ({"dtype": 2}, DTYPE), ({"total": (1 << 30) + 1}, LARGE),
    ({"heads_kv": 65536}, LARGE), ({"strides": with_stride(0, 4)}, LAYOUT), ({"strides": with_stride(3, -8)}, LAYOUT),
    ({"strides": with_stride(4, 8)}, LAYOUT), ({"strides": with_stride(6, 48)}, LAYOUT),
    ({"strides": with_stride(9, 0)}, LAYOUT), ({"strides": with_stride(5, 1 << 38)}, LAYOUT),
    ({"k": FAKE + 8}, LAYOUT), ({"v_cache": FAKE + 8}, LAYOUT), ({"slots": FAKE + 4}, LAYOUT),
    ({"k_scale": FAKE + 2}, LAYOUT)])
def test_append_refuses(lib, kw, code):
    assert lib.apex_attn_kv_append(ctypes.byref(append_args(**kw)), None) == code


PAGED_STRIDES = (256, 64, 256, 64, 2048, 1024, 64, 2048, 1024, 64)


def paged_args(**kw):
    base = dict(q=FAKE, k_cache=FAKE, v_cache=FAKE, k_scale=FAKE, v_scale=FAKE, block_table=FAKE, seq_lens=FAKE,
                cu_seqlens_q=FAKE, o=FAKE, lse=None, table_stride=4, strides=(ctypes.c_longlong * 10)(*PAGED_STRIDES),
                batch=2, heads_q=4, heads_kv=2, total_q=6, max_seqlen_q=3, head_dim=64, dtype=0, num_blocks=4,
                block_size=16, table_width=4, causal=1, window_left=-1, zero_rest=0, sm_scale=0.125)
    return _lib.PagedArgs(**{**base, **kw})


def paged(lib, workspace=FAKE, bytes_=1 << 30, **kw):
    return lib.apex_attn_fwd_paged(ctypes.byref(paged_args(**kw)), workspace, bytes_, None)


@pytest.mark.parametrize("kw,code", [({n: None}, BAD) for n in (
    "q", "k_cache", "v_cache", "k_scale", "v_scale", "block_table", "seq_lens", "o", "workspace")] + [
    ({n: 0}, BAD) for n in ("batch", "heads_q", "heads_kv", "total_q", "max_seqlen_q", "num_blocks", "table_width")] + [
    ({"heads_kv": 3}, BAD), ({"block_size": 12}, BAD), ({"window_left": -2}, BAD),
    ({"window_left": 4, "causal": 0}, BAD), ({"cu_seqlens_q": None, "total_q": 7}, BAD),
    ({"cu_seqlens_q": None, "max_seqlen_q": 2}, BAD), ({"head_dim": 80}, DIM), ({"dtype": 7}, DTYPE),
    ({"sm_scale": 0.0}, SCALE), ({"sm_scale": float("nan")}, SCALE), ({"sm_scale": float("inf")}, SCALE),
    ({"batch": 65536}, LARGE), ({"max_seqlen_q": 1 << 29}, LARGE),
    ({"table_width": 1 << 27, "table_stride": 1 << 27}, LARGE), ({"table_stride": 3}, LAYOUT),
    ({"strides": with_stride(1, 12)}, LAYOUT), ({"strides": with_stride(3, 32)}, LAYOUT),
    ({"strides": with_stride(4, 24)}, LAYOUT), ({"strides": with_stride(9, 32)}, LAYOUT),
    ({"q": FAKE + 8}, LAYOUT), ({"o": FAKE + 2}, LAYOUT), ({"k_cache": FAKE + 1}, LAYOUT),
    ({"workspace": FAKE + 4}, LAYOUT), ({"lse": FAKE + 2}, LAYOUT), ({"seq_lens": FAKE + 2}, LAYOUT),
    ({"bytes_": 0}, BAD)])
def test_attention_refuses(lib, kw, code):
    assert paged(lib, **kw) == code


def test_packed_layouts_are_the_structs():
    for packed, mirror in ((_lib.KV_PLAN_ARGS, _lib.KVPlanArgs), (_lib.KV_APPEND_ARGS, _lib.KVAppendArgs),
                           (_lib.PAGED_ARGS, _lib.PagedArgs)):
        assert -(-packed.size // 8) * 8 == ctypes.sizeof(mirror)
        values = list(range(1, len(packed.unpack(bytes(packed.size))) + 1))
        got = mirror.from_buffer_copy(packed.pack(*values).ljust(ctypes.sizeof(mirror), b"\0"))
        flat = []
        for name, _ in mirror._fields_:
            x = getattr(got, name)
            flat += list(x) if hasattr(x, "__len__") else [x]
        assert flat == values


def test_known_device_out_of_range(lib):
    assert paged(lib, known_device=65) == NODEV
    assert paged(lib, known_device=-1) == NODEV


def test_null_argument_structs(lib):
    for fn in (lib.apex_attn_kv_plan, lib.apex_attn_kv_release, lib.apex_attn_kv_append):
        assert fn(None, None) == BAD
    assert lib.apex_attn_fwd_paged(None, FAKE, 1 << 20, None) == BAD


def test_pointers_that_are_no_device_memory(lib):
    assert paged(lib) == NODEV
    assert lib.apex_attn_kv_plan(ctypes.byref(plan_args()), None) == NODEV
    assert lib.apex_attn_kv_release(ctypes.byref(plan_args()), None) == NODEV
    assert lib.apex_attn_kv_append(ctypes.byref(append_args()), None) == NODEV


def test_workspace_bytes(lib):
    ws = lib.apex_attn_fwd_paged_workspace_bytes
    assert ws(0, 1, 1, 64) == ws(1, 0, 1, 64) == ws(1, 1, 0, 64) == ws(1, 1, 1, 0) == 0
    assert ws(32, 8, 1, 128) > 0


# ------------------------------------------------------------------------ Python --
def operands(**kw):
    t = {"q": torch.zeros(2, 4, 64, dtype=torch.bfloat16), "k_cache": torch.zeros(3, 2, 16, 64).to(torch.float8_e4m3fn),
         "v_cache": torch.zeros(3, 2, 16, 64).to(torch.float8_e4m3fn), "k_scale": torch.ones(3, 2),
         "v_scale": torch.ones(3, 2), "block_table": torch.zeros(2, 4, dtype=torch.int32),
         "seq_lens": torch.ones(2, dtype=torch.int32)}
    return {**t, **kw}


def test_python_refuses_what_is_not_on_a_gpu():
    import apex_attn
    t = operands()
    with pytest.raises(ValueError):
        apex_attn.custom_attention_paged_forward(**t)
    with pytest.raises(ValueError):
        apex_attn.kv_cache_append(t["q"][:, :2], t["q"][:, :2], t["k_cache"], t["v_cache"], t["k_scale"], t["v_scale"],
                                  torch.zeros(2, dtype=torch.int64))
    one = torch.ones(1, dtype=torch.int32)
    with pytest.raises(ValueError):
        apex_attn.kv_cache_plan(t["block_table"], t["seq_lens"], t["seq_lens"], one, one, 16, 4)
    with pytest.raises(ValueError):
        apex_attn.kv_cache_release(t["block_table"], t["seq_lens"], t["seq_lens"], one, one, 16)


@pytest.mark.parametrize("kw,error", [
    ({"q": torch.zeros(2, 256, dtype=torch.bfloat16)}, ValueError),
    ({"q": torch.zeros(2, 4, 64)}, TypeError)])
def test_python_refuses_q(kw, error):
    import apex_attn
    with pytest.raises(error):
        apex_attn.custom_attention_paged_forward(**operands(**kw))


# ------------------------------------------------------------------------ oracle --
def test_oracle_rounding_is_torchs():
    x = torch.cat([torch.linspace(-448, 448, 20011), torch.linspace(-0.05, 0.05, 20011),
                   torch.tensor([0.0, 2.0 ** -10, 3 * 2.0 ** -10, 2.0 ** -9, 17.0, 19.0, 448.0])])
    assert torch.equal(ref.to_e4m3(x.double()).float(), x.to(torch.float8_e4m3fn).float())


def test_oracle_attention_is_softmax_of_the_values():
    g = torch.Generator().manual_seed(0)
    codes = [(torch.randn(4, 2, 16, 64, generator=g) * 90).clamp(-448, 448).to(torch.float8_e4m3fn).double()
             for _ in range(2)]
    scale = [torch.exp2(torch.randint(-8, -5, (4, 2), generator=g).double()) for _ in range(2)]
    q = torch.randn(3, 4, 64, generator=g, dtype=torch.float64)
    table, n = [[2, 0, 3]], 40
    o, lse, _, _ = ref.attend(q, *codes, *scale, table, [n], [0, 3], 16)
    k, v = ((c * s[..., None, None])[table[0]].transpose(0, 1).reshape(2, 48, 64)[:, :n].repeat_interleave(2, 0)
            for c, s in zip(codes, scale))
    s = torch.einsum("thd,hnd->htn", q, k) / 8
    s = s.masked_fill(torch.arange(n) > torch.tensor([37, 38, 39])[:, None], -torch.inf)
    assert torch.allclose(lse, torch.logsumexp(s, -1), atol=1e-12)
    assert torch.allclose(o, torch.einsum("htn,hnd->thd", torch.softmax(s, -1), v), atol=1e-12)


def test_oracle_plan_and_release_return_to_the_start():
    table, free = [[0] * 5 for _ in range(3)], list(range(9))
    slots, cu, lens, count, placed = ref.plan(table, [0, 0, 0], [20, 1, 33], free, 9, 16, 60)
    assert placed == [1, 1, 1] and cu == [0, 20, 21, 54] and count == 3
    assert slots[:16] == [8 * 16 + i for i in range(16)] and slots[20] == 6 * 16 and slots[54:] == [-1] * 6
    lens, count = ref.release(table, lens, [1, 1, 1], free, count, 16)
    assert lens == [0, 0, 0] and count == 9 and sorted(free) == list(range(9))


@pytest.mark.parametrize("i,value", [(4, 0), (4, 1024), (7, 2032), (5, 0), (5, 1008), (8, 64)])
def test_append_refuses_caches_that_overlap_themselves(lib, i, value):
    """Blocks, heads or tokens that share bytes (an expanded cache) would be written twice at once."""
    args = append_args(with_stride(i, value))
    assert lib.apex_attn_kv_append(ctypes.byref(args), None) == LAYOUT


@pytest.mark.parametrize("kv", [0, 1])
def test_append_takes_caches_in_any_order_of_dimensions(lib, kv):
    """Heads outside the blocks, tokens outside the heads, K and V in one storage: past the layout's
    checks, where the made-up pointers are refused."""
    for sb, sh, st in [(1024, 4096, 64), (128, 64, 512), (4096, 64, 256), (64, 16 * 256, 256)]:
        strides = [256, 64, 256, 64, 2048, 1024, 64, 2048, 1024, 64]
        strides[4 + 3 * kv:7 + 3 * kv] = [sb, sh, st]
        assert lib.apex_attn_kv_append(ctypes.byref(append_args(tuple(strides))), None) == NODEV


@pytest.mark.parametrize("tokens,heads,ok", [(256, 64, True), (64, 192, True), (0, 64, False), (128, 64, False),
                                             (64, 128, False), (192, 64, False), (1024, 256, True)])
def test_attention_refuses_outputs_whose_rows_overlap(lib, tokens, heads, ok):
    """Three tokens of four heads of 64."""
    strides = (256, 64, tokens, heads, 2048, 1024, 64, 2048, 1024, 64)
    got = paged(lib, total_q=3, heads_q=4, heads_kv=2, head_dim=64, batch=3, max_seqlen_q=1,
                strides=(ctypes.c_longlong * 10)(*strides))
    assert got == (NODEV if ok else LAYOUT)
