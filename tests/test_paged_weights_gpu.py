"""Attention over the paged 8-bit K/V cache: rows whose weights lie far apart. Needs a B200.

A row with one dominant token (an attention sink) whose V is zero is the mean of its tail, however
little of the row's weight that tail has. So the bound here is relative to the output, and has no
term in the row's largest weight:

    |o - exact| <= 2^-7 * sum_j p_j |v_j| + half a step of o's type

A weight is rounded to 11 bits (2^-11 of itself), and held to 2^-17 with the row's largest at 2^13 or
more. For the smallest tails below, 5 % over 32768 tokens, the second is at most 32768 * 2^-17 of a sum of
2^13 * 0.05 / 0.95 = 431: 2^-10.7 of it. Scores: a bf16 query value is off by up to 2^-10 where its row's
largest, here up to 32, is 256: 2^-13, over 255 keys of 0.8 each at sm_scale 1/16 that is 2^-9.3, and twice as
much for p. Sums: 3 * 1024 products of 32 tokens, 2^-23 each: 2^-11.4. Together 2^-7.8.
"""
import math

import pytest
import torch

from test_paged_gpu import DTYPES, E4M3, _b200, ints  # noqa: F401 (fixture)

pytestmark = pytest.mark.gpu

LAYOUTS = [
    # dim, heads_q, heads_kv, query tokens, dtype: the tile of 16, 32, 64 and 128 query rows of a K/V head
    (128, 4, 1, 1, "bf16"),
    (64, 32, 2, 1, "fp16"),
    (256, 16, 1, 1, "bf16"),
    (128, 24, 1, 1, "bf16"),
    (128, 8, 1, 5, "fp16"),
    (128, 8, 1, 5, "bf16"),
    (64, 4, 1, 25, "bf16"),
    (256, 8, 1, 6, "bf16"),
    (64, 8, 1, 16, "fp16"),
    (128, 16, 2, 12, "bf16"),
    (256, 16, 1, 7, "fp16"),
]


def problem(n, share, tail, peak, dim, heads_kv, heads_q, q_len, dtype, block=32, loud_block=False):
    """One request of n tokens. Every query has the same large value in dimension 0, where only the token
    at `peak` has a key; the other scores are alike (flat) or N(0, 1) (spread)."""
    g = torch.Generator(device="cuda").manual_seed(n + dim + q_len)
    blocks = -(-n // block)
    shape = (blocks, heads_kv, block, dim)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda")
    k = torch.zeros(shape, device="cuda")
    if tail == "spread":
        k[..., 1:] = rnd(blocks, heads_kv, block, dim - 1)
    k[..., 0] = 0
    k[peak // block, :, peak % block] = 0
    k[peak // block, :, peak % block, 0] = 7.0
    v = rnd(*shape) * 0.5 + 0.3
    v[peak // block, :, peak % block] = 0
    k_scale = torch.full((blocks, heads_kv), 2.0 ** -6, device="cuda")
    v_scale = torch.full((blocks, heads_kv), 2.0 ** -7, device="cuda")
    k_codes, v_codes = (k * 64).clamp(-448, 448).to(E4M3), (v * 128).clamp(-448, 448).to(E4M3)
    if loud_block:  # a block with one loud column: its scale is 2^12 times the others', its other codes 0
        loud = blocks // 2
        codes = torch.zeros((heads_kv, block, dim), device="cuda")
        codes[..., 3] = 100.0
        v_codes[loud] = codes.to(E4M3)
        v_scale[loud] *= 2.0 ** 12
    logit = math.log(n * share / (1 - share)) + (0.5 if tail == "spread" else 0.0)
    q = rnd(q_len, heads_q, dim)
    q[..., 0] = logit * math.sqrt(dim) / 7.0
    return {"q": q.to(DTYPES[dtype]), "k": k_codes, "v": v_codes, "ks": k_scale, "vs": v_scale, "n": n, "block": block}


def exact(p):
    """float64 o and sum p |v|, [query tokens, H, D]."""
    values = lambda c, s: (c.double() * s.double()[..., None, None]).transpose(0, 1).flatten(1, 2)[:, :p["n"]]
    k, v = values(p["k"], p["ks"]), values(p["v"], p["vs"])
    q_len, heads_q, dim = p["q"].shape
    group = heads_q // k.shape[0]
    k, v = k.repeat_interleave(group, 0), v.repeat_interleave(group, 0)
    s = torch.einsum("thd,hnd->thn", p["q"].double(), k) / math.sqrt(dim)
    place = p["n"] - q_len + torch.arange(q_len, device="cuda")
    hidden = torch.arange(p["n"], device="cuda") > place[:, None]
    w = torch.softmax(s.masked_fill(hidden[:, None], -torch.inf), -1)
    return torch.einsum("thn,hnd->thd", w, v), torch.einsum("thn,hnd->thd", w, v.abs())


def check(p, copies):
    """The request `copies` times in one call (the same blocks, which the call only reads)."""
    from apex_attn import custom_attention_paged_forward
    q_len = p["q"].shape[0]
    blocks = p["k"].shape[0]
    order = torch.randperm(blocks, generator=torch.Generator().manual_seed(blocks)).cuda()
    put = lambda x: torch.empty_like(x.float() if x.dtype is E4M3 else x).index_copy_(
        0, order, x.float() if x.dtype is E4M3 else x)  # block j lies at order[j]
    o = custom_attention_paged_forward(
        p["q"].repeat(copies, 1, 1), put(p["k"]).to(E4M3), put(p["v"]).to(E4M3), put(p["ks"]), put(p["vs"]),
        order.int().repeat(copies, 1), ints([p["n"]] * copies), ints([q_len * i for i in range(copies + 1)]), q_len)
    want, mass = exact(p)
    eps = torch.finfo(p["q"].dtype).eps / 2
    err = (o.double().view(copies, *want.shape) - want).abs()
    bound = 2.0 ** -7 * mass + eps * (want.abs() + 2.0 ** -7 * mass) + torch.finfo(p["q"].dtype).smallest_normal * eps
    assert (err <= bound).all(), f"off by {(err / bound).max().item():.2f} of the bound, " \
        f"{(err.norm() / want.norm() / copies ** 0.5).item():.2e} of the output"


@pytest.mark.parametrize("n", [2048, 8192, 32768])
@pytest.mark.parametrize("share", [0.5, 0.8, 0.95])
@pytest.mark.parametrize("dim,heads_q,heads_kv,q_len,dtype", LAYOUTS)
def test_one_dominant_token(n, share, dim, heads_q, heads_kv, q_len, dtype):
    for tail in ("flat", "spread"):
        for peak in (5, n - 300):
            p = problem(n, share, tail, peak, dim, heads_kv, heads_q, q_len, dtype)
            check(p, 1)     # cut into parts, one for each CTA
            check(p, 296)   # as many items as CTAs, or a multiple: every item whole


@pytest.mark.parametrize("n,share", [(2048, 0.8), (8192, 0.0005), (32768, 0.8)])
@pytest.mark.parametrize("dim,heads_q,heads_kv,q_len,dtype", LAYOUTS)
def test_one_loud_block_of_values(n, share, dim, heads_q, heads_kv, q_len, dtype):
    """A V scale 2^12 times the others': the columns that are silent in its block are the other blocks'."""
    for tail in ("flat", "spread"):
        p = problem(n, share, tail, 5, dim, heads_kv, heads_q, q_len, dtype, loud_block=True)
        check(p, 1)
        check(p, 296)


@pytest.mark.parametrize("copies", [1, 296])
@pytest.mark.parametrize("exponent", [-100, 0, 112, 118])
@pytest.mark.parametrize("dim,heads_q,heads_kv,q_len,dtype", [(64, 4, 1, 1, "bf16"), (128, 8, 1, 5, "bf16")])
def test_the_smallest_and_largest_scales_of_values(dim, heads_q, heads_kv, q_len, dtype, exponent, copies):
    """Row sums hold 1 / scale of every token: 2^100 each for 200k tokens, or 2^-118 each for some. Held to the
    bound above, and the logsumexp to 2^-16 (200k terms of fp32 sums in parts of 128 and up: 2^-20 each way)."""
    from apex_attn import custom_attention_paged_forward
    n = 200000 if exponent < 0 else 900
    p = problem(n, 0.3, "spread", 5, dim, heads_kv, heads_q, q_len, dtype, block=128)
    p["vs"] = torch.full_like(p["vs"], 2.0 ** exponent)
    if exponent > 100:  # sums of magnitudes stay below the type's largest
        p["v"] = (p["v"].float() / 64).to(E4M3)
    check(p, copies)
    table = torch.arange(p["k"].shape[0], dtype=torch.int32, device="cuda")[None]
    _, lse = custom_attention_paged_forward(p["q"], p["k"], p["v"], p["ks"], p["vs"], table, ints([n]),
                                            ints([0, q_len]), q_len, return_lse=True)
    k = (p["k"].double() * p["ks"].double()[..., None, None]).transpose(0, 1).flatten(1, 2)[0, :n]
    s = torch.einsum("thd,nd->htn", p["q"].double(), k) / math.sqrt(dim)
    s = s.masked_fill(torch.arange(n, device="cuda") > torch.arange(n - q_len, n, device="cuda")[:, None], -torch.inf)
    want = torch.logsumexp(s, -1)
    # scores: 2^-13 of 0.8 in each of 128 places at 1/8, as in the bound above
    assert ((lse.double() - want).abs() <= 2.0 ** -16 + 2.0 ** -13 * 0.8 * dim / math.sqrt(dim)).all()


@pytest.mark.parametrize("dim,heads_q,q_len,dtype", [(128, 4, 1, "fp16"), (128, 16, 8, "fp16"), (256, 16, 7, "bf16")])
def test_long_sums_of_one_sign(dim, heads_q, q_len, dtype):
    """131072 tokens with V of one sign, every item whole: three products for each 32 tokens, each sum cut by less
    than 2^-23 of itself, and weights off by 2^-11 of themselves."""
    from apex_attn import custom_attention_paged_forward
    n = 131072
    p = problem(n, 0.001, "spread", 5, dim, 1, heads_q, q_len, dtype, block=128)
    p["v"] = p["v"].float().abs().to(E4M3)
    o = custom_attention_paged_forward(p["q"].repeat(296, 1, 1), p["k"], p["v"], p["ks"], p["vs"],
                                       torch.arange(n // 128, dtype=torch.int32, device="cuda").repeat(296, 1),
                                       ints([n] * 296), ints([q_len * i for i in range(297)]), q_len)
    want, _ = exact(p)
    eps = torch.finfo(o.dtype).eps / 2
    off = ((o.double().view(296, *want.shape) - want) / want).abs().max().item()
    assert off <= 3 * n // 32 * 2.0 ** -23 + 2.0 ** -11 + eps
