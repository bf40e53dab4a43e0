"""The oracle's bound on attention over the paged 8-bit K/V cache, against weights that are held too
coarsely; needs no GPU. Mistakes are planted in a restatement of the weights' rounding."""
import math

import pytest
import torch

from oracle import paged_oracle as ref

BLOCK, DIM = 16, 64
E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2


def held(w, terms, top):
    """Weights as terms of 8 bits, the largest at 2^top."""
    a = (w / w.max() * 2.0 ** top).half().double()
    out = torch.zeros_like(a)
    for t in terms:
        x = a.float().to(t).double()
        out, a = out + x, a - x
    return out * w.max() / 2.0 ** top


def problem(n, share, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    blocks = -(-n // BLOCK)
    k, v = (torch.zeros(blocks, 1, BLOCK, DIM, dtype=torch.float64) for _ in range(2))
    v[:] = (torch.randn(v.shape, generator=g) * 60 + 40).clamp(-448, 448).to(E4M3).double()
    scale = torch.full((blocks, 1), 2.0 ** -7, dtype=torch.float64)
    q = torch.randn(1, 1, DIM, generator=g)
    if share:
        k[0, 0, 0, 0], v[0, 0, 0] = 448.0, 0.0
        q[..., 0] = math.log(n * share / (1 - share)) * math.sqrt(DIM) / 3.5
    else:
        k[:] = (torch.randn(k.shape, generator=g) * 90).clamp(-448, 448).to(E4M3).double()
    return q.to(dtype), k, v, scale, [list(range(blocks))], [n]


def over_bound(p, terms, top):
    """By how much o from such weights passes the oracle's bound at most, as a multiple of it."""
    q, k, v, scale, table, lens = p
    o, _, bound, _ = ref.attend(q, k, v, scale, scale, table, lens, [0, 1], BLOCK)
    keys, values = ((c * scale[..., None, None]).reshape(-1, DIM)[:lens[0]] for c in (k, v))
    w = torch.softmax(keys @ q[0, 0].double() / math.sqrt(DIM), 0)
    got = held(w, terms, top) @ values
    return ((got - o[0, 0]).abs() / bound[0, 0]).max().item()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,share", [(2000, 0.95), (8192, 0.95), (32768, 0.8), (40, 0), (1200, 0)])
def test_three_terms_of_e5m2_are_within_the_bound(n, share, dtype):
    assert over_bound(problem(n, share, dtype), (E5M2,) * 3, 13) <= 1


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("terms", [(E4M3,) * 2, (E4M3, E5M2), (E4M3, E4M3, E5M2)])
def test_a_lost_or_coarse_tail_passes_the_bound(terms, dtype):
    assert over_bound(problem(8192, 0.95, dtype), terms, 6) > 8


@pytest.mark.parametrize("terms,top", [((E4M3,) * 2, 6), ((E5M2,) * 2, 13), ((E4M3, E5M2), 6)])
def test_weights_of_too_few_bits_pass_the_bound(terms, top):
    worst = max(over_bound(problem(n, 0, torch.float16, seed), terms, top) for n in (2, 3, 5) for seed in range(6))
    assert worst > 1
