"""Float64 restatement of the paged 8-bit K/V cache operators, request by request and block
by block (test infrastructure only)."""
from __future__ import annotations

import torch

E4M3_MAX = 448.0
MIN_EXPONENT = -100


def to_e4m3(x: torch.Tensor) -> torch.Tensor:
    """Rounds float64 values of magnitude <= 448 to the nearest e4m3 value, ties to even; NaN
    stays. e4m3: 4 significant bits, smallest normal 2^-6, spacing 2^-9 below it."""
    mag = x.abs()
    _, e = torch.frexp(mag)  # mag = m * 2^e, m in [0.5, 1)
    step = torch.exp2((e - 4).clamp(min=-9).to(torch.float64))
    return torch.where(torch.isnan(x), x, torch.round(x / step) * step)


def scale_of(amax: float) -> float:
    e = MIN_EXPONENT
    while E4M3_MAX * 2.0 ** e < amax:
        e += 1
    return 2.0 ** e


def append(x, codes, scale, slots, block):
    """x [total, H, D]; codes [num_blocks, H, block, D] float64 values of the codes; scale
    [num_blocks, H] float64; updated in place."""
    x = x.double()
    n, t = len(slots), 0
    limit = codes.shape[0] * block
    while t < n:
        slot = slots[t]
        if not 0 <= slot < limit:
            t += 1
            continue
        blk, o = divmod(slot, block)
        end = t + 1
        while end < n and slots[end] == slots[end - 1] + 1 and slots[end] % block != 0:
            end += 1
        for h in range(codes.shape[1]):
            values = x[t:end, h]
            finite = torch.isfinite(values)
            want = scale_of(values[finite].abs().max().item() if finite.any() else 0.0)
            old = scale[blk, h].item()
            s = max(old, want) if o else want
            if o and s != old:
                codes[blk, h, :o] = to_e4m3(codes[blk, h, :o] * (old / s))
            codes[blk, h, o:o + end - t] = to_e4m3(torch.where(finite, values, torch.nan) / s)
            scale[blk, h] = s
        t = end


def plan(table, lens, new, free, count, block, max_new):
    """Returns (slots, cu, lens, count, placed); updates table (lists of lists) in place."""
    cu, out_lens, placed, slots = [0], [], [], []
    used, short = 0, False
    for b, (held, n) in enumerate(zip(lens, new)):
        held, n = max(held, 0), max(n, 0)
        have = -(-held // block)
        need = -(-(held + n) // block) - have
        fits = have + need <= len(table[b]) and cu[-1] + n <= max_new
        ok = fits and (need == 0 or (not short and used + need <= count))
        if fits and need and not ok:
            short = True
        if ok:
            for j in range(need):
                table[b][have + j] = free[count - 1 - used - j]
            used += need
        slots += [table[b][t // block] * block + t % block if ok else -1 for t in range(held, held + n)]
        cu.append(cu[-1] + n)
        out_lens.append(held + n if ok else held)
        placed.append(int(ok))
    slots = (slots + [-1] * max_new)[:max_new]
    return slots, cu, out_lens, count - used, placed


def release(table, lens, finished, free, count, block):
    out = list(lens)
    for b, done in enumerate(finished):
        if done:
            for j in range(-(-lens[b] // block)):
                free[count] = table[b][j]
                count += 1
            out[b] = 0
    return out, count


def attend(q, k_codes, v_codes, k_scale, v_scale, table, lens, cu, block, causal=True, window=None,
           sm_scale=None):
    """q [total, H, D]; codes as values [num_blocks, H_kv, block, D]. Returns o, lse and elementwise
    bounds on what the kernels' documented roundings may move them by (before o is rounded
    to its type):

    * a weight p * v_scale is rounded to 11 bits, 2^-11 of itself, and held in terms of 8 bits that add up to
      that, or to 2^-17 with the row's largest at 2^13 or more: 2^-30 of the row's largest, or the weight itself
      where it is smaller;
    * a query value in two terms (bf16) or three (fp16): exact, or off by 2^-10 (2^-17) where its row's largest
      lies above 224;
    * fp32 products and sums: 2^-21 of the sum of magnitudes in a score; in o 2^-19, and 2^-23 for each of the
      three products of 32 tokens that are added up one after another."""
    total, heads, dim = q.shape
    group = heads // k_codes.shape[1]
    sm_scale = dim ** -0.5 if sm_scale is None else sm_scale
    o = torch.zeros((total, heads, dim), dtype=torch.float64)
    lse = torch.zeros((heads, total), dtype=torch.float64)
    o_bound, lse_bound = torch.zeros_like(o), torch.zeros_like(lse)
    lost = 2.0 ** (-17 if q.dtype is torch.float16 else -10) / 224
    q = q.double()
    for b in range(len(lens)):
        n, rows = lens[b], range(cu[b], cu[b + 1])
        ids = torch.tensor(table[b][:-(-n // block)], dtype=torch.long)
        for h in range(heads):
            hk = h // group
            kc = k_codes[ids, hk].reshape(-1, dim)[:n]
            vc = v_codes[ids, hk].reshape(-1, dim)[:n]
            ks = k_scale[ids, hk].repeat_interleave(block)[:n]
            vs = v_scale[ids, hk].repeat_interleave(block)[:n]
            for r in rows:
                place = n - len(rows) + r - cu[b]
                hi = min(place + 1, n) if causal else n
                lo = max(place - window, 0) if window is not None else 0
                if hi <= lo:
                    lse[h, r] = -torch.inf
                    continue
                k, v = kc[lo:hi] * ks[lo:hi, None], vc[lo:hi] * vs[lo:hi, None]
                s = (k @ q[r, h]) * sm_scale
                lse[h, r] = torch.logsumexp(s, 0)
                p = torch.exp(s - lse[h, r])
                o[r, h] = p @ v
                biggest = q[r, h].abs().max()
                off = sm_scale * (k.abs().sum(1) * (biggest * lost) + (k.abs() @ q[r, h].abs()) * 2.0 ** -21)
                off = off.max().item() + 2.0 ** -20 * (1 + abs(lse[h, r].item()))
                lse_bound[h, r] = off
                w = p * vs[lo:hi]
                floor = torch.minimum(w, 2.0 ** -30 * w.max()) @ vc[lo:hi].abs()
                steps = 3 * -(-(hi - lo) // 32)
                o_bound[r, h] = (p @ v.abs()) * (2.0 ** -11 + 2 * off + 2.0 ** -19 + steps * 2.0 ** -23) + floor
    return o, lse, o_bound, lse_bound
