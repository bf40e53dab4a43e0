"""Workloads of the 8-bit paged K/V cache operators, for measuring them.

Three kinds of pass, each as a serving program makes it:

* ``attend``: attention of new query tokens over a cache held in e4m3 with one fp32 scale
  per (block of tokens, K/V head): ``custom_attention_paged_forward``;
* ``append``: new K/V tokens are quantised into their slots of such a cache:
  ``kv_cache_append``;
* ``plan``: one scheduling step on the GPU: the blocks of finished requests go back to the
  free list, new tokens get blocks, table entries and slots: ``kv_cache_release`` and
  ``kv_cache_plan``.

With ``own`` false, ``run`` computes the same in elementary torch operations.
"""
import math
import os
import random
import sys

import torch

own = False

E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0
MIN_EXPONENT = -100  # the smallest scale that an append writes is 2^-100

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _library():
    """The framework's package (kept below the repository's root)."""
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "apex-tune-results_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import apex_attn
    return apex_attn


# ------------------------------------------------------------------------- cases --
def _attend(name, batch, heads_q, heads_kv, dim, block, dtype, q_len, k_min, k_max, window=-1,
            token_major=False, lse=False):
    c = {"op": "attend", "batch": batch, "heads_q": heads_q, "heads_kv": heads_kv, "dim": dim, "block": block,
         "dtype": dtype, "q_len": q_len, "k_min": k_min, "k_max": k_max, "window": window,
         "token_major": token_major, "lse": lse}
    return dict(c, name=name) if name else c


def _append(name, batch, heads_kv, dim, block, dtype, new_min, new_max, held_max, token_major=False):
    c = {"op": "append", "batch": batch, "heads_kv": heads_kv, "dim": dim, "block": block, "dtype": dtype,
         "new_min": new_min, "new_max": new_max, "held_max": held_max, "token_major": token_major}
    return dict(c, name=name) if name else c


def _plan(name, batch, block, held_max, new_max, prompts):
    c = {"op": "plan", "batch": batch, "block": block, "held_max": held_max, "new_max": new_max,
         "prompts": prompts}
    return dict(c, name=name) if name else c


def listed():
    return [
        # One user's next token over a short context: latency is all that counts.
        _attend("attend_one", 1, 16, 4, 64, 16, "bf16", 1, 1000, 1000),
        # The decode step of a busy server: ragged contexts, grouped-query heads.
        _attend("attend_batch", 48, 32, 8, 128, 32, "bf16", 1, 129, 8191),
        # Two long documents: few rows, so the work has to be split along the cache. The cache
        # stores tokens before heads, and the logsumexp is kept to merge with another cache.
        _attend("attend_long", 2, 64, 8, 128, 64, "fp16", 1, 130001, 131072, token_major=True, lse=True),
        # Wide heads in small blocks.
        _attend("attend_wide", 24, 16, 2, 256, 16, "bf16", 1, 2050, 8192),
        # Draft tokens of each request verified at once, ragged counts, under a sliding window.
        _attend("attend_draft", 32, 32, 4, 128, 16, "fp16", 5, 700, 8192, window=1024, lse=True),
        # Chunks of prompts that continue a cached prefix: bound by the matrix products.
        _attend("attend_chunk", 3, 32, 8, 128, 128, "bf16", 1024, 5000, 16384),
        # The K/V write of one decode step.
        _append("append_step", 64, 8, 128, 32, "bf16", 1, 1, 8192),
        # The K/V write of a batch of prompts and continued chunks.
        _append("append_prompt", 24, 8, 128, 16, "fp16", 33, 2048, 300, token_major=True),
        # A few draft tokens for wide heads in large blocks.
        _append("append_wide", 7, 2, 256, 128, "bf16", 1, 6, 1000),
        # A decode step's bookkeeping: one token each, few requests cross into a new block.
        _plan("plan_step", 64, 16, 8192, 1, 0),
        # Many requests with a wave of admitted prompts.
        _plan("plan_prompts", 1024, 32, 16384, 1, 48),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "append", "append", "plan"])
    block = rng.choice([16, 32, 64, 128])
    if op == "plan":
        return _plan(None, _log_int(rng, 3, 1024), block, _log_int(rng, 200, 16384), rng.choice([1, 1, 2, 5]),
                     rng.randint(0, 20))
    dim = rng.choice([64, 128, 128, 256])
    dtype = rng.choice(["bf16", "fp16"])
    heads_kv = rng.choice([1, 2, 4, 8])
    if op == "append":
        new_max = rng.choice([1, 7, _log_int(rng, 16, 2048)])
        batch = _log_int(rng, 1, 200 if new_max < 16 else 16)
        return _append(None, batch, heads_kv, dim, block, dtype, rng.randint(1, new_max), new_max,
                       _log_int(rng, 1, 4096), rng.random() < 0.5)
    group = rng.choice([1, 2, 4, 5, 8])
    q_len = rng.choice([1, 1, 1, rng.randint(2, 8), _log_int(rng, 16, 700)])
    window = rng.choice([-1, -1, -1, rng.randint(1, 4000)])
    k_max = _log_int(rng, max(100, q_len), 100000 if q_len == 1 else 12000)
    batch = _log_int(rng, 1, max(1, min(128, 300000 // k_max, 2000 // q_len)))
    k_min = rng.randint(max(1, q_len), k_max)
    token_major, lse = rng.random() < 0.5, rng.random() < 0.5
    while True:  # no drawn case costs more than the largest listed one
        c = _attend(None, batch, group * heads_kv, heads_kv, dim, block, dtype, q_len, k_min, k_max, window,
                    token_major, lse)
        w = work(c)
        if batch == 1 or (w["bytes"] < 5e8 and w["flops"] < 4e11):
            return c
        batch = batch * 2 // 3


# ------------------------------------------------------------------------ inputs --
def _spread(lo, hi, n):
    """n whole numbers evenly spread over [lo, hi] (so their sum goes by the case alone)."""
    return [hi - (hi - lo) * i // max(1, n - 1) for i in range(n)]


def _shuffled(values, seed):
    values = list(values)
    random.Random(seed).shuffle(values)
    return values


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _cumulated(values):
    out = [0]
    for v in values:
        out.append(out[-1] + v)
    return out


def _cache(blocks, heads, block, dim, token_major, gen):
    """Cache values of unit size or so, whose blocks and heads differ in range: codes and scales."""
    shape = (blocks, block, heads, dim) if token_major else (blocks, heads, block, dim)
    codes = torch.empty(shape, dtype=E4M3, device="cuda")
    step = max(1, (1 << 26) // max(1, block * heads * dim))
    for i in range(0, blocks, step):
        part = torch.randn((min(step, blocks - i),) + shape[1:], generator=gen, device="cuda")
        codes[i:i + step] = part.mul_(90.0).clamp_(-E4M3_MAX, E4M3_MAX).to(E4M3)
    if token_major:
        codes = codes.transpose(1, 2)
    exponent = torch.randint(-8, -5, (blocks, heads), generator=gen, device="cuda")
    return codes, torch.exp2(exponent.float())


def _table(counts, width, spare, gen):
    """Block ids of each request in a random order, and the ids that are left over."""
    total = sum(counts)
    ids = torch.randperm(total + spare, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros((len(counts), width), dtype=torch.int32, device="cuda")
    start = torch.tensor(_cumulated(counts)[:-1], device="cuda")[:, None]
    count = torch.tensor(counts, device="cuda")[:, None]
    j = torch.arange(width, device="cuda")[None, :]
    held = j < count
    table[held] = ids[(start + j)[held]]
    return table, ids[total:].clone()


def _query_lens(case):
    """Ragged where a request brings several tokens, one each otherwise."""
    return _spread((case["q_len"] + 1) // 2, case["q_len"], case["batch"])


def _key_lens(case):
    return [max(a, b) for a, b in zip(_spread(case["k_min"], case["k_max"], case["batch"]), _query_lens(case))]


def _new_lens(case):
    return _spread(case["new_min"], case["new_max"], case["batch"])


def _held_lens(case):
    return _spread(0, case["held_max"], case["batch"])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    if case["op"] == "attend":
        order = _shuffled(range(case["batch"]), seed)
        q_lens = [_query_lens(case)[i] for i in order]
        k_lens = [_key_lens(case)[i] for i in order]
        block, dtype = case["block"], _DTYPES[case["dtype"]]
        counts = [-(-n // block) for n in k_lens]
        s["block_table"], _ = _table(counts, max(counts), 3, gen)
        s["k_cache"], s["k_scale"] = _cache(sum(counts) + 3, case["heads_kv"], block, case["dim"], case["token_major"], gen)
        s["v_cache"], s["v_scale"] = _cache(sum(counts) + 3, case["heads_kv"], block, case["dim"], case["token_major"], gen)
        s["q"] = torch.randn((sum(q_lens), case["heads_q"], case["dim"]), generator=gen, device="cuda").to(dtype)
        s["seq_lens"], s["cu_seqlens"] = _ints(k_lens), _ints(_cumulated(q_lens))
    elif case["op"] == "append":
        order = _shuffled(range(case["batch"]), seed)
        new = [_new_lens(case)[i] for i in order]
        held = _shuffled(_held_lens(case), seed + 1)
        block, dtype = case["block"], _DTYPES[case["dtype"]]
        counts = [-(-(h + n) // block) for h, n in zip(held, new)]
        blocks = (sum(held) + sum(new)) // block + len(new)  # at least sum(counts), the same for every seed
        table, _ = _table(counts, max(counts), blocks - sum(counts), gen)
        s["k_cache"], s["k_scale"] = _cache(blocks, case["heads_kv"], block, case["dim"], case["token_major"], gen)
        s["v_cache"], s["v_scale"] = _cache(blocks, case["heads_kv"], block, case["dim"], case["token_major"], gen)
        shape = (sum(new), case["heads_kv"], case["dim"])
        s["k"] = (torch.randn(shape, generator=gen, device="cuda") * 3).to(dtype)
        s["v"] = torch.randn(shape, generator=gen, device="cuda").to(dtype)
        request = torch.repeat_interleave(torch.arange(len(new), device="cuda"), torch.tensor(new, device="cuda"))
        at = (torch.arange(sum(new), device="cuda") - torch.tensor(_cumulated(new), device="cuda")[request]
              + torch.tensor(held, device="cuda")[request])
        s["slots"] = table[request, at // block].long() * block + at % block
    else:
        held, new, done = _plan_lens(case)
        order = _shuffled(range(case["batch"]), seed)
        held, new, done = ([v[i] for i in order] for v in (held, new, done))
        block = case["block"]
        counts = [-(-h // block) for h in held]
        width = max(-(-(h + n) // block) for h, n in zip(held, new))
        need = sum(-(-n // block) + 1 for n in new)
        s["block_table"], left = _table(counts, width, need + 5, gen)
        s["free_blocks"] = torch.zeros(sum(counts) + need + 5, dtype=torch.int32, device="cuda")
        s["free_blocks"][:left.numel()] = left
        s["free_count"] = _ints([left.numel()])
        s["seq_lens"], s["new_lens"], s["finished"] = _ints(held), _ints(new), _ints(done)
        s["max_new_tokens"] = sum(new) + 7  # a program pads the step to a fixed size
    return s


def _plan_lens(case):
    """Running requests, then finished ones, then admitted prompts (in rows that hold nothing)."""
    batch, prompts = case["batch"], min(case["prompts"], case["batch"] - 1)
    finished = prompts if batch - 2 * prompts > 0 else 0
    running = batch - prompts
    held = _spread(1, case["held_max"], running) + [0] * prompts
    done = [0] * (running - finished) + [1] * finished + [0] * prompts
    new = _spread(1, case["new_max"], running - finished) + [0] * finished + _spread(50, 2100, prompts)
    return held, new, done


# ----------------------------------------------------------------- plain operators --
def _plain_attend(s):
    c = s["case"]
    table, lens, cu, q = s["block_table"].long(), s["seq_lens"].long(), s["cu_seqlens"].long(), s["q"]
    batch, width = table.shape
    group, dim, longest = c["heads_q"] // c["heads_kv"], c["dim"], c["q_len"]
    length = width * c["block"]

    def gathered(codes, scale):
        x = codes[table].float() * scale[table][..., None, None]  # [B, blocks, heads, block, D]
        return x.permute(0, 2, 1, 3, 4).reshape(batch, c["heads_kv"], length, dim)

    row = torch.arange(q.shape[0], device=q.device)
    request = torch.searchsorted(cu, row, right=True) - 1
    token = row - cu[request]
    padded = torch.zeros((batch, longest, c["heads_q"], dim), device=q.device)
    padded[request, token] = q.float()
    padded = padded.view(batch, longest, c["heads_kv"], group, dim).permute(0, 2, 1, 3, 4)
    padded = padded.reshape(batch, c["heads_kv"], longest * group, dim)
    scores = torch.matmul(padded, gathered(s["k_cache"], s["k_scale"]).transpose(2, 3)) / math.sqrt(dim)
    at = torch.arange(length, device=q.device)
    here = (lens - (cu[1:] - cu[:-1]))[:, None] + torch.arange(longest, device=q.device)  # a query token's place
    seen = (at <= here[..., None]) & (at < lens[:, None, None])
    if c["window"] >= 0:
        seen &= at >= here[..., None] - c["window"]
    seen = seen.repeat_interleave(group, dim=1)[:, None]
    scores = scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    weights = scores.sub_(top).exp_()
    total = weights.sum(-1, keepdim=True)
    o = torch.matmul(weights, gathered(s["v_cache"], s["v_scale"]))
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    lse = (top + total.log())[..., 0]

    def packed(x, *tail):
        x = x.view(batch, c["heads_kv"], longest, group, *tail).transpose(1, 2)
        return x.reshape(batch, longest, c["heads_q"], *tail)[request, token]

    o = packed(o, dim).to(q.dtype)
    return [o, packed(lse).t().contiguous()] if c["lse"] else [o]


def _plain_append_one(x, cache, scale, slots, block):
    held, inverse = torch.unique(slots // block, return_inverse=True)
    offset = slots % block
    x = x.float()
    heads, dim = x.shape[1:]
    top = torch.zeros((held.numel(), heads), device=x.device)
    top.scatter_reduce_(0, inverse[:, None].expand(-1, heads), x.abs().amax(-1), "amax")
    first = torch.full((held.numel(),), block, device=x.device).scatter_reduce_(0, inverse, offset, "amin")
    mantissa, exponent = torch.frexp(top)  # top = mantissa * 2^exponent, and 448 = 0.875 * 2^9
    exponent = (exponent - torch.where(mantissa <= 0.875, 9, 8)).clamp(min=MIN_EXPONENT)
    exponent = torch.where(top == 0, MIN_EXPONENT, exponent)
    wanted = torch.ldexp(torch.ones_like(top), exponent)
    before = scale[held]
    after = torch.where(first[:, None] > 0, torch.maximum(before, wanted), wanted)
    codes = cache[held].float()
    changed = (codes * (before / after)[..., None, None]).to(E4M3)
    stays = torch.arange(block, device=x.device)[None, :] < first[:, None]
    changed = torch.where(stays[:, None, :, None], changed.float(), codes)
    changed[inverse, :, offset] = (x / after[inverse][..., None]).clamp(-E4M3_MAX, E4M3_MAX)
    cache[held] = changed.to(E4M3)
    scale[held] = after


def _plain_append(s):
    block = s["case"]["block"]
    _plain_append_one(s["k"], s["k_cache"], s["k_scale"], s["slots"], block)
    _plain_append_one(s["v"], s["v_cache"], s["v_scale"], s["slots"], block)
    return [s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]]


def _plain_plan(s):
    block, table, free = s["case"]["block"], s["block_table"], s["free_blocks"]
    lens, new, count = s["seq_lens"].long(), s["new_lens"].long(), s["free_count"].long()
    batch, width = table.shape
    column = torch.arange(width, device=table.device)
    # Finished requests: their blocks go on top of the stack of free ones, in order.
    have = (lens + block - 1) // block
    gone = torch.where(s["finished"] != 0, have, torch.zeros_like(have))
    base = gone.cumsum(0) - gone
    back = column < gone[:, None]
    free[(count + base[:, None] + column)[back]] = table[back]
    count = count + gone.sum()
    lens = torch.where(s["finished"] != 0, torch.zeros_like(lens), lens)
    # New tokens: blocks come off the top, request by request.
    have = (lens + block - 1) // block
    need = (lens + new + block - 1) // block - have
    fits = (lens + new + block - 1) // block <= width
    need = torch.where(fits, need, torch.zeros_like(need))
    base = need.cumsum(0) - need
    placed = fits & ((need == 0) | (base + need <= count))
    need = torch.where(placed, need, torch.zeros_like(need))
    taken = (column >= have[:, None]) & (column < (have + need)[:, None])
    table[taken] = free[(count - 1 - base[:, None] - column + have[:, None])[taken]]
    cu = torch.zeros(batch + 1, dtype=torch.long, device=table.device)
    cu[1:] = new.cumsum(0)
    row = torch.arange(s["max_new_tokens"], device=table.device)
    request = (torch.searchsorted(cu, row, right=True) - 1).clamp(max=batch - 1)
    at = lens[request] + row - cu[request]
    real = (row < cu[-1]) & placed[request]
    slots = table[request, (at // block).clamp(max=width - 1)].long() * block + at % block
    slots = torch.where(real, slots, torch.full_like(slots, -1))
    lens = lens + torch.where(placed, new, torch.zeros_like(new))
    count = count - need.sum()
    return [slots, cu.int(), lens.int(), count.int(), placed.int(), table, free]


# --------------------------------------------------------------- the framework's own --
def _own(s):
    lib, c = _library(), s["case"]
    if c["op"] == "attend":
        decode = c["q_len"] == 1
        got = lib.custom_attention_paged_forward(
            s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["block_table"], s["seq_lens"],
            cu_seqlens_q=None if decode else s["cu_seqlens"], max_seqlen_q=c["q_len"], return_lse=c["lse"],
            window_left=c["window"] if c["window"] >= 0 else None)
        return list(got) if c["lse"] else [got]
    if c["op"] == "append":
        lib.kv_cache_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["slots"])
        return [s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]]
    lens, count = lib.kv_cache_release(s["block_table"], s["seq_lens"], s["finished"], s["free_blocks"],
                                       s["free_count"], c["block"])
    plan = lib.kv_cache_plan(s["block_table"], lens, s["new_lens"], s["free_blocks"], count, c["block"],
                             s["max_new_tokens"])
    return [plan.slots, plan.cu_seqlens, plan.seq_lens, plan.free_count, plan.placed, s["block_table"],
            s["free_blocks"]]


def run(state):
    if own:
        return _own(state)
    return {"attend": _plain_attend, "append": _plain_append, "plan": _plain_plan}[state["case"]["op"]](state)


# -------------------------------------------------------------------------- work --
def _seen(case):
    """(query, key) pairs that the mask leaves, and keys that at least one query of their request sees."""
    pairs = keys = 0
    for q, k in zip(_query_lens(case), _key_lens(case)):
        w = case["window"] if case["window"] >= 0 else k
        at = range(k - q, k)
        pairs += sum(min(p, w) + 1 for p in at)
        keys += min(k, q + w)
    return pairs, keys


def work(case):
    if case["op"] == "attend":
        pairs, keys = _seen(case)
        rows = sum(_query_lens(case))
        blocks = keys / case["block"]
        size = 2 * keys * case["heads_kv"] * case["dim"] + 8 * blocks * case["heads_kv"] + 4 * blocks
        size += 4 * rows * case["heads_q"] * case["dim"] + (4 * rows * case["heads_q"] if case["lse"] else 0)
        return {"bytes": size, "flops": 4 * pairs * case["heads_q"] * case["dim"]}
    if case["op"] == "append":
        tokens, heads = sum(_new_lens(case)), case["heads_kv"]
        # K and V: 2 bytes read and 1 written for each value, a slot for each token, and a
        # scale read and written for each block that is written.
        blocks = sum(-(-n // case["block"]) for n in _new_lens(case))
        return {"bytes": 2 * tokens * heads * case["dim"] * 3 + 8 * tokens + 2 * 8 * blocks * heads,
                "flops": 4 * tokens * heads * case["dim"]}
    held, new, done = _plan_lens(case)
    block, batch = case["block"], case["batch"]
    back = sum(-(-h // block) for h, d in zip(held, done) if d)
    taken = sum(-(-(h + n) // block) - -(-h // block) for h, n, d in zip(held, new, done) if not d)
    # Lengths in and out, the table entries and free ids that move, and one slot per token.
    return {"bytes": 4 * 7 * batch + 8 * (back + taken) + 8 * (sum(new) + 7), "flops": 0}


# ------------------------------------------------------------------------- exact --
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attend":
        return _exact_attend(case, s)
    if case["op"] == "append":
        return _exact_append(case, s)
    return None


def _exact_attend(case, s):
    """Request by request, from the definition, in float64."""
    cu, lens, heads, group = s["cu_seqlens"].tolist(), s["seq_lens"].tolist(), case["heads_kv"], 0
    group = case["heads_q"] // heads
    o = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros((case["heads_q"], s["q"].shape[0]), dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        ids = s["block_table"][b, :-(-n // case["block"])].long()
        where = torch.arange(n, device="cuda")
        rows = slice(cu[b], cu[b + 1])
        place = torch.arange(n - (cu[b + 1] - cu[b]), n, device="cuda")
        hidden = where[None, :] > place[:, None]
        if case["window"] >= 0:
            hidden |= where[None, :] < place[:, None] - case["window"]
        for h in range(heads):
            k = (s["k_cache"][ids, h].double() * s["k_scale"][ids, h].double()[:, None, None]).reshape(-1, case["dim"])[:n]
            v = (s["v_cache"][ids, h].double() * s["v_scale"][ids, h].double()[:, None, None]).reshape(-1, case["dim"])[:n]
            mine = slice(h * group, (h + 1) * group)
            x = torch.einsum("tgd,nd->gtn", s["q"][rows, mine].double(), k) * case["dim"] ** -0.5
            x[:, hidden] = -math.inf
            norm = torch.logsumexp(x, -1)
            lse[mine, rows] = norm
            o[rows, mine] = torch.einsum("gtn,nd->tgd", torch.exp(x - norm[..., None]), v)
    return [o, lse] if case["lse"] else [o]


def _exact_append(case, s):
    """Block by block, in float64: the scales, and the quotients whose rounding the codes are."""
    out, block = [], case["block"]
    slots = s["slots"].tolist()
    runs = {}
    for t, slot in enumerate(slots):
        runs.setdefault(slot // block, []).append(t)
    if len(runs) > 4000:
        return None
    codes, scales = [], []
    for x, cache, scale in ((s["k"], s["k_cache"], s["k_scale"]), (s["v"], s["v_cache"], s["v_scale"])):
        quotient, new_scale = cache.double(), scale.double()
        values = [x[tokens[0]:tokens[-1] + 1].double().transpose(0, 1) for tokens in runs.values()]  # [heads, n, D]
        top = torch.stack([v.abs().amax((1, 2)) for v in values])
        wanted = torch.full_like(top, 2.0 ** MIN_EXPONENT)
        for _ in range(250):  # the smallest power of two whose 448-fold holds every value
            wanted = torch.where(wanted * E4M3_MAX < top, wanted * 2, wanted)
        for (blk, tokens), value, want in zip(runs.items(), values, wanted):
            start = slots[tokens[0]] % block
            if start:
                want = torch.maximum(want, new_scale[blk])
                quotient[blk, :, :start] *= (new_scale[blk] / want)[:, None, None]
            quotient[blk, :, start:start + len(tokens)] = value / want[:, None, None]
            new_scale[blk] = want
        codes.append(quotient)
        scales.append(new_scale)
    return codes + scales
