"""What the attention side of a layer is measured on: the plan of a paged K/V cache, the store into it, attention
over packed prompts, and attention of new tokens over the pages.

Each case names one operator (`op`) and its sizes. run() computes it in a plain form out of elementary torch
operations in 32 bits, or, where `own` is true, through halo_flash_b200.ops. exact() computes it again in 64 bits.

Shapes: the full-size layer (16 query heads, 2 key/value heads, head size 256), the tiny layer (4, 2, 64), prompts
of 4096 tokens and their chunks, decode of 1 to 8 sessions at positions up to 262144; the other head layouts, head
and page sizes are generic.
"""
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    full = {"q_heads": 16, "kv_heads": 2, "dim": 256}
    tiny = {"q_heads": 4, "kv_heads": 2, "dim": 64}
    return [
        # the tiny layer's few tokens, three short prompts: nothing but latency
        {"name": "packed_tiny", "op": "packed", "dtype": "fp16", "batch": 3, "tokens": 32, "mix": 1, **tiny},
        # a prefill chunk that is one whole prompt
        {"name": "packed_4096", "op": "packed", "dtype": "bf16", "batch": 1, "tokens": 4096, "mix": 0, **full},
        # nine prompts of any length packed into one prefill batch, another head layout
        {"name": "packed_ragged", "op": "packed", "dtype": "fp16", "batch": 9, "tokens": 5003, "mix": 3,
         "q_heads": 12, "kv_heads": 4, "dim": 128},
        # a long document as one prompt
        {"name": "packed_16384", "op": "packed", "dtype": "bf16", "batch": 1, "tokens": 16384, "mix": 0, **full},
        # one session's decode step early in its conversation
        {"name": "decode_1", "op": "paged", "dtype": "bf16", "batch": 1, "tokens": 1, "past": 1500, "even": True,
         "page": 64, "mix": 5, **full},
        # eight sessions' decode step, positions anywhere up to the longest context
        {"name": "decode_8_long", "op": "paged", "dtype": "bf16", "batch": 8, "tokens": 8, "past": 262144, "even": False,
         "page": 64, "mix": 6, **full},
        # one session's 2048-token prefill chunk behind 30000 cached tokens
        {"name": "chunk_2048", "op": "paged", "dtype": "bf16", "batch": 1, "tokens": 2048, "past": 30000, "even": True,
         "page": 64, "mix": 7, **full},
        # a serving step: decoding sessions beside short chunks, small pages, another head layout
        {"name": "mixed_step", "op": "paged", "dtype": "fp16", "batch": 24, "tokens": 700, "past": 6000, "even": False,
         "page": 16, "mix": 8, "q_heads": 24, "kv_heads": 8, "dim": 128},
        # the plan of a decode step of eight sessions, and of a large serving step with prompt chunks
        {"name": "plan_decode_8", "op": "plan", "batch": 8, "tokens": 8, "past": 262144, "even": False, "page": 64, "mix": 9},
        {"name": "plan_1024", "op": "plan", "batch": 1024, "tokens": 65536, "past": 8192, "even": False, "page": 16, "mix": 10},
        # the store of a decode step, and of a long prefill
        {"name": "store_decode_8", "op": "store", "dtype": "bf16", "cache": "bf16", "batch": 8, "tokens": 8, "past": 5000,
         "even": False, "page": 64, "mix": 11, "kv_heads": 2, "dim": 256},
        {"name": "store_65536", "op": "store", "dtype": "bf16", "cache": "bf16", "batch": 5, "tokens": 65536, "past": 1000,
         "even": False, "page": 64, "mix": 12, "kv_heads": 2, "dim": 256},
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return min(high, max(low, round(low * (high / low) ** rng.random())))


def draw(rng):
    op = rng.choice(["packed", "packed", "paged", "paged", "paged", "plan", "store"])
    case = {"op": op, "mix": rng.randrange(1, 1 << 20)}
    if op == "plan":
        batch = _spread(rng, 1, 1024)
        return {**case, "batch": batch, "tokens": _spread(rng, batch, 65536), "past": _spread(rng, 16, 32768),
                "even": rng.random() < 0.2, "page": rng.choice([16, 32, 64, 128])}
    if op == "store":
        return {**case, "dtype": rng.choice(["bf16", "fp16", "fp32"]), "cache": rng.choice(["bf16", "fp16"]),
                "batch": rng.randint(1, 16), "tokens": _spread(rng, 16, 32768), "past": _spread(rng, 16, 8192), "even": False,
                "page": rng.choice([16, 32, 64, 128]), "kv_heads": rng.randint(1, 8), "dim": rng.choice([64, 96, 128, 256])}
    kv_heads = rng.choice([1, 2, 2, 4, 8])
    case |= {"dtype": rng.choice(["bf16", "fp16"]), "kv_heads": kv_heads,
             "q_heads": kv_heads * rng.choice([1, 2, 3, 4, 6, 7, 8]), "dim": rng.choice([64, 96, 128, 256, 256])}
    batch = _spread(rng, 1, 32)
    pairs = 16 * 4096 * 4096 // (batch * case["q_heads"])  # query-key pairs of one sequence and head that are let through
    if op == "packed":
        longest = max(1, int(pairs ** 0.5))
        return {**case, "batch": batch, "tokens": _spread(rng, batch, max(batch, min(6000, longest)))}
    case |= {"batch": batch, "page": rng.choice([16, 32, 64, 128]), "even": rng.random() < 0.3}
    tokens = batch if rng.random() < 0.5 else _spread(rng, batch, max(batch, min(2048, pairs // 64)))
    past = _spread(rng, 16, max(64, min(65536 // max(1, kv_heads // 2) // max(1, batch // 8), pairs // tokens)))
    return {**case, "tokens": tokens, "past": past}


def _lengths(case):
    """(past, new) tokens of each sequence: part of the case, made from its own numbers. Of the new tokens each
    sequence has one, and what is left falls to some of them."""
    rng = random.Random(case["mix"])
    batch, tokens = case["batch"], case["tokens"]
    weights = [rng.expovariate(1.0) if rng.random() < 0.6 else 0.0 for _ in range(batch)]
    if not any(weights):
        weights[rng.randrange(batch)] = 1.0
    rest, total = tokens - batch, sum(weights)
    new = [1 + int(rest * w / total) for w in weights]
    new[max(range(batch), key=weights.__getitem__)] += tokens - sum(new)
    past = [0] * batch
    if "past" in case:
        past = [case["past"] if case["even"] else rng.randint(0, case["past"]) for _ in range(batch)]
    return past, new


def _randn(gen, *shape, dtype):
    return torch.randn(*shape, generator=gen, device=DEV).to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _prefix(values):
    out = [0]
    for v in values:
        out.append(out[-1] + v)
    return out


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    op, (past, new) = case["op"], _lengths(case)
    state = {"case": case, "tokens": sum(new), "cu": _ints(_prefix(new))}
    if op != "packed":
        page = case["page"]
        held = [-(-p // page) for p in past]  # pages of the tokens that are already there
        want = [-(-(p + n) // page) for p, n in zip(past, new)]
        columns, extra = max(want), 8
        pages = sum(want) + extra
        order = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32)
    if op == "plan":
        table = torch.full((case["batch"], columns), -1, dtype=torch.int32, device=DEV)
        first = torch.tensor(_prefix(held)[:-1], device=DEV)
        column = torch.arange(columns, device=DEV)
        mine = column[None] < torch.tensor(held, device=DEV)[:, None]
        at = (first[:, None] + column[None]).clamp(max=pages - 1)
        return {**state, "table": torch.where(mine, order[at], table), "past": _ints(past), "new": _ints(new),
                "free": order[sum(held):].contiguous()}
    dtype = DTYPES[case["dtype"]]
    kv_heads, dim = case["kv_heads"], case["dim"]
    if op == "packed":
        return {**state, "q": _randn(gen, sum(new), case["q_heads"], dim, dtype=dtype),
                "k": _randn(gen, sum(new), kv_heads, dim, dtype=dtype), "v": _randn(gen, sum(new), kv_heads, dim, dtype=dtype)}
    first = torch.tensor(_prefix(want)[:-1], device=DEV)
    table = order[(first[:, None] + torch.arange(columns, device=DEV)[None]).clamp(max=pages - 1)].contiguous()
    state |= {"table": table, "kv_len": _ints([p + n for p, n in zip(past, new)])}
    if op == "paged":
        return {**state, "q": _randn(gen, sum(new), case["q_heads"], dim, dtype=dtype),
                "k_cache": _randn(gen, pages, page, kv_heads, dim, dtype=dtype),
                "v_cache": _randn(gen, pages, page, kv_heads, dim, dtype=dtype)}
    cache = DTYPES[case["cache"]]
    row = torch.repeat_interleave(torch.arange(case["batch"], device=DEV), torch.tensor(new, device=DEV))
    place = torch.arange(sum(new), device=DEV) - state["cu"].long()[row] + torch.tensor(past, device=DEV)[row]
    state |= {"slot": table.long()[row, place // page] * page + place % page}
    return {**state, "k": _randn(gen, sum(new), kv_heads, dim, dtype=dtype), "v": _randn(gen, sum(new), kv_heads, dim, dtype=dtype),
            "k_cache": torch.zeros(pages, page, kv_heads, dim, dtype=cache, device=DEV),
            "v_cache": torch.zeros(pages, page, kv_heads, dim, dtype=cache, device=DEV)}


# ---- the plain forms ---------------------------------------------------------------------------------------------


def _attend(q, k, v, visible, scale):
    """softmax(q k^T scale) v over the visible keys, and the logarithm of the softmax's denominator, of padded
    batches q [B, N, Hq, D], k and v [B, L, Hk, D] with visible [B, N, L]; a row that sees nothing gives zeros."""
    batch, rows, q_heads, dim = q.shape
    length, kv_heads = k.shape[1:3]
    group = q_heads // kv_heads
    q = q.float().view(batch, rows, kv_heads, group, dim).permute(0, 2, 3, 1, 4).reshape(batch, kv_heads, group * rows, dim)
    s = (q * scale) @ k.float().permute(0, 2, 3, 1)
    s = s.view(batch, kv_heads, group, rows, length).masked_fill_(~visible[:, None, None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
    p = s.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = p.view(batch, kv_heads, group * rows, length) @ v.float().permute(0, 2, 1, 3)
    o = o.view(batch, kv_heads, group, rows, dim) / torch.where(total == 0, torch.ones_like(total), total)
    lse = (total.log() + top)[..., 0]
    return o.permute(0, 3, 1, 2, 4).reshape(batch, rows, q_heads, dim), lse.permute(0, 3, 1, 2).reshape(batch, rows, q_heads)


def _padded(state):
    """The packed tokens' places in a padded batch: index [B, N], which of them there are, and each token's (b, n)."""
    past, new = _lengths(state["case"])
    longest, cu = max(new), state["cu"].long()
    at = torch.arange(longest, device=DEV)
    there = at[None] < (cu[1:] - cu[:-1])[:, None]
    index = (cu[:-1, None] + at[None]).clamp(max=state["tokens"] - 1)
    token = torch.arange(state["tokens"], device=DEV)
    b = torch.searchsorted(cu[1:], token, right=True)
    return index, there, b, token - cu[b]


def _plain_packed(state):
    q, k, v = state["q"], state["k"], state["v"]
    index, there, b, n = _padded(state)
    at = torch.arange(index.shape[1], device=DEV)
    visible = there[:, None, :] & (at[None, None, :] <= at[None, :, None])
    o, lse = _attend(q[index], k[index], v[index], visible, q.shape[-1] ** -0.5)
    return {"out": o[b, n].to(q.dtype), "lse": lse[b, n]}


def _plain_paged(state):
    q, k_cache, v_cache, kv_len = state["q"], state["k_cache"], state["v_cache"], state["kv_len"].long()
    past, new = _lengths(state["case"])
    page, length = state["case"]["page"], max(p + n for p, n in zip(past, new))
    index, there, b, n = _padded(state)
    key = torch.arange(length, device=DEV)
    block = state["table"].long()[:, key // page]
    here = key[None] < kv_len[:, None]
    block = torch.where(here, block, torch.zeros_like(block))
    k, v = k_cache[block, key % page], v_cache[block, key % page]
    count = (state["cu"][1:] - state["cu"][:-1]).long()
    last = (kv_len - count)[:, None] + torch.arange(index.shape[1], device=DEV)[None]
    visible = here[:, None, :] & (key[None, None, :] <= last[:, :, None])
    o, lse = _attend(q[index], k, v, visible, q.shape[-1] ** -0.5)
    return {"out": o[b, n].to(q.dtype), "lse": lse[b, n]}


def _plain_plan(state):
    page, table = state["case"]["page"], state["table"]
    past, new, free = state["past"].long(), state["new"].long(), state["free"]
    zero = torch.zeros(1, dtype=torch.int64, device=DEV)
    held, want = (past + page - 1) // page, (past + new + page - 1) // page
    first = torch.cat([zero, (want - held).cumsum(0)])
    cu = torch.cat([zero, new.cumsum(0)])
    column = torch.arange(table.shape[1], device=DEV)[None]
    taken = (column >= held[:, None]) & (column < want[:, None])
    at = (first[:-1, None] + column - held[:, None]).clamp(0, free.numel() - 1)
    table = torch.where(taken, free[at], table)
    token = torch.arange(state["tokens"], device=DEV)
    row = torch.searchsorted(cu[1:], token, right=True)
    pos = token - cu[row] + past[row]
    slot = table.long()[row, pos // page] * page + pos % page
    status = torch.cat([first[-1:], zero, cu[-1:]])
    return {"table": table, "slot": slot, "pos": pos.int(), "cu": cu.int(), "kv_len": (past + new).int(), "status": status.int()}


def _plain_store(state):
    k_cache, v_cache, slot = state["k_cache"], state["v_cache"], state["slot"]
    for rows, cache in ((state["k"], k_cache), (state["v"], v_cache)):
        cache.view(-1, *cache.shape[2:])[slot] = rows.to(cache.dtype)
    return {"k_cache": k_cache, "v_cache": v_cache}


# ---- the framework's operators -----------------------------------------------------------------------------------


def _own_packed(state):
    from halo_flash_b200 import ops
    q = state["q"]
    out, lse = torch.empty_like(q), torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
    ops.attention_packed(q, state["k"], state["v"], state["cu"], out, lse=lse)
    return {"out": out, "lse": lse}


def _own_paged(state):
    from halo_flash_b200 import ops
    q = state["q"]
    out, lse = torch.empty_like(q), torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
    ops.attention_paged(q, state["k_cache"], state["v_cache"], state["table"], state["kv_len"], state["cu"], out, lse=lse)
    return {"out": out, "lse": lse}


def _own_plan(state):
    from halo_flash_b200 import ops
    table, batch = state["table"], state["case"]["batch"]
    new = lambda n, dtype=torch.int32: torch.empty(n, dtype=dtype, device=table.device)  # noqa: E731
    slot, pos, cu, kv_len, status = new(state["tokens"], torch.int64), new(state["tokens"]), new(batch + 1), new(batch), new(3)
    ops.paged_plan(table, state["past"], state["new"], state["free"], state["case"]["page"], slot, pos=pos, cu=cu, kv_len=kv_len,
                   status=status)
    return {"table": table, "slot": slot, "pos": pos, "cu": cu, "kv_len": kv_len, "status": status}


def _own_store(state):
    from halo_flash_b200 import ops
    ops.paged_store(state["k"], state["v"], state["k_cache"], state["v_cache"], state["slot"])
    return {"k_cache": state["k_cache"], "v_cache": state["v_cache"]}


PLAIN = {"packed": _plain_packed, "paged": _plain_paged, "plan": _plain_plan, "store": _plain_store}
OWN = {"packed": _own_packed, "paged": _own_paged, "plan": _own_plan, "store": _own_store}


def run(state):
    return (OWN if own else PLAIN)[state["case"]["op"]](state)


# ---- what a pass cannot do without, and its values in 64 bits ----------------------------------------------------


def work(case):
    past, new = _lengths(case)
    tokens, op = sum(new), case["op"]
    if op == "plan":
        pages = sum(-(-(p + n) // case["page"]) - -(-p // case["page"]) for p, n in zip(past, new))
        # lengths in, prefix and lengths out; a free page in and a table entry out for each new page; the page that a
        # sequence had begun; a slot and a position out for each token
        return {"bytes": 16 * case["batch"] + 8 * pages + 4 * case["batch"] + 12 * tokens, "flops": 0}
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    row = case["kv_heads"] * case["dim"]
    if op == "store":
        return {"bytes": tokens * (8 + 2 * row * (size[case["dtype"]] + size[case["cache"]])), "flops": 0}
    keys = sum(p + n for p, n in zip(past, new))
    seen = sum(n * p + n * (n + 1) // 2 for p, n in zip(past, new))
    return {"bytes": 2 * keys * row * 2 + tokens * case["q_heads"] * (2 * case["dim"] * 2 + 4),
            "flops": 4 * seen * case["q_heads"] * case["dim"]}


def _exact_rows(q, k, v, offset):
    """One sequence in 64 bits, head by head: row i sees the keys up to offset + i."""
    rows, q_heads, dim = q.shape
    group = q_heads // k.shape[1]
    out = torch.empty(rows, q_heads, dim, dtype=torch.float64, device=q.device)
    lse = torch.empty(rows, q_heads, dtype=torch.float64, device=q.device)
    step = max(1, (1 << 28) // max(1, k.shape[0]))
    for h in range(q_heads):
        kh, vh = k[:, h // group].double(), v[:, h // group].double()
        for a in range(0, rows, step):
            b = min(rows, a + step)
            logits = torch.einsum("nd,ld->nl", q[a:b, h].double(), kh) / dim ** 0.5
            limit = torch.arange(a, b, device=q.device) + offset
            logits[torch.arange(k.shape[0], device=q.device)[None] > limit[:, None]] = float("-inf")
            lse[a:b, h] = torch.logsumexp(logits, 1)
            out[a:b, h] = torch.einsum("nl,ld->nd", (logits - lse[a:b, h, None]).exp(), vh)
    return out, lse


def exact(case, seed):
    op, (past, new) = case["op"], _lengths(case)
    if op == "plan":
        return None  # whole numbers: nothing is rounded
    state = prepare(case, seed)
    if op == "store":
        page, found = case["page"], {}
        for name in ("k", "v"):
            flat = torch.zeros(state[name + "_cache"].numel() // (case["kv_heads"] * case["dim"]), case["kv_heads"], case["dim"],
                               dtype=torch.float64, device=DEV)
            flat.index_copy_(0, state["slot"], state[name].double())
            found[name + "_cache"] = flat.view(-1, page, case["kv_heads"], case["dim"])
        return found
    outs, lses = [], []
    for b, (p, n) in enumerate(zip(past, new)):
        begin = sum(new[:b])
        q = state["q"][begin:begin + n]
        if op == "packed":
            k, v = state["k"][begin:begin + n], state["v"][begin:begin + n]
        else:
            pages = state["table"][b, : -(-(p + n) // case["page"])].long()
            k, v = (state[c][pages].flatten(0, 1)[: p + n] for c in ("k_cache", "v_cache"))
        o, lse = _exact_rows(q, k, v, p)
        outs.append(o)
        lses.append(lse)
    return {"out": torch.cat(outs), "lse": torch.cat(lses)}
