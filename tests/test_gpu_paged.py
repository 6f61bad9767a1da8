"""The plan of a paged cache and the store into it, and a run of them with the attention that reads it (GPU only).
Whole numbers and copies: everything is compared for equality."""
import random

import pytest
import torch

from halo_flash_b200 import ops
from tests.test_gpu_attention import BF16, DEV, F16, _gen, _i32, _prefix, _randn, check, exact_rows

pytestmark = pytest.mark.gpu


def plan_on_host(table, past, fresh, free, page, tokens):
    """The definition, request by request."""
    table = [list(r) for r in table]
    cols, at, full = len(table[0]) if table else 0, 0, False
    slot, pos, kv_len, refused = [], [], [], 0
    for r, (p, f) in enumerate(zip(past, fresh)):
        held, want = -(-p // page), -(-(p + f) // page)
        need = want - held
        ok = want <= cols
        if ok and need:
            full = full or at + need > len(free)
            ok = not full
        if ok:
            table[r][held:want] = free[at:at + need]
            at += need
        refused += not ok
        kv_len.append(p + f if ok else p)
        for i in range(p, p + f):
            slot.append(table[r][i // page] * page + i % page if ok else -1)
            pos.append(i)
    total = len(slot)
    slot, pos = (slot + [-1] * tokens)[:tokens], (pos + [0] * tokens)[:tokens]
    return table, slot, pos, _prefix(fresh), kv_len, [at, refused, total]


def run_plan(table, past, fresh, free, page, tokens):
    t = torch.tensor(table, dtype=torch.int32, device=DEV)
    new = lambda n: torch.full((n,), 77, dtype=torch.int32, device=DEV)  # noqa: E731
    slot, pos, cu, kv_len, status = torch.full((tokens,), 77, dtype=torch.int64, device=DEV), new(tokens), new(len(past) + 1), new(len(past)), new(3)
    ops.paged_plan(t, _i32(past), _i32(fresh), _i32(free), page, slot, pos=pos, cu=cu, kv_len=kv_len, status=status)
    return [x.tolist() for x in (t, slot, pos, cu, kv_len, status)]


@pytest.mark.parametrize("batch,page,cols,most,free,slack", [
    (1, 16, 4, 30, 10, 0), (8, 64, 40, 1000, 200, 3), (33, 8, 30, 100, 600, 0), (700, 16, 64, 300, 40000, 50), (3000, 256, 8, 600, 9000, 0), (16384, 16, 3, 20, 30000, 7),
    (20, 16, 8, 80, 30, 5),      # the free list ends
    (20, 16, 3, 40, 300, -40),   # some need more pages than a table row has; fewer slots than tokens
    (5, 32, 4, 50, 0, 0),        # no free page at all
])
def test_plan(batch, page, cols, most, free, slack):
    rng = random.Random(batch * page)
    past = [rng.randint(0, min(most, cols * page)) for _ in range(batch)]
    fresh = [rng.choice([0, 1, 1, rng.randint(0, most)]) for _ in range(batch)]
    if free != 30 and cols > 4:
        fresh = [min(f, cols * page - p) for p, f in zip(past, fresh)]
    ids = rng.sample(range(1 << 20), batch * cols + free)
    table = [ids[r * cols:(r + 1) * cols] for r in range(batch)]
    tokens = max(0, sum(fresh) + slack)
    assert run_plan(table, past, fresh, ids[batch * cols:], page, tokens) == list(plan_on_host(table, past, fresh, ids[batch * cols:], page, tokens))


def test_plan_takes_views_and_optional_outputs():
    wide = torch.full((3, 10), -5, dtype=torch.int32, device=DEV)
    table = wide[:, 2:6]
    slot = torch.empty(6, dtype=torch.int64, device=DEV)
    ops.paged_plan(table, _i32([0, 7, 8]), _i32([1, 2, 3]), _i32([11, 12, 13, 14]), 8, slot)
    # request 1 holds page -5 (whatever stood there) for its token 7
    assert slot.tolist() == [88, -5 * 8 + 7, 96, 104, 105, 106]
    assert wide[:, :2].eq(-5).all() and wide[:, 6:].eq(-5).all()
    assert table.tolist() == [[11, -5, -5, -5], [-5, 12, -5, -5], [-5, 13, -5, -5]]


@pytest.mark.parametrize("src,dst", [(torch.float32, torch.float32), (torch.float32, F16), (torch.float32, BF16), (F16, F16), (F16, BF16), (BF16, BF16), (BF16, F16)])
@pytest.mark.parametrize("heads,d,page", [(2, 256, 64), (1, 64, 8), (3, 20, 16), (4, 1, 32)])
def test_store(src, dst, heads, d, page):
    g, tokens, pages = _gen(d), 301, 45
    k, v = _randn(g, tokens, heads, d, dtype=src), _randn(g, tokens, heads, d, dtype=src)
    slot = torch.randperm(pages * page, generator=g, device=DEV)[:tokens]
    slot[7] = -1
    slot[9] = pages * page  # outside: skipped
    slot[10] = -(1 << 40)
    kc, vc = (torch.full((pages, page, heads, d), 3.0, dtype=dst, device=DEV) for _ in range(2))
    want_k, want_v = kc.clone(), vc.clone()
    keep = (slot >= 0) & (slot < pages * page)
    for rows, cache in ((k, want_k), (v, want_v)):
        cache.view(-1, heads, d)[slot[keep]] = rows[keep].to(dst)
    ops.paged_store(k, v, kc, vc, slot)
    assert torch.equal(kc, want_k) and torch.equal(vc, want_v)


def test_store_views():
    """Rows out of one projection buffer, caches as [pages, heads, rows, d] and as halves of one buffer."""
    g, t, heads, d, page = _gen(2), 50, 2, 64, 16
    buf = _randn(g, t, 6 * d, dtype=BF16)
    k, v = buf[:, 2 * d:4 * d].view(t, heads, d), buf[:, 4 * d:].view(t, heads, d)
    slot = torch.randperm(8 * page, generator=g, device=DEV)[:t]
    for make in (lambda: [torch.zeros(8, heads, page, d, dtype=BF16, device=DEV).transpose(1, 2) for _ in range(2)],
                 lambda: list(torch.zeros(8, 2, page, heads, d, dtype=BF16, device=DEV).unbind(1))):
        kc, vc = make()
        ops.paged_store(k, v, kc, vc, slot)
        for rows, cache in ((k, kc), (v, vc)):
            assert torch.equal(cache[slot // page, slot % page], rows) and int((cache != 0).any(-1).sum()) == t * heads


def test_store_past_32_bit_offsets():
    """A cache of more than 2^32 elements: the last page is written and read where it is."""
    pages, page, heads, d = (1 << 32) // (64 * 2 * 256) + 3, 64, 2, 256
    kc = torch.zeros(pages, page, heads, d, dtype=BF16, device=DEV)
    vc = torch.zeros_like(kc)
    g = _gen(3)
    k, v = _randn(g, page + 5, heads, d, dtype=BF16), _randn(g, page + 5, heads, d, dtype=BF16)
    table = _i32([[pages - 1, pages - 2]])
    slot = torch.cat([torch.arange(page) + (pages - 1) * page, torch.arange(5) + (pages - 2) * page]).to(DEV)
    ops.paged_store(k, v, kc, vc, slot)
    assert torch.equal(kc[pages - 1], k[:page]) and torch.equal(vc[pages - 2, :5], v[page:])
    q = _randn(g, 1, 16, d, dtype=BF16)
    out = torch.empty_like(q)
    ops.attention_paged(q, kc, vc, table, _i32([page + 5]), _i32([0, 1]), out)
    check(out, None, exact_rows(q, k, v, True, d ** -0.5), BF16, page + 5, 7.0, "far pages")


def test_a_conversation_step_by_step():
    """Three sessions: prompts in chunks, then decode steps, through plan, store and attention, with the lengths living
    on the GPU from step to step; every step's outputs against each session's whole history in 64 bits."""
    g, hq, hk, d, page, pages = _gen(4), 16, 2, 256, 16, 64
    kc, vc = (torch.full((pages, page, hk, d), float("nan"), dtype=BF16, device=DEV) for _ in range(2))
    table = torch.full((3, 24), -1, dtype=torch.int32, device=DEV)
    free = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    past, taken = _i32([0, 0, 0]), 0
    seen = [[], [], []]
    for fresh in ([70, 3, 0], [50, 1, 129], [1, 1, 1], [1, 0, 1], [2, 60, 1]):
        t = sum(fresh)
        slot, cu, kv_len, status = torch.empty(t + 4, dtype=torch.int64, device=DEV), _i32([0] * 4), _i32([0] * 3), _i32([0] * 3)
        ops.paged_plan(table, past, _i32(fresh), free[taken:], page, slot, cu=cu, kv_len=kv_len, status=status)
        q, k, v = (_randn(g, t + 4, h, d, dtype=BF16) for h in (hq, hk, hk))
        ops.paged_store(k, v, kc, vc, slot)
        out = torch.full_like(q, 9.0)
        ops.attention_paged(q, kc, vc, table, kv_len, cu, out)
        assert (out[t:] == 9.0).all()
        got, refused, total = status.tolist()
        assert refused == 0 and total == t
        taken += got
        for b, (a, e) in enumerate(zip(cu.tolist()[:-1], cu.tolist()[1:])):
            seen[b].append((k[a:e], v[a:e]))
            ks, vs = (torch.cat([s[x] for s in seen[b]]) for x in (0, 1))
            check(out[a:e], None, exact_rows(q[a:e], ks, vs, True, d ** -0.5), BF16, ks.shape[0], 7.0, f"session {b} after {fresh}")
        past = kv_len


def test_a_layer_step_with_rotation():
    """plan -> rotation table at the planned positions -> norm + RoPE of Q and K -> store -> attention, on one stream
    without a look at the device in between; the attention of the rotated rows against 64 bits."""
    g, hq, hk, d, page = _gen(5), 16, 2, 256, 64
    past, fresh = [300, 0, 77], [1, 40, 1]
    t, pages = sum(fresh), 24
    table = torch.full((3, 8), -1, dtype=torch.int32, device=DEV)
    ids = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    at = 0
    for r, p in enumerate(past):
        n = -(-p // page)
        table[r, :n] = ids[at:at + n]
        at += n
    kc, vc = (_randn(g, pages, page, hk, d, dtype=BF16) for _ in range(2))
    slot, pos, cu, kv_len = torch.empty(t, dtype=torch.int64, device=DEV), _i32([0] * t), _i32([0] * 4), _i32([0] * 3)
    ops.paged_plan(table, _i32(past), _i32(fresh), ids[at:], page, slot, pos=pos, cu=cu, kv_len=kv_len)
    q, k, v = (_randn(g, t, h, d, dtype=BF16) for h in (hq, hk, hk))
    rot = torch.empty(t, 64, device=DEV)
    ops.rope_table(rot, 64, 1e7, params=pos, pstride=1)
    w = torch.zeros(d, device=DEV)
    before = k.clone()
    ops.norm_rope_qk_table(q, k, w, w, 1e-6, 64, rot)
    ops.paged_store(k, v, kc, vc, slot)
    out = torch.empty_like(q)
    ops.attention_paged(q, kc, vc, table, kv_len, cu, out)
    assert pos.tolist() == [300] + list(range(40)) + [77] and not torch.equal(before, k)
    for b, (p, n) in enumerate(zip(past, fresh)):
        a = sum(fresh[:b])
        ks, vs = (c[table[b].long()].flatten(0, 1)[:p + n] for c in (kc, vc))
        assert torch.equal(ks[p:], k[a:a + n]) and torch.equal(vs[p:], v[a:a + n])
        check(out[a:a + n], None, exact_rows(q[a:a + n], ks, vs, True, d ** -0.5), BF16, p + n, 7.0, f"request {b}")
