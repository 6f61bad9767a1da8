"""Layouts in which outputs stand beside inputs in one buffer, which the checks for shared memory have to let pass (GPU only):
each gives the bits of the same call on tensors of their own."""
import pytest
import torch

from halo_flash_b200 import ops
from tests.test_gpu_attention import BF16, DEV, _gen, _i32, _randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hq,hk,d,t", [(8, 2, 128, 700), (4, 4, 64, 1), (16, 1, 256, 90)])
def test_rows_of_one_projection(hq, hk, d, t):
    """q, k and v side by side in the rows of one buffer; out in place of q, or behind v, or in the heads' order."""
    g, cu = _gen(41), _i32([0, t // 3, t])
    for extra in (0, hq * d):
        buf = _randn(g, t, (hq + 2 * hk) * d + extra, dtype=BF16)
        q, k, v = (x.view(t, -1, d) for x in buf[:, :(hq + 2 * hk) * d].split([hq * d, hk * d, hk * d], 1))
        want = ops.attention_packed(*(x.contiguous() for x in (q, k, v)), cu, torch.empty(t, hq, d, dtype=BF16, device=DEV))
        by_head = torch.empty(hq, t, d, dtype=BF16, device=DEV).transpose(0, 1)
        assert torch.equal(ops.attention_packed(q, k, v, cu, by_head), want)
        if extra:
            assert torch.equal(ops.attention_packed(q, k, v, cu, buf[:, -hq * d:].view(t, hq, d)), want)
        k0, v0 = k.clone(), v.clone()
        assert torch.equal(ops.attention_packed(q, k, v, cu, q), want)
        assert torch.equal(k, k0) and torch.equal(v, v0)


def test_heads_of_one_projection():
    """[q and k and v heads][tokens][d]: heads as the outer axis of one buffer."""
    g, hq, hk, d, t = _gen(42), 8, 2, 64, 333
    buf = _randn(g, hq + 2 * hk, t, d, dtype=BF16).transpose(0, 1)
    q, k, v = buf.split([hq, hk, hk], 1)
    cu = _i32([0, 300, t])
    want = ops.attention_packed(*(x.contiguous() for x in (q, k, v)), cu, torch.empty(t, hq, d, dtype=BF16, device=DEV))
    assert torch.equal(ops.attention_packed(q, k, v, cu, q), want)


def test_out_between_the_pages_of_a_cache():
    """An arena whose pages hold K, V and a strip of something else, in which out lies."""
    g, hq, hk, d, page, pages = _gen(43), 16, 2, 128, 16, 9
    arena = _randn(g, pages, 3, page, hk, d, dtype=BF16)
    kc, vc, strip = arena.unbind(1)
    out = strip.flatten(1)[:, :hq * d].view(pages, hq, d)
    q, table, cu = _randn(g, pages, hq, d, dtype=BF16), _i32([[3, 1, 4, 8]]), _i32([0, pages])
    want = ops.attention_paged(q, kc.contiguous(), vc.contiguous(), table, _i32([60]), cu, torch.empty_like(q))
    before = arena[:, :2].clone()
    assert torch.equal(ops.attention_paged(q, kc, vc, table, _i32([60]), cu, out), want)
    assert torch.equal(arena[:, :2], before)


@pytest.mark.parametrize("make", [
    lambda p, n, h, d: torch.zeros(p, 2, n, h, d, dtype=BF16, device=DEV).unbind(1), lambda p, n, h, d: torch.zeros(2, p, n, h, d, dtype=BF16, device=DEV).unbind(0),
    lambda p, n, h, d: torch.zeros(p, n, 2, h, d, dtype=BF16, device=DEV).unbind(2), lambda p, n, h, d: torch.zeros(p, n, h, 2, d, dtype=BF16, device=DEV).unbind(3),
    lambda p, n, h, d: torch.zeros(p, n, h, 2 * d, dtype=BF16, device=DEV).split(d, 3),
    lambda p, n, h, d: [x.permute(1, 2, 0, 3) for x in torch.zeros(2, h, p, n, d, dtype=BF16, device=DEV).unbind(0)],
    lambda p, n, h, d: [x.permute(1, 0, 2, 3) for x in torch.zeros(n, 2, p, h, d, dtype=BF16, device=DEV).unbind(1)]])
def test_caches_in_one_buffer(make):
    g, pages, page, heads, d, t = _gen(44), 7, 16, 2, 64, 50
    kc, vc = make(pages, page, heads, d)
    k, v = (_randn(g, t, heads, d, dtype=BF16) for _ in range(2))
    slot = torch.randperm(pages * page, generator=g, device=DEV)[:t]
    ops.paged_store(k, v, kc, vc, slot)
    for rows, cache in ((k, kc), (v, vc)):
        assert torch.equal(cache[slot // page, slot % page], rows) and int((cache != 0).any(-1).sum()) == t * heads


def test_rows_moved_within_a_cache():
    """A source that lies in the cache: rows of pages 0 and 1 stored into page 5."""
    g, page, heads, d = _gen(45), 16, 2, 64
    kc, vc = (_randn(g, 6, page, heads, d, dtype=BF16) for _ in range(2))
    want_k, want_v = kc.clone(), vc.clone()
    want_k[5], want_v[5] = kc.view(-1, heads, d)[8:24], vc.view(-1, heads, d)[8:24]
    ops.paged_store(kc.view(-1, heads, d)[8:24], vc.view(-1, heads, d)[8:24], kc, vc, torch.arange(5 * page, 6 * page, device=DEV))
    assert torch.equal(kc, want_k) and torch.equal(vc, want_v)


def test_plan_in_one_buffer():
    """Inputs and outputs as neighbouring slices of one buffer, the table as columns of it."""
    buf = torch.full((40, 10), 9, dtype=torch.int32, device=DEV)
    table, flat = buf[:3, 2:6], buf.view(-1)
    past, fresh, free, cu, kv_len, status, pos = flat[100:103], flat[103:106], flat[106:110], flat[110:114], flat[114:117], flat[117:120], flat[120:126]
    past.copy_(_i32([0, 7, 8])), fresh.copy_(_i32([1, 2, 3])), free.copy_(_i32([11, 12, 13, 14]))
    slot = torch.empty(6, dtype=torch.int64, device=DEV)
    ops.paged_plan(table, past, fresh, free, 8, slot, pos=pos, cu=cu, kv_len=kv_len, status=status)
    assert slot.tolist() == [88, 79, 96, 104, 105, 106] and pos.tolist() == [0, 7, 8, 8, 9, 10]
    assert cu.tolist() == [0, 1, 3, 6] and kv_len.tolist() == [1, 9, 11] and status.tolist() == [3, 0, 6]
    assert table.tolist() == [[11, 9, 9, 9], [9, 12, 9, 9], [9, 13, 9, 9]] and buf[:, :2].flatten()[:6].eq(9).all()
