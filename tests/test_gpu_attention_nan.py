"""NaN in what a query attends to is in its result, whether its job is computed whole or cut into pieces (GPU only).

A NaN score makes the softmax's denominator NaN: out and lse of that query are NaN. A NaN in V alone leaves lse as it is.
That holds for keys whose weight underflows too (0 * NaN is NaN). Queries that do not see the NaN keep their values,
against 64 bits with the tolerance of test_gpu_attention.py.
"""
import pytest
import torch

from halo_flash_b200 import ops
from tests.test_gpu_attention import BF16, DEV, F16, _gen, _i32, _prefix, _randn, check, exact_rows

pytestmark = pytest.mark.gpu

NAN = float("nan")


def _cache(g, lens, hk, d, page, dtype):
    """Caches, a table and each sequence's rows as views of page runs (sequence b owns neighbouring pages)."""
    want = [-(-n // page) for n in lens]
    at = _prefix(want)
    kc, vc = (_randn(g, at[-1], page, hk, d, dtype=dtype) for _ in range(2))
    table = torch.zeros(len(lens), max(want), dtype=torch.int32, device=DEV)
    for b, n in enumerate(want):
        table[b, :n] = torch.arange(at[b], at[b + 1], dtype=torch.int32, device=DEV)
    rows = [(kc[at[b]:at[b + 1]].view(-1, hk, d)[:n], vc[at[b]:at[b + 1]].view(-1, hk, d)[:n]) for b, n in enumerate(lens)]
    return kc, vc, table, rows


def _run(q, kc, vc, table, lens, cu, causal=True):
    out, lse = torch.full_like(q, 5.0), torch.full(q.shape[:2], 5.0, device=DEV)
    ops.attention_paged(q, kc, vc, table, _i32(lens), _i32(cu), out, causal=causal, lse=lse)
    return out, lse


# one session cut into many pieces; sessions cut into a few; chunks whose tiles two CTAs share, cut into many and a few;
# and calls of which each job is whole
FORMS = [
    (BF16, 16, 2, 256, [1501], [1]), (F16, 8, 2, 128, [20000], [1]), (BF16, 4, 2, 64, [5000, 700], [1, 1]),
    (BF16, 16, 2, 256, [1500] * 24, [1] * 24), (F16, 16, 2, 128, [700] * 40, [1] * 40),
    (BF16, 16, 2, 256, [20000], [64]), (F16, 32, 2, 128, [6000], [40]), (BF16, 16, 2, 256, [1500], [1500]), (F16, 8, 1, 128, [2100], [1700]),
    (BF16, 4, 4, 64, [90, 120, 33], [5, 1, 33]), (BF16, 8, 1, 256, [60, 50], [50, 50]),
]


@pytest.mark.parametrize("dtype,hq,hk,d,lens,new", FORMS)
def test_a_query_of_nan_gives_nan(dtype, hq, hk, d, lens, new):
    """A query with one NaN has NaN scores everywhere, hence no maximum."""
    g, cu = _gen(31), _prefix(new)
    kc, vc, table, rows = _cache(g, lens, hk, d, 16, dtype)
    q = _randn(g, cu[-1], hq, d, dtype=dtype)
    hit = torch.zeros(cu[-1], hq, dtype=torch.bool, device=DEV)
    hit[0, 0] = hit[-1, hq - 1] = hit[cu[-1] // 2, hq // 2] = True
    q[hit] = torch.where(torch.arange(d, device=DEV) == 3, NAN, q[hit].float()).to(dtype)
    out, lse = _run(q, kc, vc, table, lens, cu)
    assert torch.isnan(out[hit]).all() and torch.isnan(lse[hit]).all()
    clean = torch.where(hit[..., None], torch.zeros_like(q), q)
    for b, (k, v) in enumerate(rows):
        r = slice(cu[b], cu[b + 1])
        o, a, want = exact_rows(clean[r], k, v, True, d ** -0.5)
        fine = ~hit[r]
        check(out[r][fine], lse[r][fine], (o[fine], a[fine], want[fine]), dtype, lens[b], 6.0, f"sequence {b}")


@pytest.mark.parametrize("dtype,hq,hk,d,lens,new", FORMS)
@pytest.mark.parametrize("where", ["first", "middle"])
def test_keys_of_nan_give_nan(dtype, hq, hk, d, lens, new, where):
    """A run of NaN keys, longer than a piece where the sequence is long: every query that sees one of them."""
    g, cu = _gen(32), _prefix(new)
    kc, vc, table, rows = _cache(g, lens, hk, d, 16, dtype)
    q = _randn(g, cu[-1], hq, d, dtype=dtype)
    at = 0 if where == "first" else lens[0] // 3
    clean = rows[0][0].clone()
    rows[0][0][at:at + max(1, lens[0] // 4)] = NAN
    out, lse = _run(q, kc, vc, table, lens, cu)
    sees = lens[0] - new[0] + torch.arange(new[0], device=DEV) >= at
    n = new[0]
    assert torch.isnan(out[:n][sees]).all() and torch.isnan(lse[:n][sees]).all()
    for b, (k, v) in enumerate(rows):
        r = slice(cu[b], cu[b + 1])
        o, a, want = exact_rows(q[r], clean if b == 0 else k, v, True, d ** -0.5)
        fine = ~sees if b == 0 else torch.ones(new[b], dtype=torch.bool, device=DEV)
        check(out[r][fine], lse[r][fine], (o[fine], a[fine], want[fine]), dtype, lens[b], 6.0, f"sequence {b}")


@pytest.mark.parametrize("dtype,hq,hk,d,lens,new", FORMS)
@pytest.mark.parametrize("what", ["k", "v"])
def test_nan_behind_a_weight_that_underflows(dtype, hq, hk, d, lens, new, what):
    """The first keys' scores lie 400 below the last ones', so that their weights are 0 in fp32; one of them is NaN, or its
    value is. Every query of the first sequence sees it (it is key 0)."""
    g, cu = _gen(33), _prefix(new)
    kc, vc, table, rows = _cache(g, lens, hk, d, 16, dtype)
    q = _randn(g, cu[-1], hq, d, dtype=dtype)
    q[..., 0] = 40.0
    k, v = rows[0]
    k[:, :, 0] = 0.0
    k[lens[0] // 2:, :, 0] = 10.0 * d ** 0.5
    (k if what == "k" else v)[0] = NAN
    out, lse = _run(q, kc, vc, table, lens, cu)
    n = new[0]
    assert torch.isnan(out[:n]).all()
    assert torch.isnan(lse[:n]).all() if what == "k" else torch.isfinite(lse[:n]).all()
    assert torch.isfinite(out[n:]).all() and torch.isfinite(lse[n:]).all()


@pytest.mark.parametrize("hq,hk,d", [(4, 2, 64), (16, 2, 128), (16, 2, 256)])
@pytest.mark.parametrize("length", [2, 3, 5])
def test_nan_tiles_of_whole_jobs(hq, hk, d, length):
    """All tiles of keys but the last one are NaN (tiles are of 64 or 128 keys): out and lse are NaN, in jobs that no border cuts too."""
    for tile in (64, 128):
        g, n = _gen(34), tile * (length - 1) + 9
        batch = 1 if length == 2 else 300
        q, k, v = (_randn(g, batch * n, h, d, dtype=BF16) for h in (hq, hk, hk))
        k.view(batch, n, hk, d)[:, :n - 9] = NAN
        out, lse = torch.empty_like(q), torch.empty(batch * n, hq, device=DEV)
        ops.attention_packed(q, k, v, torch.arange(0, batch * n + 1, n, dtype=torch.int32, device=DEV), out, causal=False, lse=lse)
        assert torch.isnan(out).all() and torch.isnan(lse).all()
