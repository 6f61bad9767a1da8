"""Attention in fp16, at the tolerance that its factor 2^6 on the weights allows (GPU only).

p is kept as 2^6 p relative to a reference that no row's maximum falls below, so l >= 2^6 in the same units. A weight below the
smallest normal, 2^-14, is off by at most 2^-25, which is 2^-31 of l: keys * 2^-31 max |v| beside the roundings (eps / 2 of the
output and of each weight) and the fp32 sums (2^-13, scores as in test_gpu_attention.py). Without the factor it would be
2^-25 a key. Where scores are four times as large, sum |q k| scale is below 0.64 * 4 * 16 = 41, and 16 partial sums rounded at
2^-23 of that move a weight by 2^-13.6: 2^-12 in all. lse moves by as much as a weight does relative to itself, and by the roundings of
fp32 values below 50 (1e-5).
"""
import pytest
import torch

from halo_flash_b200 import ops
from tests.test_gpu_attention import DEV, F16, _gen, _i32, _prefix, _randn, exact_rows

pytestmark = pytest.mark.gpu


def _check(out, lse, want, keys, vmax, sums=2.0 ** -13):
    o, a, want_lse = want
    bound = 2.0 ** -11 * (o.abs() + a) + sums * a + keys * 2.0 ** -31 * vmax + 1e-30
    off = (out.double() - o).abs()
    assert (off <= bound).all(), float((off / bound).max())
    assert (lse.double() - want_lse).abs().max() < sums + 1e-5


def _paged(g, k, v, page):
    n, hk, d = k.shape
    pages = -(-n // page)
    caches = [torch.zeros(pages, page, hk, d, dtype=F16, device=DEV) for _ in range(2)]
    for cache, rows in zip(caches, (k, v)):
        cache.view(-1, hk, d)[:n] = rows
    order = torch.randperm(pages, generator=g, device=DEV)
    table = torch.empty(1, pages, dtype=torch.int32, device=DEV)
    table[0] = order.argsort().to(torch.int32)
    return [c[order] for c in caches], table


@pytest.mark.parametrize("hq,hk,d", [(4, 2, 64), (12, 4, 96), (8, 2, 128), (16, 2, 256)])
@pytest.mark.parametrize("past,new,spread", [(1336, 1, 1.0), (6000, 1, 4.0), (900, 70, 1.0), (0, 700, 4.0), (3, 1, 4.0)])
def test_paged(hq, hk, d, past, new, spread):
    g, n = _gen(51), past + new
    q, k, v = _randn(g, new, hq, d, dtype=F16), _randn(g, n, hk, d, dtype=F16), _randn(g, n, hk, d, dtype=F16)
    q = q * spread
    (kc, vc), table = _paged(g, k, v, 32)
    out, lse = torch.empty_like(q), torch.empty(new, hq, device=DEV)
    ops.attention_paged(q, kc, vc, table, _i32([n]), _i32([0, new]), out, lse=lse)
    _check(out, lse, exact_rows(q, k, v, True, d ** -0.5), n, float(v.float().abs().max()), 2.0 ** -13 if spread == 1.0 else 2.0 ** -12)


@pytest.mark.parametrize("hq,hk,d", [(4, 2, 64), (8, 2, 128), (16, 2, 256)])
@pytest.mark.parametrize("lens", [[700, 1, 0, 257], [2000]])
def test_packed(hq, hk, d, lens):
    g, cu = _gen(52), _prefix(lens)
    q, k, v = (_randn(g, cu[-1], h, d, dtype=F16) for h in (hq, hk, hk))
    out, lse = torch.empty_like(q), torch.empty(cu[-1], hq, device=DEV)
    ops.attention_packed(q, k, v, _i32(cu), out, lse=lse)
    for a, b in zip(cu[:-1], cu[1:]):
        if b > a:
            _check(out[a:b], lse[a:b], exact_rows(q[a:b], k[a:b], v[a:b], True, d ** -0.5), b - a, float(v.float().abs().max()))


@pytest.mark.parametrize("hq,hk,d", [(4, 2, 64), (8, 2, 128), (16, 2, 256)])
@pytest.mark.parametrize("new", [1, 128])
def test_weights_of_a_few_steps_of_the_smallest_subnormal(hq, hk, d, new):
    """One key in 64 holds nearly all of the weight and a value of 0, in every tile, so that each reference is theirs; the result is
    what the others of relative weight 2^-22.5 (2.8 steps of fp16, which would be rounded to 3) add up to. l is at least 2^6 for
    each of the large ones: 64 keys * 2^-31 max |v|."""
    g, n = _gen(53), 20000
    q, k, v = torch.zeros(new, hq, d, dtype=F16, device=DEV), torch.zeros(n, hk, d, dtype=F16, device=DEV), _randn(g, n, hk, d, dtype=F16)
    q[..., 0] = 8.0
    k[7::64, :, 0] = 22.5 * 0.6931471805599453 * d ** 0.5 / 8.0
    v = (v + 1.0) * 64.0
    v[7::64] = 0.0
    (kc, vc), table = _paged(g, k, v, 64)
    out, lse = torch.empty_like(q), torch.empty(new, hq, device=DEV)
    ops.attention_paged(q, kc, vc, table, _i32([n]), _i32([0, new]), out, lse=lse)
    # a causal row may end inside a run of 64: two runs' keys for each whole one at most
    _check(out, lse, exact_rows(q, k, v, True, d ** -0.5), 2 * 64, float(v.float().abs().max()))
