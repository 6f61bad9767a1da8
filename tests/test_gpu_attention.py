"""Attention over packed prompts and over a paged K/V cache against softmax attention in 64 bits (GPU only).

Tolerance, derived before the first run. With p_j the softmax weights and A = sum p_j |v_j| of an output element o:
  * o is rounded once to the 16-bit type: eps / 2 |o|; p is rounded once for the second product: eps / 2 A;
  * fp32: S = <q, k> is a sum of exact products, its error (at most 16 partial sums, 2^-23 each, of values that
    add up to about 10 after scaling) moves p by a few 1e-5 relative, the sums over the keys lose at most 2^-23 for
    each of the (at most 512) partial sums: together below 2^-13 A;
  * fp16 only: p is taken relative to a reference that the row's maximum exceeds by at most 2^8, so l >= 1, and a p
    below the smallest normal 2^-14 is off by at most 2^-25: keys * 2^-25 max |v|.
lse is fp32 arithmetic: 1e-5 absolute (hardware exp2 and log2 are good to 2^-22, values are below 30).
"""
import pytest
import torch

from halo_flash_b200 import HaloError, lib, ops

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, F16 = torch.bfloat16, torch.float16


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _randn(g, *shape, dtype):
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _prefix(values):
    out = [0]
    for v in values:
        out.append(out[-1] + v)
    return out


def exact_rows(q, k, v, causal, scale):
    """One sequence in 64 bits: (o, A, lse) of q [n, Hq, d] over k, v [L, Hk, d]."""
    n, hq, d = q.shape
    length, group = k.shape[0], hq // k.shape[1]
    o = torch.zeros(n, hq, d, dtype=torch.float64, device=q.device)
    a = torch.zeros_like(o)
    lse = torch.full((n, hq), float("-inf"), dtype=torch.float64, device=q.device)
    if length == 0:
        return o, a, lse
    last = length - n + torch.arange(n, device=q.device) if causal else torch.full((n,), length - 1, device=q.device)
    hidden = torch.arange(length, device=q.device)[None] > last[:, None]
    sees = ~hidden.all(1)
    for h in range(hq):
        s = q[:, h].double() @ k[:, h // group].double().T * scale
        s[hidden] = float("-inf")
        lse[:, h] = torch.logsumexp(s, 1)
        p = torch.where(sees[:, None], (s - torch.where(sees, lse[:, h], 0.0)[:, None]).exp(), 0.0)
        vh = v[:, h // group].double()
        o[:, h] = p @ vh
        a[:, h] = p @ vh.abs()
    return o, a, lse


def check(out, lse, want, dtype, keys, vmax, what):
    o, a, want_lse = want
    half = torch.finfo(dtype).eps / 2
    bound = half * (o.abs() + a) + 2.0 ** -13 * a + 1e-30
    if dtype == F16:
        bound = bound + keys * 2.0 ** -25 * vmax
    bad = ~((out.double() - o).abs() <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst {float(((out.double() - o).abs() / bound).max()):.2f}"
    if lse is not None:
        assert torch.equal(torch.isinf(lse), torch.isinf(want_lse)), f"{what}: lse of empty rows"
        fine = torch.isfinite(want_lse)
        assert (lse.double()[fine] - want_lse[fine]).abs().max() < 1e-5 if fine.any() else True, f"{what}: lse"


def packed(lens, hq, hk, d, dtype, causal=True, seed=0, scale=None, spread=1.0, workspace=None):
    g = _gen(seed)
    t = sum(lens)
    q, k, v = (_randn(g, t, h, d, dtype=dtype) for h in (hq, hk, hk))
    q = q * spread
    out = torch.full_like(q, float("nan"))
    lse = torch.full((t, hq), float("nan"), device=DEV)
    cu = _prefix(lens)
    ops.attention_packed(q, k, v, _i32(cu), out, causal=causal, lse=lse, scale=scale, workspace=workspace)
    for b, n in enumerate(lens):
        r = slice(cu[b], cu[b + 1])
        want = exact_rows(q[r], k[r], v[r], causal, d ** -0.5 if scale is None else scale)
        check(out[r], lse[r], want, dtype, n, float(v.float().abs().max()), f"sequence {b} of {n}")
    return q, k, v, out


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("hq,hk,d", [(4, 2, 64), (16, 2, 256), (8, 8, 128)])
@pytest.mark.parametrize("lens", [[1], [7], [64], [130], [1, 23, 8], [200, 0, 77, 129]])
def test_packed_prompts(dtype, hq, hk, d, lens):
    packed(lens, hq, hk, d, dtype)


@pytest.mark.parametrize("hq,hk,d", [(3, 1, 64), (6, 2, 96), (7, 1, 256), (12, 4, 80), (5, 5, 8), (24, 2, 200), (32, 1, 128), (128, 1, 64), (40, 8, 32)])
def test_packed_head_layouts(hq, hk, d):
    packed([33, 150, 5], hq, hk, d, BF16, seed=3)


@pytest.mark.parametrize("dtype,hq,hk,d,lens", [(BF16, 16, 2, 256, [1500]), (F16, 4, 2, 64, [2000, 611]), (BF16, 8, 2, 128, [5, 1300, 0, 1, 900])])
@pytest.mark.parametrize("causal", [True, False])
def test_packed_long(dtype, hq, hk, d, lens, causal):
    packed(lens, hq, hk, d, dtype, causal=causal, seed=4)


def test_packed_many_sequences():
    lens = [(37 * i * i + 11 * i) % 90 for i in range(150)]
    packed(lens, 4, 2, 64, BF16, seed=5)


@pytest.mark.parametrize("d", [64, 256])
def test_large_scores_move_the_reference(d):
    """Scores whose maximum keeps growing along the keys: every tile makes the reference follow."""
    g = _gen(6)
    n, hq, hk = 700, 4, 2
    ramp = torch.linspace(0.0, 60.0, n, device=DEV)[:, None, None]
    q, k, v = (_randn(g, n, h, d, dtype=BF16) for h in (hq, hk, hk))
    q[..., 0] = 1.0
    k[..., 0] = (ramp[..., 0] * d ** 0.5).to(BF16)
    out = torch.empty_like(q)
    lse = torch.empty(n, hq, device=DEV)
    ops.attention_packed(q, k, v, _i32([0, n]), out, lse=lse)
    o, a, want = exact_rows(q, k, v, True, d ** -0.5)
    # scores up to 60 sum products of up to 60 sqrt(d): fp32 rounds them at 2^-23 * 60 a partial sum, p by 2^-13
    bad = (out.double() - o).abs() > 2.0 ** -8 * (o.abs() + a) + 2.0 ** -11 * a
    assert not bad.any()
    assert (lse.double() - want).abs().max() < 1e-3


def test_packed_strides_and_rows_behind():
    """q, k, v as views of one projection buffer, out as a view, rows behind the last sequence untouched."""
    g, t, hq, hk, d = _gen(7), 300, 8, 2, 128
    buf = _randn(g, t, (hq + 2 * hk) * d + 64, dtype=BF16)
    q = buf[:, : hq * d].view(t, hq, d)
    k = buf[:, hq * d:(hq + hk) * d].view(t, hk, d)
    v = buf[:, (hq + hk) * d:(hq + 2 * hk) * d].view(t, hk, d)
    store = torch.full((t, hq, 2 * d), 7.0, dtype=BF16, device=DEV)
    out = store[..., :d]
    buf[250:] = float("nan")  # behind the last sequence
    lse = torch.full((t, hq), 3.0, device=DEV)
    ops.attention_packed(q, k, v, _i32([0, 99, 250]), out, lse=lse)
    for a, b in ((0, 99), (99, 250)):
        check(out[a:b], lse[a:b], exact_rows(q[a:b], k[a:b], v[a:b], True, d ** -0.5), BF16, b - a, 6.0, "view")
    assert (store[250:] == 7.0).all() and (store[..., d:] == 7.0).all() and (lse[250:] == 3.0).all()


def test_neighbouring_sequence_with_nan_stays_there():
    g, d = _gen(8), 64
    q, k, v = (_randn(g, 100, h, d, dtype=F16) for h in (4, 2, 2))
    k[40:] = float("nan")
    v[40:] = float("inf")
    out = torch.empty_like(q)
    ops.attention_packed(q, k, v, _i32([0, 40, 100]), out)
    check(out[:40], None, exact_rows(q[:40], k[:40], v[:40], True, d ** -0.5), F16, 40, 6.0, "first")
    assert torch.isnan(out[40:]).all()


# ---- paged --------------------------------------------------------------------------------------------------------
def paged(past, new, hq, hk, d, page, dtype, seed=0, causal=True, layout="slot", lens=None, rows_behind=0):
    g = _gen(seed)
    total = [p + n for p, n in zip(past, new)] if lens is None else lens
    want = [-(-x // page) for x in total]
    pages, cols = sum(want) + 3, max(max(want), 1) + 1
    order = torch.randperm(pages, generator=g, device=DEV).tolist()
    # entries behind the last key: anything
    table = torch.full((len(new), cols), 0x7FFFFFF0, dtype=torch.int32, device=DEV)
    if layout == "slot":
        kc, vc = (torch.full((pages, page, hk, d), float("nan"), dtype=dtype, device=DEV) for _ in range(2))
    elif layout == "head":  # [pages, heads, rows, d]
        kc, vc = (torch.full((pages, hk, page, d), float("nan"), dtype=dtype, device=DEV).transpose(1, 2) for _ in range(2))
    else:  # K and V beside each other in one buffer
        both = torch.full((pages, 2, page, hk, d), float("nan"), dtype=dtype, device=DEV)
        kc, vc = both[:, 0], both[:, 1]
    ks, vs, at = [], [], 0
    for b, n in enumerate(total):
        mine = order[at:at + want[b]]
        at += want[b]
        table[b, : want[b]] = _i32(mine) if mine else _i32([])
        k, v = _randn(g, n, hk, d, dtype=dtype), _randn(g, n, hk, d, dtype=dtype)
        for i, p in enumerate(mine):
            part = min(page, n - i * page)
            kc[p, :part], vc[p, :part] = k[i * page:i * page + part], v[i * page:i * page + part]
        ks.append(k), vs.append(v)
    t, cu = sum(new), _prefix(new)
    q = _randn(g, t + rows_behind, hq, d, dtype=dtype)
    out = torch.full_like(q, 5.0)
    lse = torch.full((t + rows_behind, hq), 5.0, device=DEV)
    ops.attention_paged(q, kc, vc, table, _i32(total), _i32(cu), out, causal=causal, lse=lse)
    for b, n in enumerate(new):
        r = slice(cu[b], cu[b + 1])
        check(out[r], lse[r], exact_rows(q[r], ks[b], vs[b], causal, d ** -0.5), dtype, total[b], 7.0, f"sequence {b}: {n} new of {total[b]}")
    assert (out[t:] == 5.0).all() and (lse[t:] == 5.0).all()
    return out


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("hq,hk,d", [(16, 2, 256), (4, 2, 64), (24, 8, 128)])
@pytest.mark.parametrize("page", [8, 16, 64, 256])
def test_decode(dtype, hq, hk, d, page):
    paged([0, 1, 63, 64, 500, 1337], [1] * 6, hq, hk, d, page, dtype, seed=page)


@pytest.mark.parametrize("hq,hk,d,page", [(16, 2, 256, 32), (6, 2, 128, 16), (7, 1, 64, 128), (8, 8, 96, 64)])
def test_chunks_beside_single_tokens(hq, hk, d, page):
    paged([0, 300, 17, 1000, 64], [65, 1, 130, 200, 3], hq, hk, d, page, BF16, seed=11)


@pytest.mark.parametrize("layout", ["slot", "head", "both"])
@pytest.mark.parametrize("causal", [True, False])
def test_cache_layouts(layout, causal):
    paged([70, 5], [40, 1], 8, 2, 128, 16, BF16, seed=12, layout=layout, causal=causal, rows_behind=3)


@pytest.mark.parametrize("d", [64, 256])
def test_sequences_without_keys_and_more_rows_than_keys(d):
    """kv_len 0, kv_len below the number of rows (the first rows see nothing), a sequence without rows."""
    paged([0, 0, 0, 0], [3, 40, 0, 200], 8, 2, d, 16, BF16, seed=13, lens=[0, 7, 50, 150])


@pytest.mark.parametrize("hq,hk,d", [(16, 2, 256), (8, 1, 128)])
def test_one_long_sequence_is_split(hq, hk, d):
    paged([20000], [1], hq, hk, d, 64, BF16, seed=14)
    paged([9000, 3, 30], [2, 1, 1], hq, hk, d, 64, BF16, seed=15)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("hq,hk,d,page", [(32, 2, 256, 8), (16, 1, 128, 64), (30, 2, 200, 256)])
def test_many_rows_a_sequence(dtype, hq, hk, d, page):
    """Groups of 15 and 16 heads: the batches whose tiles two CTAs share, with the edges of the ones above."""
    paged([0, 0, 0, 0], [3, 40, 0, 200], hq, hk, d, page, dtype, seed=21, lens=[0, 7, 50, 150])
    paged([9000, 3, 30], [40, 30, 20], hq, hk, d, page, dtype, seed=22)
    paged([70, 5], [40, 31], hq, hk, d, page, dtype, seed=23, layout="both", causal=False, rows_behind=3)
    packed([33, 0, 150, 5], hq, hk, d, dtype, seed=24)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_broadcast_inputs_and_out_in_place_of_q(d):
    """Strides of 0 repeat a row or head; out may be q. Both give the bits of the plain call."""
    g, n = _gen(25), 700
    q, k, v = (_randn(g, n, h, d, dtype=BF16) for h in (16, 1, 1))
    cu = _i32([0, 100, n])
    heads = [x.expand(n, 2, d) for x in (k, v)]
    want = ops.attention_packed(q, *(x.contiguous() for x in heads), cu, torch.empty_like(q))
    assert torch.equal(ops.attention_packed(q, *heads, cu, torch.empty_like(q)), want)
    own = q.clone()
    assert torch.equal(ops.attention_packed(own, *heads, cu, own), want)
    rows = q[:1].expand(n, 16, d), k[:1].expand(n, 1, d)
    want = ops.attention_packed(*(x.contiguous() for x in rows), v, cu, torch.empty_like(q))
    assert torch.equal(ops.attention_packed(*rows, v, cu, torch.empty_like(q)), want)


def test_same_call_gives_the_same_bits_and_shares_no_state():
    g, d = _gen(16), 128
    q, k, v = (_randn(g, 900, h, d, dtype=BF16) for h in (8, 2, 2))
    cu = _i32([0, 100, 900])
    ws = ops.attention_workspace(d)
    first = ops.attention_packed(q, k, v, cu, torch.empty_like(q), workspace=ws)
    ws.fill_(255)  # whatever an earlier call left there
    assert torch.equal(first, ops.attention_packed(q, k, v, cu, torch.empty_like(q), workspace=ws))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.attention_packed(q, k, v, cu, torch.empty_like(q))
    torch.cuda.synchronize()
    assert torch.equal(first, other)


def test_captured_calls_follow_their_lengths():
    """A graph of the paged call replays over whatever the lengths say by then."""
    g, hq, hk, d, page = _gen(17), 16, 2, 256, 64
    kc, vc = (_randn(g, 40, page, hk, d, dtype=BF16) for _ in range(2))
    table = torch.arange(40, dtype=torch.int32, device=DEV).view(2, 20)
    kv_len, cu, q = _i32([10, 700]), _i32([0, 1, 2]), _randn(g, 2, hq, d, dtype=BF16)
    out = torch.empty_like(q)
    ws = ops.attention_workspace(d)
    ops.attention_paged(q, kc, vc, table, kv_len, cu, out, workspace=ws)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.attention_paged(q, kc, vc, table, kv_len, cu, out, workspace=ws)
    for lens in ([10, 700], [1280, 1], [64, 65]):
        kv_len.copy_(_i32(lens))
        graph.replay()
        for b, n in enumerate(lens):
            k, v = (c[table[b].long()].flatten(0, 1)[:n] for c in (kc, vc))
            check(out[b:b + 1], None, exact_rows(q[b:b + 1], k, v, True, d ** -0.5), BF16, n, 7.0, f"{lens}")


def test_no_wait_ran_out():
    import ctypes as C
    n, err = C.c_uint(99), C.create_string_buffer(256)
    assert lib().cdll.halo_b200_stage_timeouts(C.byref(n), err, len(err)) == 0 and n.value == 0


def test_tensor_refusals():
    """What ops checks of the tensors; each call is refused on the host, before anything is launched."""
    q, k, out = (torch.zeros(6, h, 64, dtype=BF16, device=DEV) for h in (4, 2, 4))
    cu, lens, table = _i32([0, 6]), _i32([6]), _i32([[0, 1]])
    kc = torch.zeros(3, 16, 2, 64, dtype=BF16, device=DEV)
    slot = torch.zeros(6, dtype=torch.int64, device=DEV)
    packed = lambda **kw: ops.attention_packed(**{**dict(q=q, k=k, v=k, cu=cu, out=out), **kw})  # noqa: E731
    paged = lambda **kw: ops.attention_paged(**{**dict(q=q, k_cache=kc, v_cache=kc, table=table, kv_len=lens, cu=cu, out=out), **kw})  # noqa: E731
    store = lambda **kw: ops.paged_store(**{**dict(k=k, v=k, k_cache=kc, v_cache=kc, slot=slot), **kw})  # noqa: E731
    plan = lambda **kw: ops.paged_plan(**{**dict(table=table, past=lens, fresh=lens, free_pages=lens, page_size=16, slot=slot), **kw})  # noqa: E731
    for error, word, call in (
            (TypeError, "dtype", lambda: packed(q=q.float())), (TypeError, "out's|q's", lambda: packed(out=out.half())),
            (TypeError, "q's", lambda: packed(k=k.half())), (ValueError, "axes", lambda: packed(q=q[0])), (ValueError, "shape of q", lambda: packed(out=out[:5])),
            (ValueError, "do not fit", lambda: packed(k=k[:5])), (ValueError, "do not fit", lambda: packed(v=k[..., :32])),
            (ValueError, "contiguous", lambda: packed(q=q.transpose(1, 2))), (TypeError, "dtype", lambda: packed(cu=cu.long())),
            (ValueError, "batch", lambda: packed(cu=cu[:0])), (ValueError, "entries", lambda: packed(lse=torch.zeros(5, device=DEV))),
            (TypeError, "dtype", lambda: packed(lse=torch.zeros(24, device=DEV, dtype=BF16))), (HaloError, "workspace", lambda: packed(workspace=slot)),
            (HaloError, "scale", lambda: packed(scale=0.0)), (HaloError, "strides", lambda: packed(q=torch.zeros(6, 4, 68, dtype=BF16, device=DEV)[..., :64])),
            (HaloError, "multiple of 8", lambda: packed(q=q[..., :60], k=k[..., :60], v=k[..., :60], out=out[..., :60])),
            (HaloError, "aligned", lambda: packed(q=torch.zeros(6 * 256 + 1, dtype=BF16, device=DEV)[1:].view(6, 4, 64))),
            (HaloError, "kv_heads", lambda: packed(k=torch.zeros(6, 3, 64, dtype=BF16, device=DEV), v=torch.zeros(6, 3, 64, dtype=BF16, device=DEV))),
            (ValueError, "same shape", lambda: paged(v_cache=kc[:2])), (ValueError, "same shape", lambda: paged(v_cache=kc.transpose(1, 2).contiguous().transpose(1, 2))),
            (TypeError, "q's", lambda: paged(k_cache=kc.half(), v_cache=kc.half())), (ValueError, "do not fit", lambda: paged(table=_i32([[0], [1]]))),
            (ValueError, "entries", lambda: paged(kv_len=_i32([1, 2]))), (TypeError, "CUDA", lambda: paged(kv_len=None)), (TypeError, "CUDA", lambda: paged(table=table.cpu())),
            (HaloError, "page size", lambda: paged(k_cache=kc[:, :15], v_cache=kc[:, :15])), (ValueError, "do not fit", lambda: store(k=k[..., :32], v=k[..., :32])),
            (ValueError, "entries", lambda: store(slot=slot[:5])), (TypeError, "dtype", lambda: store(slot=slot.int())), (TypeError, "k's", lambda: store(v=k.half())),
            (HaloError, "dtype combination", lambda: store(k_cache=kc.float(), v_cache=kc.float())), (ValueError, "entries", lambda: plan(past=_i32([1, 2]))),
            (HaloError, "page size", lambda: plan(page_size=17)), (ValueError, "out of range", lambda: plan(page_size=-16)), (TypeError, "integer", lambda: plan(page_size="x")),
            (ValueError, "entries", lambda: plan(cu=_i32([0]))), (ValueError, "contiguous", lambda: plan(table=torch.zeros(1, dtype=torch.int32, device=DEV).expand(2, 3), past=_i32([0, 0]), fresh=_i32([0, 0]))),
            (ValueError, "overlap", lambda: plan(table=torch.zeros(1, 3, dtype=torch.int32, device=DEV).expand(2, 3), past=_i32([0, 0]), fresh=_i32([0, 0])))):
        with pytest.raises(error, match=word):
            call()


@pytest.mark.parametrize("hq,hk,d", [(4, 2, 64), (8, 2, 128), (8, 1, 256), (2, 2, 256)])
def test_scores_far_from_zero(hq, hk, d):
    """Scaled scores near -900 and near +900: the softmax is the one of their differences, whatever the type of P."""
    for sign in (-1.0, 1.0):
        g = _gen(18)
        n = 400
        q, k, v = (_randn(g, n, h, d, dtype=F16) for h in (hq, hk, hk))
        q[..., 0] = 90.0
        k[..., 0] = sign * 10.0 * d ** 0.5
        out, lse = torch.empty_like(q), torch.empty(n, hq, device=DEV)
        ops.attention_packed(q, k, v, _i32([0, n]), out, lse=lse)
        o, a, want = exact_rows(q, k, v, True, d ** -0.5)
        # fp32 sums of terms up to 900 sqrt(d), at most 16 of them rounded at 2^-23: scores are off by up to 16 * 900 * 2^-23
        # = 2^-9.2, so are p relative to each other
        bad = ~((out.double() - o).abs() <= 2.0 ** -11 * (o.abs() + a) + 2.0 ** -8 * a + n * 2.0 ** -25 * 6.0)
        assert not bad.any(), (sign, int(bad.sum()))
        assert (lse.double() - want).abs().max() < 900 * 2.0 ** -17


def test_table_entries_outside_the_cache_read_as_zeros():
    g, hq, hk, d, page = _gen(19), 8, 2, 128, 16
    kc, vc = (_randn(g, 6, page, hk, d, dtype=BF16) for _ in range(2))
    table, n = _i32([[3, -1, 0, 6, 0x7FFFFFFF, 5]]), 6 * page - 5
    q = _randn(g, 3, hq, d, dtype=BF16)
    out = torch.empty_like(q)
    ops.attention_paged(q, kc, vc, table, _i32([n]), _i32([0, 3]), out)
    zeros = torch.zeros_like(kc[0])
    k, v = (torch.cat([c[3], zeros, c[0], zeros, zeros, c[5]])[:n] for c in (kc, vc))
    check(out, None, exact_rows(q, k, v, True, d ** -0.5), BF16, n, 6.0, "outside")


def test_large_batches_of_short_sequences():
    """More sequences than a warp scans at once, some empty, beside one long one; and the same as single tokens over pages."""
    g, hq, hk, d = _gen(20), 4, 2, 64
    lens = [(i * 7) % 5 for i in range(400)]
    lens[200] = 900
    packed(lens, hq, hk, d, F16, seed=21)
    past = [(i * 37) % 200 for i in range(300)]
    past[17] = 4000
    paged(past, [1] * 300, hq, hk, d, 16, F16, seed=22)


def test_two_streams_at_once():
    """Calls that overlap on the GPU, each with a workspace of its own (from torch's allocator, as by default)."""
    g, d = _gen(23), 128
    sets = [tuple(_randn(g, 1500, h, d, dtype=BF16) for h in (8, 2, 2)) for _ in range(4)]
    cu = _i32([0, 1500])
    alone = [ops.attention_packed(q, k, v, cu, torch.empty_like(q)) for q, k, v in sets]
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in sets], [torch.full_like(s[0], float("nan")) for s in sets]
    for _ in range(5):
        for s, (q, k, v), out in zip(streams, sets, outs):
            with torch.cuda.stream(s):
                ops.attention_packed(q, k, v, cu, out)
    torch.cuda.synchronize()
    for a, b in zip(alone, outs):
        assert torch.equal(a, b)


def test_many_small_weights_in_fp16():
    """One key with weight 1 and 60000 with 2^-17 each, whose sum is what the result mostly is: P of these is far below the
    smallest normal fp16 relative to the maximum."""
    g, d, n = _gen(24), 64, 60000
    q, k, v = (_randn(g, r, 1, d, dtype=F16) for r in (1, n, n))
    q[...] = 0.0
    q[..., 0] = 8.0
    k[...] = 0.0
    k[7, 0, 0] = 17 * 0.6931471805599453  # q k d^-0.5 = 17 ln 2
    v += 1.0
    page = 64
    pages = -(-n // page)
    kc, vc = (torch.zeros(pages, page, 1, d, dtype=F16, device=DEV) for _ in range(2))
    kc.view(-1, 1, d)[:n], vc.view(-1, 1, d)[:n] = k, v
    out = torch.empty_like(q)
    lse = torch.empty(1, 1, device=DEV)
    ops.attention_paged(q, kc, vc, torch.arange(pages, dtype=torch.int32, device=DEV)[None], _i32([n]), _i32([0, 1]), out, lse=lse)
    # p = 2^(6 - 17) here: normal in fp16, so each is rounded at 2^-12 at most, and `keys * 2^-25` is not called upon
    o, a, want = exact_rows(q, k, v, True, d ** -0.5)
    assert ((out.double() - o).abs() <= 2.0 ** -12 * (o.abs() + a) + 2.0 ** -13 * a).all()
    assert (lse.double() - want).abs().max() < 1e-5
