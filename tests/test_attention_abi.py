"""Refusals of the paged-cache and attention entry points, and their no-ops: host only, nothing is launched."""
import pytest

from halo_flash_b200 import _lib

A = 4096  # stands for an aligned device address; none of these calls gets as far as using it


def _fails(name, *args):
    with pytest.raises(_lib.HaloError) as e:
        _lib.lib().call(name, None, *args)
    return str(e.value)


def _packed(**kw):
    a = dict(q=A, qr=1024, qh=128, k=A, kr=256, kh=128, v=A, vr=256, vh=128, out=A, orow=1024, oh=128, dtype=2, cu=A, batch=1,
             tokens=8, hq=8, hk=2, d=128, scale=0.1, causal=1, lse=None, ws=A, bytes=1 << 40)
    a.update(kw)
    return list(a.values())


def _paged(**kw):
    a = dict(q=A, qr=1024, qh=128, k=A, v=A, page=1 << 14, row=256, head=128, pages=9, size=64, table=A, tstride=4, cols=4, kv=A,
             out=A, orow=1024, oh=128, dtype=2, cu=A, batch=1, tokens=8, hq=8, hk=2, d=128, scale=0.1, causal=1, lse=None, ws=A,
             bytes=1 << 40)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("name,make", [("attention_packed", _packed), ("attention_paged", _paged)])
@pytest.mark.parametrize("change,word", [
    ({"q": None}, "null"), ({"out": None}, "null"), ({"cu": None}, "null"), ({"dtype": 0}, "fp16 or bf16"), ({"dtype": 9}, "fp16 or bf16"),
    ({"d": 264}, "multiple of 8"), ({"d": 100}, "multiple of 8"), ({"d": 0}, "multiple of 8"), ({"hq": 9}, "kv_heads"), ({"hk": 0}, "kv_heads"),
    ({"hq": 0}, "kv_heads"), ({"hq": 258, "hk": 2}, "128"), ({"scale": 0.0}, "scale"), ({"scale": -1.0}, "scale"), ({"scale": float("nan")}, "scale"),
    ({"scale": float("inf")}, "scale"), ({"causal": 2}, "causal"), ({"q": A + 8}, "aligned"), ({"out": A + 2}, "aligned"), ({"cu": A + 2}, "aligned"),
    ({"lse": A + 1}, "aligned"), ({"qr": 1028}, "strides"), ({"oh": 4}, "strides"), ({"ws": None}, "workspace"), ({"ws": A + 4}, "workspace"),
    ({"bytes": 1000}, "workspace"), ({"tokens": 1 << 31}, "2^31")])
def test_attention_refuses(name, make, change, word):
    assert word in _fails(name, *make(**change))


@pytest.mark.parametrize("name,make", [("attention_packed", _packed), ("attention_paged", _paged)])
@pytest.mark.parametrize("change,word", [({"orow": 0}, "overlap"), ({"oh": 0}, "overlap"), ({"oh": 120}, "overlap"), ({"out": A}, "memory of"),
                                         ({"out": 2 * A, "v": 2 * A}, "memory of")])
def test_attention_refuses_outputs_that_overlap(name, make, change, word):
    assert word in _fails(name, *make(**{"out": 3 * A, **change}))


@pytest.mark.parametrize("ps,rs,hs", [(0, 128, 64), (8192, 0, 64), (8192, 128, 0), (8192, 56, 64)])
def test_store_refuses_cache_rows_that_overlap(ps, rs, hs):
    assert "overlap" in _fails("paged_store", A, 128, 64, A, 128, 64, 2, A, A, 2, ps, rs, hs, 3, 64, A, 2, 64, 5)


def test_paged_attention_refuses():
    for change, word in (({"size": 48}, "page size"), ({"size": 4}, "page size"), ({"size": 512}, "page size"), ({"table": None}, "null"),
                         ({"kv": None}, "null"), ({"pages": 0}, "no pages"), ({"row": 260}, "strides"), ({"pages": 1 << 31}, "2^31")):
        assert word in _fails("attention_paged", *_paged(**change))


def test_workspace_grows_with_the_head_size():
    size = _lib.lib().cdll.halo_b200_attention_workspace
    assert 0 < size(64) == size(8) < size(128) == size(72) < size(256) == size(136) < 1 << 26
    assert "workspace" in _fails("attention_packed", *_packed(d=256, qr=2048, qh=256, bytes=size(128)))


def test_plan_and_store_refuse():
    plan = lambda table=A, stride=4, cols=4, past=A, fresh=A, free=A, n_free=3, page=64, slot=A, pos=None, cu=None, kv=None, st=None, batch=2, tokens=5: \
        [table, stride, cols, past, fresh, free, n_free, page, slot, pos, cu, kv, st, batch, tokens]  # noqa: E731
    for change, word in (({"page": 65}, "page size"), ({"table": None}, "table"), ({"past": None}, "null"), ({"fresh": None}, "null"),
                         ({"slot": None}, "slot"), ({"free": None}, "free list"), ({"stride": 3}, "overlap"), ({"batch": 16385}, "16384"),
                         ({"slot": A + 4}, "aligned"), ({"st": A + 1}, "aligned"), ({"n_free": 1 << 31}, "2^31"), ({"kv": A}, "must not be"), ({"cu": A}, "must not be")):
        assert word in _fails("paged_plan", *plan(**change))
    store = lambda k=A, kr=128, kh=64, v=A, vr=128, vh=64, dt=2, kc=A, vc=A, ct=2, ps=8192, rs=128, hs=64, pages=3, page=64, slot=A, heads=2, d=64, tokens=5: \
        [k, kr, kh, v, vr, vh, dt, kc, vc, ct, ps, rs, hs, pages, page, slot, heads, d, tokens]  # noqa: E731
    for change, word in (({"page": 0}, "page size"), ({"dt": 5}, "dtype"), ({"k": None}, "null"), ({"vc": None}, "null"), ({"slot": None}, "null"),
                         ({"slot": A + 4}, "aligned"), ({"k": A + 1}, "aligned"), ({"dt": 2, "ct": 0}, "dtype combination")):
        assert word in _fails("paged_store", *store(**change))


def test_empty_calls_are_no_ops():
    lib = _lib.lib()
    lib.call("attention_packed", None, *_packed(tokens=0))
    lib.call("attention_packed", None, *_packed(batch=0))
    lib.call("attention_paged", None, *_paged(tokens=0))
    lib.call("paged_store", None, A, 1, 1, A, 1, 1, 2, A, A, 2, 1, 1, 1, 4, 64, A, 2, 64, 0)
    lib.call("paged_plan", None, None, 0, 0, None, None, None, 0, 64, None, None, None, None, None, 0, 0)


def test_ops_refuse_what_is_no_cuda_tensor():
    """The extension module's own checks, as far as they go without a device."""
    import torch
    from halo_flash_b200 import ops
    t = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    c = torch.zeros(3, 16, 2, 64, dtype=torch.bfloat16)
    i = torch.zeros(4, dtype=torch.int32)
    for call in (lambda: ops.attention_packed(t, t, t, i, t), lambda: ops.attention_packed(None, t, t, i, t),
                 lambda: ops.attention_paged(t, c, c, i[None], i, i, t), lambda: ops.paged_store(t, t, c, c, i.long()),
                 lambda: ops.paged_plan(i[None], i, i, i, 16, i.long()), lambda: ops.paged_plan([1], i, i, i, 16, i.long())):
        with pytest.raises(TypeError, match="CUDA tensor"):
            call()
