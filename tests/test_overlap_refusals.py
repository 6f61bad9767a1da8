"""Which outputs the paged-cache and attention entry points refuse for lying in memory that the call reads or writes
elsewhere: host only, nothing is launched."""
import pytest

from halo_flash_b200 import _lib
from tests.test_attention_abi import _packed, _paged

M = 1 << 20  # addresses far from each other
Q, K, V, OUT, WS, CU = (i << 32 for i in range(1, 7))


def _message(name, *args):
    with pytest.raises(_lib.HaloError) as e:
        _lib.lib().call(name, None, *args)
    return str(e.value)


def packed(**kw):
    return _message("attention_packed", *_packed(**{**dict(q=Q, k=K, v=V, out=OUT, ws=WS, cu=CU), **kw}))


def paged(**kw):
    return _message("attention_paged", *_paged(**{**dict(q=Q, k=K, v=V, out=OUT, ws=WS, cu=CU, table=CU + M, kv=CU + 2 * M), **kw}))


@pytest.mark.parametrize("call", [packed, paged])
@pytest.mark.parametrize("change,word", [
    ({"orow": 128, "oh": 128}, "rows of out"), ({"orow": 256, "oh": 128}, "rows of out"),  # token t, head 1 is token t + 1, head 0
    ({"orow": 1024, "oh": 128, "hq": 16}, "rows of out"), ({"orow": 128, "oh": 512}, "rows of out"),
    ({"out": K + 256}, "memory of k"), ({"out": V + 3 * 512}, "memory of k"), ({"out": K - 1024 * 7 * 2}, "memory of k"),
    ({"out": Q + 256}, "memory of q"), ({"out": Q + 2048}, "memory of q"), ({"out": Q, "orow": 2048}, "memory of q"),
    ({"out": Q, "orow": 128, "oh": 1024}, "memory of q")])
def test_attention_refuses_outputs_in_other_memory(call, change, word):
    assert word in call(**change)


def test_attention_refuses_an_output_across_k_of_one_projection():
    """q, k and v side by side in rows of one buffer, out shifted from q into k."""
    row = (8 + 2 + 2) * 128
    assert "memory of k" in packed(qr=row, kr=row, vr=row, orow=row, k=Q + 1024 * 2, v=Q + 1280 * 2, out=Q + 256, tokens=4000)


@pytest.mark.parametrize("ps,rs,hs", [(8192, 64, 64), (64, 128, 64), (8191, 128, 64), (64, 64 * 2, 64 * 64 * 8), (4096, 128, 64)])
def test_store_refuses_cache_rows_that_overlap(ps, rs, hs):
    assert "cache rows overlap" in _message("paged_store", Q, 128, 64, Q + M, 128, 64, 2, K, V, 2, ps, rs, hs, 3, 64, CU, 2, 64, 5)


@pytest.mark.parametrize("gap,ps", [(0, 8192), (8192 * 2, 8192), (8192 * 2 - 128, 16384), (128, 16384), (-8192 * 4, 8192)])
def test_store_refuses_caches_that_overlap(gap, ps):
    assert "k_cache and v_cache" in _message("paged_store", Q, 128, 64, Q + M, 128, 64, 2, K, K + gap, 2, ps, 128, 64, 3, 64, CU, 2, 64, 5)


def plan(**kw):
    a = dict(table=Q, stride=4, cols=4, past=Q + M, fresh=Q + 2 * M, free=Q + 3 * M, n_free=30, page=64, slot=Q + 4 * M, pos=Q + 5 * M, cu=Q + 6 * M,
             kv=Q + 7 * M, st=Q + 8 * M, batch=6, tokens=50)
    a.update(kw)
    return _message("paged_plan", *a.values())


@pytest.mark.parametrize("name", ["table", "slot", "pos", "cu", "kv", "st"])
@pytest.mark.parametrize("into,size", [("past", 24), ("fresh", 24), ("free", 120)])
def test_plan_refuses_outputs_in_its_inputs(name, into, size):
    at = {"past": Q + M, "fresh": Q + 2 * M, "free": Q + 3 * M}[into]
    for offset in (0, size - 8):
        assert "memory of past" in plan(**{name: at + offset})


def test_plan_refuses_outputs_in_each_other():
    for change in ({"kv": Q + 6 * M}, {"st": Q + 5 * M + 192}, {"pos": Q + 4 * M + 396}, {"cu": Q + 8}, {"slot": Q + 7 * M + 16}):
        assert "share memory" in plan(**change)
