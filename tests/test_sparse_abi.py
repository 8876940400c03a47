"""Refusals of the page bounds and sparse attention entry points, and their
64-bit statement on small inputs, without a GPU."""
import numpy as np
import pytest
import torch

import _sparseref as S
from xllms_b200 import _native
from xllms_b200 import operator_api as PA

F = 1 << 20  # an aligned address; nothing is launched, so it is never read


def test_statement_keeps_the_better_page_and_the_earlier_of_two():
    q = np.array([[[1.0, -1.0]]], np.float16)
    bnd = np.zeros((6, 1, 2, 2), np.float16)
    bnd[:, 0, 1, 0] = [1, 3, 2, 3, 0, 0]  # scores
    t, n = np.arange(6, dtype=np.int32)[None], [6 * 16]
    assert S.select(q, bnd, t, n, 16, 2, 0, 1, 1.0, 6).tolist() == [[[1, 5]]]
    assert S.select(q, bnd, t, n, 16, 3, 1, 1, 1.0, 6).tolist() == [[[0, 1, 5]]]
    assert S.select(q, bnd, t, n, 16, 3, 0, 1, -1.0, 6).tolist() == [[[0, 1, 5]]]
    assert S.select(q, bnd, t, n, 16, 4, 0, 1, 1.0, 3).tolist() == [[[0, 1, 2, -1]]]


def _bounds(lib, q4=False, bnd=F, kc=F, bt=F, sl=F, B=2, hkv=2, d=64, mb=4, bs=16, ds=2, ks=1.0,
            kbs=1152, khs=576, new=0):
    if q4:
        return lib.nxt_page_bounds_q4(bnd, kc, bt, sl, B, hkv, d, mb, bs, ks, kbs, khs, 8, new,
                                      None, None)
    return lib.nxt_page_bounds(bnd, kc, bt, sl, B, hkv, d, mb, bs, ds, kbs, khs, 8, new, None, None)


BAD_BOUNDS = [dict(bnd=None), dict(kc=None), dict(bt=None), dict(sl=None), dict(B=-1),
              dict(hkv=0), dict(d=0), dict(d=257), dict(mb=-1), dict(bs=0), dict(kbs=-16),
              dict(khs=-16), dict(new=-1), dict(bnd=F + 1), dict(kc=F + 1)]


@pytest.mark.parametrize("q4", [False, True])
@pytest.mark.parametrize("bad", BAD_BOUNDS, ids=str)
def test_bounds_refuse(bad, q4):
    assert _bounds(_native.xpa(), q4=q4, **bad) == _native.NXT_PA_EINVAL


@pytest.mark.parametrize("bad", [dict(d=72), dict(bs=8), dict(ks=0.0), dict(ks=float("nan")),
                                 dict(kc=F + 8), dict(kbs=1160), dict(khs=8)], ids=str)
def test_4_bit_bounds_refuse(bad):
    assert _bounds(_native.xpa(), q4=True, **bad) == _native.NXT_PA_EINVAL


def test_bounds_refuse_other_types_and_do_nothing_without_sequences():
    lib = _native.xpa()
    assert _bounds(lib, ds=1) == _native.NXT_PA_EINVAL
    assert _bounds(lib, ds=4, kc=F + 2) == _native.NXT_PA_EINVAL
    assert _bounds(lib, B=0) == _native.NXT_PA_OK
    assert _bounds(lib, mb=0) == _native.NXT_PA_OK


def _call(lib, kind, out=F, q=F, kc=F, vc=F, bnd=F, bt=F, sl=F, tab=F, B=2, hq=4, d=64, hkv=2,
          scale=0.1, mb=40, bs=16, ds=2, ks=1.0, vs=1.0, kbs=1152, khs=576, keep=8, sink=1,
          recent=2, ws=None):
    tail = (kbs, khs, 8, keep, sink, recent, ws, 0, F, None)
    if kind == "select":
        return lib.nxt_select_pages(tab, out, None, q, bnd, bt, sl, B, hq, d, hkv, scale, mb, bs,
                                    ds, *tail)
    head = (out, q, kc, vc, bnd, bt, sl, None, B, hq, d, hkv, scale, mb, bs)
    if kind == "q4":
        return lib.nxt_paged_attention_q4_sparse_ex(*head, ks, vs, *tail)
    return lib.nxt_paged_attention_sparse_ex(*head, ds, *tail)


BAD = [dict(out=None), dict(q=None), dict(bnd=None), dict(bt=None), dict(sl=None), dict(B=-1),
       dict(hq=3), dict(hkv=0), dict(d=0), dict(d=272), dict(mb=-1), dict(bs=0), dict(kbs=-16),
       dict(keep=0), dict(sink=-1), dict(recent=0), dict(sink=7), dict(keep=2 ** 28),
       dict(scale=float("nan")), dict(kbs=1168), dict(kbs=576), dict(khs=0), dict(ws=F + 8),
       dict(bnd=F + 1), dict(q=F + 1)]


@pytest.mark.parametrize("kind", ["plain", "q4", "select"])
@pytest.mark.parametrize("bad", BAD, ids=str)
def test_sparse_calls_refuse(bad, kind):
    assert _call(_native.xpa(), kind, **bad) == _native.NXT_PA_EINVAL


@pytest.mark.parametrize("bad", [dict(kc=None), dict(vc=None)], ids=str)
@pytest.mark.parametrize("kind", ["plain", "q4"])
def test_attention_needs_its_pools(bad, kind):
    assert _call(_native.xpa(), kind, **bad) == _native.NXT_PA_EINVAL


def test_kinds_own_refusals():
    lib = _native.xpa()
    for bad in (dict(ds=1), dict(ds=8)):
        assert _call(lib, "plain", **bad) == _native.NXT_PA_EINVAL
    for bad in (dict(d=72), dict(bs=24), dict(ks=0.0), dict(vs=float("inf")), dict(kc=F + 4),
                dict(kbs=1154, khs=577)):
        assert _call(lib, "q4", **bad) == _native.NXT_PA_EINVAL
    assert _call(lib, "select", tab=None) == _native.NXT_PA_EINVAL


@pytest.mark.parametrize("kind", ["plain", "q4", "select"])
def test_no_sequences_do_nothing(kind):
    assert _call(_native.xpa(), kind, B=0) == _native.NXT_PA_OK


def test_workspace_query():
    fn = _native.xpa().nxt_paged_attention_sparse_workspace_size
    assert fn(0, 8, 64, 2, 10, 16, 2, 4) == 0 and fn(1, 8, 64, 2, 10, 16, 2, 0) == 0
    rows, mb, keep = 4 * 2, 100, 10
    assert fn(4, 8, 64, 2, mb, 16, 2, keep) >= rows * mb * 16 + rows * keep * 4 + rows * 4


def test_python_wrappers_refuse_host_tensors():
    pool = torch.zeros(4, 2, 16, 64, dtype=torch.float16)
    bnd = torch.zeros(4, 2, 2, 64, dtype=torch.float16)
    q = torch.zeros(1, 4, 64, dtype=torch.float16)
    t, n = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for call in (lambda: PA.page_bounds(pool, t, n, bnd),
                 lambda: PA.select_pages(q, pool, bnd, t, n, 4),
                 lambda: PA.paged_attention_sparse(q, pool, pool, bnd, t, n, 4),
                 lambda: PA.paged_attention_sparse(q, pool, pool, bnd, t, n, 4, k_scale=1.0)):
        with pytest.raises(PA.PagedAttentionError):
            call()
