"""Sparse decode attention, and its selection, on the paths that longer and odder
calls take."""

import numpy as np
import pytest

from test_sparse_gpu import _case, _t
from xllms_b200 import _native
from xllms_b200 import operator_api as PA

pytestmark = pytest.mark.gpu
KS, VS = 0.011, 0.0073


@pytest.mark.parametrize("kind", ["tensor cores", "scalar"])
def test_pages_that_are_not_there_widen_no_error_bound(cuda, kind):
    """The bounds of page 0 where no row names it: an infinite or huge entry
    there sends no page more to the pass in 64 bits (seen by how much of the
    workspace a call writes) and changes nothing that is kept."""
    import torch
    dtype = np.float16 if kind == "tensor cores" else np.float32
    rng = np.random.default_rng(12)
    hq, hkv, D, bs, n, keep = 8, 2, 64, 16, 100, 20
    bnd = np.sort(rng.standard_normal((n + 1, hkv, 2, D)), 2).astype(dtype)
    table = (1 + rng.permutation(n)).astype(np.int32)[None]
    table[0, [3, 50]] = -1
    q, lens = _t(rng.standard_normal((1, hq, D)).astype(dtype), cuda), _t(np.array([n * bs], np.int32), cuda)
    tt = _t(table, cuda)
    es = np.dtype(dtype).itemsize
    need = PA.sparse_workspace_size(1, hq, D, hkv, n, keep, bs, es)
    seen = []
    for first in (0.0, float(np.finfo(dtype).max), np.inf, np.nan):
        bnd[0] = first
        bt = _t(bnd, cuda)
        ws = torch.full((need,), 0xa7, dtype=torch.uint8, device=cuda)
        tables, slens, pages = (torch.zeros(s, dtype=torch.int32, device=cuda)
                                for s in ((hkv, keep), (hkv,), (1, hkv, keep)))
        rc = _native.xpa().nxt_select_pages(
            tables.data_ptr(), slens.data_ptr(), pages.data_ptr(), q.data_ptr(), bt.data_ptr(),
            tt.data_ptr(), lens.data_ptr(), 1, hq, D, hkv, 0.125, n, bs, es, hkv * bs * D, bs * D,
            n + 1, keep, 1, 1, ws.data_ptr(), need, None, torch.cuda.current_stream().cuda_stream)
        assert rc == _native.NXT_PA_OK
        words = ws[:need // 4 * 4].view(torch.int32)
        sentinel = torch.full((4,), 0xa7, dtype=torch.uint8, device=cuda).view(torch.int32)
        seen.append((int((words != sentinel).sum()), pages.cpu().numpy().tolist()))
    PA.device_status(clear=True)
    assert all(s == seen[0] for s in seen[1:]), [s[0] for s in seen]


def test_selected_tables_of_4_bit_pools(cuda):
    """select_pages over a 4-bit pool: the tables of its pages, per KV head."""
    import torch
    hq, hkv, D, bs, keep = 8, 2, 64, 32, 7
    q, k, v, table, lens = _case(41, [900, 0, 77], hq, hkv, D, bs)
    kc = torch.zeros(PA.q4_pool_shape(len(k), hkv, bs, D), dtype=torch.uint8, device=cuda)
    vc = torch.zeros_like(kc)
    rows = lambda x: _t(x.transpose(0, 2, 1, 3).reshape(-1, hkv, D), cuda)
    PA.reshape_and_cache_q4(rows(k), rows(v), kc, vc, torch.arange(len(k) * bs, device=cuda), KS, VS)
    qt, tt, lt = _t(q, cuda), _t(table, cuda), _t(lens, cuda)
    bnd = PA.page_bounds(kc, tt, lt, torch.zeros(len(k), hkv, 2, D, dtype=torch.float16,
                                                 device=cuda), k_scale=KS)
    kept = torch.empty(3, hkv, keep, dtype=torch.int32, device=cuda)
    want = PA.paged_attention_sparse(qt, kc, vc, bnd, tt, lt, keep, selected=kept, k_scale=KS,
                                     v_scale=VS)
    tables, slens, pages = PA.select_pages(qt, kc, bnd, tt, lt, keep)
    assert torch.equal(pages, kept)
    one = lambda x: x.view(len(k) * hkv, 1, bs // 16, 9 * D)
    got = PA.paged_attention_q4(qt.view(3 * hkv, hq // hkv, D), one(kc), one(vc), tables, slens, KS, VS)
    assert torch.equal(got.view_as(want), want)
