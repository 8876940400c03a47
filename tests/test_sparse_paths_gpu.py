"""Sparse decode attention, and its selection, on the paths that longer and odder
calls take."""
import math
import threading

import numpy as np
import pytest

import _q4ref as R
import _sparseref as S
from _helpers import check_close
from test_sparse_gpu import _bounds_of, _case, _sparse_reference, _t
from xllms_b200 import _native
from xllms_b200 import operator_api as PA

pytestmark = pytest.mark.gpu
KS, VS = 0.011, 0.0073


def _guarded(cuda, *sizes):
    """A workspace of exactly the size asked for, with a guard behind it."""
    import torch
    need = PA.sparse_workspace_size(*sizes)
    buf = torch.full((need + 256,), 0x5a, dtype=torch.uint8, device=cuda)
    return buf[:need], buf[need:]


def _unused(table, lens, nb, bs):
    """[nb, bs]: slots that hold no token of any sequence."""
    free = np.ones((nb, bs), bool)
    for b, n in enumerate(lens):
        at = np.arange(n)
        free[table[b, at // bs], at % bs] = False
    return free


@pytest.mark.parametrize("hq,hkv,D,bs,keep", [
    (20, 5, 112, 16, 64), (8, 1, 208, 64, 24), (13, 1, 256, 32, 40), (6, 2, 32, 16, 100),
    (12, 1, 48, 48, 30), (16, 2, 128, 16, 200), (4, 1, 16, 16, 256)])
def test_split_rows(cuda, hq, hkv, D, bs, keep):
    """More than 512 kept tokens: some rows in one partition, some in several.
    What lies behind a sequence's last token is NaN and reaches nothing."""
    import torch
    assert keep * bs > 512
    lens = [keep * bs, 0, 5, 3 * keep * bs + 7, 40, 2 * keep * bs - 1, keep * bs // 2 + 1]
    q, k, v, table, lens = _case(hq + D + keep, lens, hq, hkv, D, bs)
    bnd = _bounds_of(k, table, lens, np.float16)
    want = S.select(q, bnd, table, lens, bs, keep, 1, 2, 1.0, len(k))
    ref, _ = _sparse_reference(q, k.astype(np.float64), v.astype(np.float64), want, table, lens,
                               1 / math.sqrt(D))
    free = np.broadcast_to(_unused(table, lens, len(k), bs)[:, None], k.shape[:3])
    k[free] = np.nan
    v[free] = np.nan
    ws, guard = _guarded(cuda, len(lens), hq, D, hkv, table.shape[1], keep, bs, 2)
    kept = torch.empty(len(lens), hkv, keep, dtype=torch.int32, device=cuda)
    args = [_t(x, cuda) for x in (q, k, v, bnd, table, lens)]
    out = PA.paged_attention_sparse(*args, keep, sink_pages=1, recent_pages=2, selected=kept,
                                    workspace=ws)
    np.testing.assert_array_equal(kept.cpu().numpy(), want)
    assert (guard == 0x5a).all()
    check_close(out, ref)
    assert torch.equal(out, PA.paged_attention_sparse(*args, keep, sink_pages=1, recent_pages=2))


@pytest.mark.parametrize("hq,hkv,D,bs,keep", [
    (8, 2, 128, 16, 64), (32, 2, 64, 16, 256), (5, 1, 80, 32, 40), (10, 1, 256, 16, 64)])
def test_split_rows_of_4_bit_pools(cuda, hq, hkv, D, bs, keep):
    """The same over 4-bit pools; the unused slots' scale bytes are NaN."""
    import torch
    lens = [keep * bs, 0, 5, 3 * keep * bs + 7, 40, 2 * keep * bs - 1]
    rng = np.random.default_rng(D + keep)
    q, k, _, table, lens = _case(D + keep, lens, hq, hkv, D, bs)
    nb = len(k)
    c = rng.integers(0, 16, (2, nb, hkv, bs, D)).astype(np.uint8)
    sb = rng.integers(30, 70, (2, nb, hkv, bs, D // 16)).astype(np.uint8)
    kv = [R.values(c[i], sb[i], s) for i, s in enumerate((KS, VS))]
    free = np.broadcast_to(_unused(table, lens, nb, bs)[:, None], (nb, hkv, bs))
    sb[:, free] = 0x7f
    kc, vc = (_t(R.pack(c[i], sb[i], i == 0), cuda) for i in (0, 1))
    tt, lt = _t(table, cuda), _t(lens, cuda)
    bnd = PA.page_bounds(kc, tt, lt, torch.zeros(nb, hkv, 2, D, dtype=torch.float16, device=cuda),
                         k_scale=KS)
    want = S.select(q, bnd.cpu().numpy(), table, lens, bs, keep, 1, 1, 1.0, nb)
    ref, bound = _sparse_reference(q, *kv, want, table, lens, 1 / math.sqrt(D))
    ws, guard = _guarded(cuda, len(lens), hq, D, hkv, table.shape[1], keep, bs, 2)
    kept = torch.empty(len(lens), hkv, keep, dtype=torch.int32, device=cuda)
    kind = dict(k_scale=KS, v_scale=VS, sink_pages=1)
    out = PA.paged_attention_sparse(_t(q, cuda), kc, vc, bnd, tt, lt, keep, selected=kept,
                                    workspace=ws, **kind)
    np.testing.assert_array_equal(kept.cpu().numpy(), want)
    assert (guard == 0x5a).all()
    x = out.double().cpu().numpy()
    assert np.isfinite(x).all()
    assert np.max(np.abs(x - ref) / np.maximum(bound, 1e-30)) <= 1.0
    assert torch.equal(out, PA.paged_attention_sparse(_t(q, cuda), kc, vc, bnd, tt, lt, keep, **kind))


@pytest.mark.parametrize("scale", [0.25, 0.0, -0.3])
@pytest.mark.parametrize("hq,hkv,D,bs", [(6, 2, 16, 16), (6, 3, 32, 32), (5, 1, 48, 16),
                                         (20, 5, 112, 16), (13, 1, 256, 16)])
def test_page_kernel_at_small_heads_and_other_scales(cuda, hq, hkv, D, bs, scale):
    keep = 9
    lens = [0, 1, 17, keep * bs, 40 * bs + 3, 77 * bs]
    q, k, v, table, lens = _case(hq * D, lens, hq, hkv, D, bs)
    bnd = _bounds_of(k, table, lens, np.float16)
    want = S.select(q, bnd, table, lens, bs, keep, 1, 1, scale, len(k))
    ref, _ = _sparse_reference(q, k.astype(np.float64), v.astype(np.float64), want, table, lens,
                               scale)
    out = PA.paged_attention_sparse(*(_t(x, cuda) for x in (q, k, v, bnd, table, lens)), keep,
                                    sink_pages=1, scale=scale)
    check_close(out, ref)


@pytest.mark.parametrize("few", [True, False])
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_more_pages_than_shared_memory_holds(cuda, dtype, few):
    """Rows of up to 40001 pages: their keys stay in the workspace. With few
    distinct bounds thousands of pages tie at the border."""
    rng = np.random.default_rng(11)
    hq, hkv, D, bs, n = 4, 2, 16, 1, 40001
    nb = 50 if few else n
    bnd = np.sort(rng.standard_normal((3 if few else nb, hkv, 2, D)), 2).astype(dtype)
    if few:
        bnd = bnd[rng.integers(0, 3, nb)]
    table = rng.integers(0, nb, (3, n)).astype(np.int32)
    table[0, 5::97] = -1
    lens = np.array([n, 32769, 32768], np.int32)
    q = rng.standard_normal((3, hq, D)).astype(dtype)
    args = [_t(x, cuda) for x in (q, np.zeros((nb, hkv, bs, D), dtype), bnd, table, lens)]
    for keep, sink, recent in ((70, 1, 2), (20000, 0, 1)):
        _, slens, pages = PA.select_pages(*args, keep, sink_pages=sink, recent_pages=recent)
        want = S.select(q, bnd, table, lens, bs, keep, sink, recent, 1.0, nb)
        np.testing.assert_array_equal(pages.cpu().numpy(), want)
        np.testing.assert_array_equal(slens.view(3, hkv).cpu().numpy(), (want >= 0).sum(-1))


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


# ── streams, threads and graphs ───────────────────────────────────────────
def _calls(cuda):
    """Sparse calls of each kind whose rows are split, as (call(out, stream), result)."""
    import torch
    calls = []
    for seed, (hq, hkv, D, bs, keep) in enumerate([(32, 8, 128, 16, 90), (20, 5, 112, 16, 80),
                                                   (8, 2, 64, 32, 64)]):
        q, k, v, table, lens = _case(60 + seed, [4000, 100, 2700, 5000], hq, hkv, D, bs)
        bnd = _bounds_of(k, table, lens, np.float16)
        args = [_t(x, cuda) for x in (q, k, v, bnd, table, lens)]

        def call(out, stream=None, args=args, keep=keep):
            return PA.paged_attention_sparse(*args, keep, sink_pages=1, out=out, stream=stream)
        want = call(None)
        kc = torch.zeros(PA.q4_pool_shape(len(k), hkv, bs, D), dtype=torch.uint8, device=cuda)
        vc = torch.zeros_like(kc)
        rows = lambda x: _t(x.transpose(0, 2, 1, 3).reshape(-1, hkv, D), cuda)
        PA.reshape_and_cache_q4(rows(k), rows(v), kc, vc, torch.arange(len(k) * bs, device=cuda), KS,
                                VS)

        def call4(out, stream=None, args=args, keep=keep, kc=kc, vc=vc):
            return PA.paged_attention_sparse(args[0], kc, vc, *args[3:], keep, sink_pages=1,
                                             k_scale=KS, v_scale=VS, out=out, stream=stream)
        calls += [(call, want), (call4, call4(None))]
    torch.cuda.synchronize()
    return calls


def test_streams_and_threads_at_once(cuda):
    import torch
    calls = _calls(cuda)
    got = [[] for _ in range(6)]

    def work(i):
        st = torch.cuda.Stream()
        for n in range(8):
            call, want = calls[(i + n) % len(calls)]
            got[i].append((call(torch.zeros_like(want), st), want))
        st.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(6)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert all(len(g) == 8 and all(torch.equal(a, b) for a, b in g) for g in got)


def test_graphs_side_by_side(cuda):
    """Graphs captured on one stream replayed on several, beside eager calls on
    the stream of their capture."""
    import torch
    calls = _calls(cuda)
    side = torch.cuda.Stream()
    graphs = []
    for call, want in calls[:4]:
        out, graph = torch.zeros_like(want), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            for _ in range(3):
                call(out)
        graphs.append((graph, out, want, torch.cuda.Stream()))
    for _ in range(15):
        for _, out, _, _ in graphs:
            out.zero_()
        torch.cuda.synchronize()
        for graph, _, _, st in graphs:
            with torch.cuda.stream(st):
                graph.replay()
        eager = [(call(torch.zeros_like(want), side), want) for call, want in calls]
        torch.cuda.synchronize()
        assert all(torch.equal(out, want) for _, out, want, _ in graphs)
        assert all(torch.equal(out, want) for out, want in eager)
