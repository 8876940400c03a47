"""Page bounds and sparse decode attention on the GPU against their statement
in 64 bits (_sparseref.py): bounds and kept pages exactly, outputs within the
bound of the attention over those pages."""
import math

import numpy as np
import pytest

import _q4ref as R
import _sparseref as S
from _helpers import check_close
from xllms_b200 import _native
from xllms_b200 import operator_api as PA

pytestmark = pytest.mark.gpu
KS, VS = 0.011, 0.0073


def _t(x, dev):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x)).to(dev)


def _case(seed, lens, hq, hkv, D, bs, dtype=np.float16, mb=None, extra=3):
    rng = np.random.default_rng(seed)
    lens = np.asarray(lens, np.int32)
    pages = -(-lens // bs)
    nb = int(pages.sum()) + extra
    mb = max(1, int(pages.max())) if mb is None else mb
    k = (rng.standard_normal((nb, hkv, bs, D)) + rng.standard_normal((nb, hkv, 1, D))).astype(dtype)
    v = rng.standard_normal((nb, hkv, bs, D)).astype(dtype)
    table = np.full((len(lens), mb), -1, np.int32)
    table[np.arange(mb)[None] < pages[:, None]] = rng.permutation(nb)[:pages.sum()]
    q = rng.standard_normal((len(lens), hq, D)).astype(dtype)
    return q, k, v, table, lens


def _bounds_of(k, table, lens, dtype):
    nb, hkv, _, D = k.shape
    return S.bounds(k, table, lens, 0, np.zeros((nb, hkv, 2, D), dtype), dtype)


# ── bounds ────────────────────────────────────────────────────────────────
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("hkv,D,bs", [(2, 128, 16), (3, 64, 16), (1, 80, 32), (2, 33, 16),
                                      (2, 256, 8), (1, 8, 1), (2, 96, 64), (1, 4, 5), (1, 200, 16)])
def test_bounds_are_exact_over_valid_tokens(cuda, hkv, D, bs, dtype):
    _, k, _, table, lens = _case(D * bs, [0, 1, bs, bs + 1, 7 * bs - 1, 300], hkv, hkv, D, bs, dtype)
    rng = np.random.default_rng(0)
    flat = k.reshape(-1, D)
    for value in (np.nan, np.inf, -np.inf):
        flat[rng.integers(0, len(flat), 9), rng.integers(0, D, 9)] = value
    used = np.zeros((len(k), bs), bool)
    for b, n in enumerate(lens):
        used[table[b, np.arange(n) // bs], np.arange(n) % bs] = True
    k = np.where(used[:, None, :, None], k, np.nan).astype(dtype)  # past the lengths: NaN
    old = rng.standard_normal((len(k), hkv, 2, D)).astype(dtype)
    table[5, 2] = -1
    table[4, 1] = len(k)
    kt, tt, lt = _t(k, cuda), _t(table, cuda), _t(lens, cuda)
    for new in (0, 1, 2, bs + 1, 10 ** 6):
        got = PA.page_bounds(kt, tt, lt, _t(old, cuda), num_new_tokens=new)
        np.testing.assert_array_equal(got.cpu().numpy(), S.bounds(k, table, lens, new, old, dtype))
    assert PA.device_status(clear=True) == _native.NXT_PA_DEV_BAD_PAGE


@pytest.mark.parametrize("hkv,D,bs", [(2, 128, 16), (1, 16, 16), (3, 80, 32), (2, 256, 16)])
def test_bounds_of_4_bit_keys_are_those_of_the_rows_read_back(cuda, hkv, D, bs):
    import torch
    _, k, _, table, lens = _case(D, [0, 1, 16, 45, 200], hkv, hkv, D, bs)
    pool = torch.zeros(PA.q4_pool_shape(len(k), hkv, bs, D), dtype=torch.uint8, device=cuda)
    slots = torch.arange(len(k) * bs, device=cuda)
    rows = _t(k.transpose(0, 2, 1, 3).reshape(-1, hkv, D), cuda)
    PA.reshape_and_cache_q4(rows, rows, pool, pool.clone(), slots, KS, VS)
    back, _ = PA.read_cache_q4(pool, pool, slots, KS, VS)
    back = back.cpu().numpy().reshape(len(k), bs, hkv, D).transpose(0, 2, 1, 3)
    old = np.zeros((len(k), hkv, 2, D), np.float16)
    for new in (0, 3):
        got = PA.page_bounds(pool, _t(table, cuda), _t(lens, cuda), _t(old, cuda),
                             num_new_tokens=new, k_scale=KS)
        np.testing.assert_array_equal(got.cpu().numpy(),
                                      S.bounds(back, table, lens, new, old, np.float16))


def test_strided_keys_and_unaligned_rows(cuda):
    """Pools with padded pages and bases off the wide boundary give the same bounds."""
    import torch
    hkv, D, bs = 2, 64, 16
    _, k, _, table, lens = _case(77, [100, 33], hkv, hkv, D, bs)
    want = _bounds_of(k, table, lens, np.float16)
    nb = len(k)
    tt, lt = _t(table, cuda), _t(lens, cuda)
    for lead, pad in ((0, 8), (1, 3)):
        big = torch.full((lead + nb * (hkv * bs * D + pad),), float("nan"), dtype=torch.float16,
                         device=cuda)
        big[lead:].view(nb, -1)[:, :hkv * bs * D] = _t(k.reshape(nb, -1), cuda)
        bnd = torch.zeros(nb, hkv, 2, D, dtype=torch.float16, device=cuda)
        rc = _native.xpa().nxt_page_bounds(
            bnd.data_ptr(), big.data_ptr() + 2 * lead, tt.data_ptr(), lt.data_ptr(), 2, hkv, D, table.shape[1], bs, 2, hkv * bs * D + pad,
            bs * D, nb, 0, None, torch.cuda.current_stream().cuda_stream)
        assert rc == _native.NXT_PA_OK
        np.testing.assert_array_equal(bnd.cpu().numpy(), want)


# ── selection ─────────────────────────────────────────────────────────────
SHAPES = [
    # hq, hkv, D, bs, dtype
    (8, 2, 128, 16, np.float16), (32, 4, 64, 16, np.float16), (12, 12, 64, 16, np.float32),
    (20, 2, 256, 16, np.float16), (5, 1, 80, 32, np.float16), (3, 1, 36, 8, np.float16),
    (34, 1, 40, 16, np.float16), (6, 2, 33, 16, np.float32), (16, 1, 24, 4, np.float16),
    (32, 2, 256, 16, np.float16), (20, 1, 64, 16, np.float16), (33, 1, 128, 16, np.float16),
]


def _select(cuda, q, bnd, table, lens, k, keep, sink, recent, scale=None, status=None):
    return PA.select_pages(_t(q, cuda), _t(k, cuda), _t(bnd, cuda), _t(table, cuda),
                           _t(lens, cuda), keep, sink_pages=sink, recent_pages=recent, scale=scale,
                           device_status=status)


@pytest.mark.parametrize("keep,sink,recent", [(1, 0, 1), (6, 1, 2), (17, 0, 17), (40, 3, 1)])
@pytest.mark.parametrize("hq,hkv,D,bs,dtype", SHAPES)
def test_kept_pages_are_exact(cuda, hq, hkv, D, bs, dtype, keep, sink, recent):
    lens = [0, 1, bs, keep * bs, keep * bs + 1, 61 * bs - 3, 300 * bs]
    q, k, _, table, lens = _case(hq * D + keep, lens, hq, hkv, D, bs, dtype)
    bnd = _bounds_of(k, table, lens, dtype)
    tables, slens, pages = _select(cuda, q, bnd, table, lens, k, keep, sink, recent)
    want = S.select(q, bnd, table, lens, bs, keep, sink, recent, 1.0, len(k))
    np.testing.assert_array_equal(pages.cpu().numpy(), want)
    ids = np.where(want >= 0, np.take_along_axis(table[:, None], np.maximum(want, 0), 2) * hkv
                   + np.arange(hkv)[None, :, None], -1)
    np.testing.assert_array_equal(tables.cpu().numpy(), ids.reshape(-1, keep))
    n_pages = -(-lens // bs)
    short = np.where((want == (n_pages - 1)[:, None, None]).any(-1), (n_pages * bs - lens)[:, None], 0)
    np.testing.assert_array_equal(slens.cpu().numpy().reshape(len(lens), hkv),
                                  (want >= 0).sum(-1) * bs - short)


@pytest.mark.parametrize("scale", [-0.3, 0.0])
def test_other_signs_of_the_scale(cuda, scale):
    q, k, _, table, lens = _case(3, [2000, 700], 8, 2, 128, 16)
    bnd = _bounds_of(k, table, lens, np.float16)
    _, _, pages = _select(cuda, q, bnd, table, lens, k, 9, 1, 2, scale)
    np.testing.assert_array_equal(pages.cpu().numpy(),
                                  S.select(q, bnd, table, lens, 16, 9, 1, 2, scale, len(k)))


@pytest.mark.parametrize("dtype,n_pages", [(np.float16, 200), (np.float16, 3001),
                                           (np.float32, 1500), (np.float16, 12001)])
def test_ties_go_to_the_earlier_page(cuda, dtype, n_pages):
    """Few distinct bounds, so that hundreds or thousands of pages tie at the border."""
    rng = np.random.default_rng(n_pages)
    hq, hkv, D, bs, nb = 4, 2, 16, 1, 50
    few = rng.standard_normal((3, hkv, 2, D)).astype(dtype)
    few[:, :, 1] = np.abs(few[:, :, 1])
    few[:, :, 0] = -np.abs(few[:, :, 0])
    bnd = few[rng.integers(0, 3, nb)]
    table = rng.integers(0, nb, (2, n_pages)).astype(np.int32)
    lens = np.array([n_pages, n_pages // 2], np.int32)
    q = rng.standard_normal((2, hq, D)).astype(dtype)
    k = np.zeros((nb, hkv, bs, D), dtype)
    for keep, sink, recent in ((70, 1, 2), (n_pages // 2, 0, 1)):
        _, _, pages = _select(cuda, q, bnd, table, lens, k, keep, sink, recent)
        np.testing.assert_array_equal(
            pages.cpu().numpy(), S.select(q, bnd, table, lens, bs, keep, sink, recent, 1.0, nb))
    q[:] = 0  # every score is 0
    _, _, pages = _select(cuda, q, bnd, table, lens, k, 70, 1, 2)
    np.testing.assert_array_equal(pages.cpu().numpy(),
                                  S.select(q, bnd, table, lens, bs, 70, 1, 2, 1.0, nb))


def test_scores_closer_than_fp32_tells_apart(cuda):
    """Pages whose scores differ by less than an fp32 sum of them resolves are still ordered."""
    rng = np.random.default_rng(8)
    hq, hkv, D, bs, n = 2, 1, 128, 1, 900
    base = rng.standard_normal((1, hkv, 2, D)) * 4
    bnd = np.sort(np.broadcast_to(base, (n, hkv, 2, D)), axis=2).astype(np.float16)
    # tiny steps in a channel whose query is small
    bnd[:, 0, 1, 7] = (rng.permutation(n) * 2.0 ** -18).astype(np.float16)
    bnd[:, 0, 0, 7] = 0
    q = rng.standard_normal((1, hq, D)).astype(np.float16)
    q[:, :, 7] = 2.0 ** -6
    table = np.arange(n, dtype=np.int32)[None]
    lens = np.array([n], np.int32)
    _, _, pages = _select(cuda, q, bnd, table, lens, np.zeros((n, hkv, bs, D), np.float16), 100, 0, 1)
    np.testing.assert_array_equal(pages.cpu().numpy(),
                                  S.select(q, bnd, table, lens, bs, 100, 0, 1, 1.0, n))


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_extreme_bounds_and_queries(cuda, dtype):
    """The largest finite values (their fp32 scores overflow), NaN and infinite queries."""
    rng = np.random.default_rng(1)
    hq, hkv, D, bs, n = 4, 2, 32, 1, 500
    big = float(np.finfo(dtype).max)
    bnd = np.sort(rng.choice([-big, -1.0, 0.0, 1.0, big / 2, big], (n, hkv, 2, D)), 2).astype(dtype)
    q = rng.choice([-big, -2.0, 0.0, 0.5, big], (1, hq, D)).astype(dtype)
    q[0, 0, 0], q[0, 1, 1], q[0, 2, 2] = np.nan, np.inf, -np.inf
    table = rng.permutation(n).astype(np.int32)[None]
    lens = np.array([n], np.int32)
    _, _, pages = _select(cuda, q, bnd, table, lens, np.zeros((n, hkv, bs, D), dtype), 60, 0, 1)
    got = pages.cpu().numpy()
    # 64-bit sums of such terms round too: only sums that are exact are compared
    assert (got >= 0).all() and (np.diff(got) > 0).all()
    if dtype == np.float16:
        np.testing.assert_array_equal(got, S.select(q, bnd, table, lens, bs, 60, 0, 1, 1.0, n))


def test_bounds_that_no_call_wrote_stay_in_range(cuda):
    """NaN and infinite bounds select some pages, in order, and nothing out of range."""
    import torch
    rng = np.random.default_rng(4)
    bnd = rng.integers(0, 65536, (400, 2, 2, 128)).astype(np.uint16).view(np.float16)
    table = rng.permutation(400).astype(np.int32)[None]
    lens = np.array([400 * 16], np.int32)
    q = rng.standard_normal((1, 8, 128)).astype(np.float16)
    _, slens, pages = _select(cuda, q, bnd, table, lens, np.zeros((400, 2, 16, 128), np.float16),
                              50, 1, 1)
    got = pages.cpu().numpy()
    assert (got >= 0).all() and (got < 400).all() and (np.diff(got) > 0).all()
    assert (slens == 800).all()
    torch.cuda.synchronize()


def test_masked_pages_are_never_kept(cuda):
    import torch
    q, k, _, table, lens = _case(13, [1000, 100, 900, 640], 8, 2, 128, 16)
    bnd = _bounds_of(k, table, lens, np.float16)
    table[0, [0, 7, 30]] = -1
    table[0, 62] = len(k)       # the last, partial page
    table[1, 2] = -5
    table[2, :] = -1
    lens = lens.copy()
    lens[3] = 10 ** 8
    table[3, 40:] = -1
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    _, slens, pages = _select(cuda, q, bnd, table, lens, k, 12, 1, 2, status=status)
    want = S.select(q, bnd, table, lens, 16, 12, 1, 2, 1.0, len(k))
    np.testing.assert_array_equal(pages.cpu().numpy(), want)
    assert int(status) == _native.NXT_PA_DEV_BAD_PAGE | _native.NXT_PA_DEV_SEQ_CLAMPED
    assert slens.view(4, 2)[2].eq(0).all()


# ── attention ─────────────────────────────────────────────────────────────
def _sparse_reference(q, k, v, kept, table, lens, scale):
    """64-bit attention over the kept pages of each KV head; rows of heads as tables."""
    B, Hq, D = q.shape
    nb, hkv, bs, _ = k.shape
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    G = Hq // hkv
    for b in range(B):
        for h in range(hkv):
            at = kept[b, h][kept[b, h] >= 0]
            tok = (at[:, None] * bs + np.arange(bs)).ravel()
            tok = tok[tok < lens[b]]
            if not len(tok):
                continue
            page = table[b, tok // bs]
            rows = [x[page, h, tok % bs][None, None] for x in (k, v)]
            o, e = R.attention(q[b:b + 1, h * G:(h + 1) * G], *rows, np.zeros((1, 1), np.int32),
                               [len(tok)], scale)
            out[b, h * G:(h + 1) * G], bound[b, h * G:(h + 1) * G] = o[0], e[0]
    return out, bound


@pytest.mark.parametrize("hq,hkv,D,bs,dtype", SHAPES)
def test_sparse_attention_is_attention_over_the_kept_pages(cuda, hq, hkv, D, bs, dtype):
    import torch
    keep, sink, recent = 11, 1, 2
    lens = [0, 1, keep * bs, 40 * bs + 1, 200 * bs - 1]
    q, k, v, table, lens = _case(hq + D, lens, hq, hkv, D, bs, dtype)
    bnd = _bounds_of(k, table, lens, dtype)
    kept = torch.full((len(lens), hkv, keep), -7, dtype=torch.int32, device=cuda)
    ws = torch.empty(PA.sparse_workspace_size(len(lens), hq, D, hkv, table.shape[1], keep, bs,
                                              np.dtype(dtype).itemsize), dtype=torch.uint8,
                     device=cuda)
    args = (_t(q, cuda), _t(k, cuda), _t(v, cuda), _t(bnd, cuda), _t(table, cuda), _t(lens, cuda))
    out = PA.paged_attention_sparse(*args, keep, sink_pages=sink, recent_pages=recent,
                                    selected=kept, workspace=ws)
    want = S.select(q, bnd, table, lens, bs, keep, sink, recent, 1.0, len(k))
    np.testing.assert_array_equal(kept.cpu().numpy(), want)
    ref, _ = _sparse_reference(q, k.astype(np.float64), v.astype(np.float64), want, table, lens,
                               1 / math.sqrt(D))
    check_close(out, ref)  # the tolerance of the attention that runs over the pages
    assert not out[0].any()
    own = PA.paged_attention_sparse(*args, keep, sink_pages=sink, recent_pages=recent)
    assert torch.equal(out, own)
    with pytest.raises(PA.PagedAttentionError):
        PA.paged_attention_sparse(*args, keep, sink_pages=sink, recent_pages=recent,
                                  workspace=ws[:256])


@pytest.mark.parametrize("hq,hkv,D,bs", [(8, 2, 128, 16), (32, 2, 64, 16), (5, 1, 80, 32),
                                         (6, 3, 256, 16)])
def test_sparse_attention_over_4_bit_pools(cuda, hq, hkv, D, bs):
    import torch
    keep, sink, recent = 7, 1, 1
    q, k, v, table, lens = _case(D + 1, [0, 5, 7 * bs, 33 * bs + 2, 150 * bs], hq, hkv, D, bs)
    kc = torch.zeros(PA.q4_pool_shape(len(k), hkv, bs, D), dtype=torch.uint8, device=cuda)
    vc = torch.zeros_like(kc)
    slots = torch.arange(len(k) * bs, device=cuda)
    as_rows = lambda x: _t(x.transpose(0, 2, 1, 3).reshape(-1, hkv, D), cuda)
    PA.reshape_and_cache_q4(as_rows(k), as_rows(v), kc, vc, slots, KS, VS)
    tt, lt = _t(table, cuda), _t(lens, cuda)
    bnd = PA.page_bounds(kc, tt, lt, torch.zeros(len(k), hkv, 2, D, dtype=torch.float16,
                                                 device=cuda), k_scale=KS)
    kept = torch.empty(len(lens), hkv, keep, dtype=torch.int32, device=cuda)
    out = PA.paged_attention_sparse(_t(q, cuda), kc, vc, bnd, tt, lt, keep, sink_pages=sink,
                                    recent_pages=recent, selected=kept, k_scale=KS, v_scale=VS)
    want = S.select(q, bnd.cpu().numpy(), table, lens, bs, keep, sink, recent, 1.0, len(k))
    np.testing.assert_array_equal(kept.cpu().numpy(), want)
    kv = [R.values(*R.unpack(p.cpu().numpy(), i), s) for p, i, s in ((kc, True, KS), (vc, False, VS))]
    ref, bound = _sparse_reference(q, *kv, want, table, lens, 1 / math.sqrt(D))
    assert np.max(np.abs(out.double().cpu().numpy() - ref) / np.maximum(bound, 1e-30)) <= 1.0


def test_everything_kept_is_plain_attention(cuda):
    import torch
    q, k, v, table, lens = _case(15, [1, 500, 333], 32, 8, 128, 16)
    bnd = np.full((len(k), 8, 2, 128), np.nan, np.float16)  # not read
    args = [_t(x, cuda) for x in (q, k, v)]
    tt, lt = _t(table, cuda), _t(lens, cuda)
    full = PA.paged_attention(*args, tt, lt)
    out = PA.paged_attention_sparse(*args, _t(bnd, cuda), tt, lt, 32)
    check_close(out, full.double().cpu().numpy())


def test_selected_tables_serve_other_attention_calls(cuda):
    """nxt_select_pages' tables over the fp16 pool, and over an fp8 copy of it."""
    import torch
    hq, hkv, D, bs, keep = 8, 2, 128, 16, 9
    q, k, v, table, lens = _case(16, [700, 90], hq, hkv, D, bs)
    bnd = _bounds_of(k, table, lens, np.float16)
    kt, vt = _t(k, cuda), _t(v, cuda)
    tables, slens, pages = _select(cuda, q, bnd, table, lens, k, keep, 1, 1)
    qv = _t(q, cuda).view(2 * hkv, hq // hkv, D)
    one = lambda x: x.view(-1, 1, bs, D)
    want = PA.paged_attention_sparse(_t(q, cuda), kt, vt, _t(bnd, cuda), _t(table, cuda),
                                     _t(lens, cuda), keep, sink_pages=1)
    got = PA.paged_attention(qv, one(kt), one(vt), tables, slens)
    assert torch.equal(got.view_as(want), want)
    k8, v8 = (x.to(torch.float8_e4m3fn).view(torch.uint8) for x in (kt, vt))
    got8 = PA.paged_attention_fp8(qv, one(k8), one(v8), tables, slens, "e4m3", 1.0, 1.0)
    ref, _ = _sparse_reference(q, *(x.view(torch.float8_e4m3fn).double().cpu().numpy()
                                    for x in (k8, v8)), pages.cpu().numpy(), table, lens,
                               1 / math.sqrt(D))
    check_close(got8.view_as(want), ref)


def test_padded_pages_and_one_kv_head(cuda):
    """Pools whose pages are padded by whole heads; any page stride with one KV head."""
    import torch
    for hkv, pad in ((2, 1), (1, 0)):
        hq, D, bs, keep = 4 * hkv, 64, 16, 6
        q, k, v, table, lens = _case(17 + hkv, [400, 77], hq, hkv, D, bs)
        bnd = _bounds_of(k, table, lens, np.float16)
        want = S.select(q, bnd, table, lens, bs, keep, 0, 1, 1.0, len(k))
        ref, _ = _sparse_reference(q, k.astype(np.float64), v.astype(np.float64), want, table, lens,
                                   0.125)
        extra = pad * bs * D if hkv > 1 else 40
        big = torch.zeros(2, len(k), hkv * bs * D + extra, dtype=torch.float16, device=cuda)
        big[0, :, :hkv * bs * D] = _t(k.reshape(len(k), -1), cuda)
        big[1, :, :hkv * bs * D] = _t(v.reshape(len(k), -1), cuda)
        out = torch.empty(q.shape, dtype=torch.float16, device=cuda)
        ins = [_t(q, cuda), big[0], big[1], _t(bnd, cuda), _t(table, cuda), _t(lens, cuda)]
        rc = _native.xpa().nxt_paged_attention_sparse_ex(
            out.data_ptr(), *(x.data_ptr() for x in ins), None, 2, hq, D, hkv, 0.125,
            table.shape[1], bs, 2, hkv * bs * D + extra, bs * D, len(k), keep, 0, 1, None, 0, None,
            torch.cuda.current_stream().cuda_stream)
        assert rc == _native.NXT_PA_OK
        check_close(out, ref)


def test_graph_replays_and_streams_give_the_same_bits(cuda):
    import torch
    q, k, v, table, lens = _case(19, [4000, 100, 1700], 32, 8, 128, 16)
    bnd = _bounds_of(k, table, lens, np.float16)
    args = [_t(x, cuda) for x in (q, k, v, bnd, table, lens)]
    want = PA.paged_attention_sparse(*args, 20)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    out = torch.empty_like(want)
    with torch.cuda.stream(side):
        PA.paged_attention_sparse(*args, 20, out=out)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            PA.page_bounds(args[1], args[4], args[5], args[3], num_new_tokens=1)
            PA.paged_attention_sparse(*args, 20, out=out)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    # new queries reach the replayed graph
    args[0].neg_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, PA.paged_attention_sparse(*args, 20))


def test_decode_steps_with_bounds_kept_up_to_date(cuda):
    """Append, refresh the newest page's bounds, attend: the bounds stay those of the whole cache."""
    import torch
    hq, hkv, D, bs, n0, keep = 8, 2, 64, 16, 150, 5
    rng = np.random.default_rng(23)
    nb = 14
    k = torch.zeros(nb, hkv, bs, D, dtype=torch.float16, device=cuda)
    v = torch.zeros_like(k)
    bnd = torch.full((nb, hkv, 2, D), 99.0, dtype=torch.float16, device=cuda)
    order = rng.permutation(nb)
    table = _t(order[None].astype(np.int32), cuda)
    slot = order[np.arange(nb * bs) // bs] * bs + np.arange(nb * bs) % bs
    rows = _t(rng.standard_normal((2, nb * bs, hkv, D)).astype(np.float16), cuda)
    PA.reshape_and_cache(rows[0, :n0], rows[1, :n0], k, v, _t(slot[:n0], cuda))
    PA.page_bounds(k, table, _t(np.array([n0], np.int32), cuda), bnd)
    for n in range(n0 + 1, n0 + 20):
        PA.reshape_and_cache(rows[0, n - 1:n], rows[1, n - 1:n], k, v, _t(slot[n - 1:n], cuda))
        lens = np.array([n], np.int32)
        PA.page_bounds(k, table, _t(lens, cuda), bnd, num_new_tokens=1)
        q = rng.standard_normal((1, hq, D)).astype(np.float16)
        kept = torch.empty(1, hkv, keep, dtype=torch.int32, device=cuda)
        out = PA.paged_attention_sparse(_t(q, cuda), k, v, bnd, table, _t(lens, cuda), keep,
                                        sink_pages=1, selected=kept)
        kn, vn = k.cpu().numpy(), v.cpu().numpy()
        tab = table.cpu().numpy()
        whole = S.bounds(kn, tab, lens, 0, np.full(bnd.shape, 99, np.float16), np.float16)
        np.testing.assert_array_equal(bnd.cpu().numpy(), whole)
        want = S.select(q, whole, tab, lens, bs, keep, 1, 1, 1.0, nb)
        np.testing.assert_array_equal(kept.cpu().numpy(), want)
        ref, _ = _sparse_reference(q, kn.astype(np.float64), vn.astype(np.float64), want, tab, lens,
                                   1 / math.sqrt(D))
        check_close(out, ref)


@pytest.mark.parametrize("hq,hkv,D,bs,dtype", [
    (32, 4, 128, 32, np.float16), (10, 5, 64, 64, np.float16), (16, 2, 256, 48, np.float16),
    (20, 1, 128, 64, np.float16), (32, 2, 208, 64, np.float16), (48, 3, 144, 16, np.float32),
    (13, 1, 256, 32, np.float16), (22, 1, 64, 32, np.float32)])
def test_long_pages_and_wide_groups(cuda, hq, hkv, D, bs, dtype):
    """Pages that attention takes in pieces, groups that it takes in parts; with
    pages that are not there, and with the number of blocks unknown."""
    keep, sink, recent = 6, 1, 1
    lens = [0, 1, bs - 1, bs + 17, 4 * bs, 23 * bs + 5, 40 * bs]
    q, k, v, table, lens = _case(hq + D + bs, lens, hq, hkv, D, bs, dtype)
    bnd = _bounds_of(k, table, lens, dtype)
    table[5, 2:20:3] = -1
    table[6, 1:30:2] = len(k) + 5
    want = S.select(q, bnd, table, lens, bs, keep, sink, recent, 1.0, len(k))
    ref, _ = _sparse_reference(q, k.astype(np.float64), v.astype(np.float64), want, table, lens,
                               1 / math.sqrt(D))
    import torch
    args = [_t(x, cuda) for x in (q, k, v, bnd, table, lens)]
    kept = torch.empty(len(lens), hkv, keep, dtype=torch.int32, device=cuda)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    ws = torch.empty(PA.sparse_workspace_size(len(lens), hq, D, hkv, table.shape[1], keep, bs,
                                              np.dtype(dtype).itemsize), dtype=torch.uint8,
                     device=cuda)
    out = PA.paged_attention_sparse(*args, keep, sink_pages=sink, recent_pages=recent,
                                    selected=kept, workspace=ws, device_status=status)
    np.testing.assert_array_equal(kept.cpu().numpy(), want)
    assert int(status) == _native.NXT_PA_DEV_BAD_PAGE
    check_close(out, ref)
    args[4][args[4] > len(k)] = -1  # the number of blocks bounds no id now
    out = PA.paged_attention_sparse(*args, keep, sink_pages=sink, recent_pages=recent,
                                    selected=kept, num_blocks=-1)
    np.testing.assert_array_equal(kept.cpu().numpy(), want)
    check_close(out, ref)


@pytest.mark.parametrize("hkv,pad", [(2, 2), (1, 16), (1, 8)])
def test_long_pages_of_padded_pools(cuda, hkv, pad):
    """Page strides that hold a whole number of 16-token pieces, and one that does not."""
    import torch
    hq, D, bs, keep = 4 * hkv, 64, 32, 5
    q, k, v, table, lens = _case(80 + pad, [700, 77, 33], hq, hkv, D, bs)
    bnd = _bounds_of(k, table, lens, np.float16)
    want = S.select(q, bnd, table, lens, bs, keep, 0, 1, 1.0, len(k))
    ref, _ = _sparse_reference(q, k.astype(np.float64), v.astype(np.float64), want, table, lens,
                               0.125)
    extra = pad * bs * D if hkv > 1 else pad * D
    big = torch.zeros(2, len(k), hkv * bs * D + extra, dtype=torch.float16, device=cuda)
    big[0, :, :hkv * bs * D] = _t(k.reshape(len(k), -1), cuda)
    big[1, :, :hkv * bs * D] = _t(v.reshape(len(k), -1), cuda)
    out = torch.empty(q.shape, dtype=torch.float16, device=cuda)
    ins = [_t(q, cuda), big[0], big[1], _t(bnd, cuda), _t(table, cuda), _t(lens, cuda)]
    rc = _native.xpa().nxt_paged_attention_sparse_ex(
        out.data_ptr(), *(x.data_ptr() for x in ins), None, 3, hq, D, hkv, 0.125, table.shape[1],
        bs, 2, hkv * bs * D + extra, bs * D, len(k), keep, 0, 1, None, 0, None,
        torch.cuda.current_stream().cuda_stream)
    assert rc == _native.NXT_PA_OK
    check_close(out, ref)


def test_more_new_tokens_than_a_cache_can_hold(cuda):
    _, k, _, table, lens = _case(90, [70, 5], 2, 2, 16, 1)
    old = np.zeros((len(k), 2, 2, 16), np.float16)
    got = PA.page_bounds(_t(k, cuda), _t(table, cuda), _t(lens, cuda), _t(old, cuda),
                         num_new_tokens=2 ** 31 - 1)
    np.testing.assert_array_equal(got.cpu().numpy(),
                                  S.bounds(k, table, lens, 0, old, np.float16))


def test_host_workspaces_and_status_words_are_refused(cuda):
    import torch
    q, k, v, table, lens = _case(91, [300], 8, 2, 64, 16)
    bnd = _bounds_of(k, table, lens, np.float16)
    args = [_t(x, cuda) for x in (q, k, v, bnd, table, lens)]
    pool = torch.zeros(PA.q4_pool_shape(len(k), 2, 16, 64), dtype=torch.uint8, device=cuda)
    host = torch.zeros(1 << 20, dtype=torch.uint8)
    word = torch.zeros(1, dtype=torch.int32)
    for bad in (dict(workspace=host), dict(device_status=word),
                dict(device_status=word.to(cuda).float())):
        with pytest.raises(PA.PagedAttentionError):
            PA.paged_attention_sparse(*args, 4, **bad)
        with pytest.raises(PA.PagedAttentionError):
            PA.paged_attention_q4(args[0], pool, pool, args[4], args[5], KS, VS, **bad)
        if "device_status" not in bad:
            continue
        with pytest.raises(PA.PagedAttentionError):
            PA.select_pages(args[0], args[1], *args[3:], 4, **bad)
        with pytest.raises(PA.PagedAttentionError):
            PA.page_bounds(args[1], args[4], args[5], args[3], **bad)
        rows = torch.zeros(1, 2, 64, dtype=torch.float16, device=cuda)
        slots = torch.zeros(1, dtype=torch.int64, device=cuda)
        with pytest.raises(PA.PagedAttentionError):
            PA.paged_attention_q4_append(args[0], pool, pool, args[4], args[5], rows, rows, slots,
                                         KS, VS, **bad)
