"""The 4-bit KV cache on the GPU against its statement in 64 bits (_q4ref.py):
rows written and read back, attention over them, a decode step of both."""
import math
import threading

import numpy as np
import pytest

import _q4ref as R
from xllms_b200 import _native
from xllms_b200 import operator_api as PA

pytestmark = pytest.mark.gpu
KS, VS = 0.011, 0.0073


def _t(x, dev):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x)).to(dev)


def _rows(rng, T, hkv, D):
    """fp16 rows with what a format can trip over: zeros, one large channel,
    ties, tiny and huge values."""
    x = rng.standard_normal((T, hkv, D)).astype(np.float16)
    flat = x.reshape(-1, D)
    flat[0::7, :16] = 0
    flat[1::7, 3] = 300
    flat[2::7] = (rng.integers(-24, 25, flat[2::7].shape) / 4 * 0.011 * 16).astype(np.float16)
    flat[3::11] *= np.float16(2.0 ** -12)
    flat[4::13, 5] = -65504
    flat[5::17, 1] = -0.0
    return x


def _slots(rng, T, nb, bs):
    return rng.permutation(nb * bs)[:T].astype(np.int64)


def _expected(x, ps):
    v = R.values(*R.encode(x, ps), ps)
    return v, np.clip(v, -65504, 65504).astype(np.float32).astype(np.float16)


@pytest.mark.parametrize("T,hkv,D,bs", [(1, 1, 16, 16), (3, 2, 48, 32), (64, 8, 128, 16),
                                        (130, 3, 64, 16), (37, 5, 80, 48), (70, 2, 256, 64),
                                        (33, 1, 208, 16)])
def test_write_stores_the_formats_bytes_and_read_returns_its_values(cuda, T, hkv, D, bs):
    import torch
    rng = np.random.default_rng(T * D)
    nb = -(-T // bs) + 2
    k, v = _rows(rng, T, hkv, D), _rows(rng, T, hkv, D)
    slots = _slots(rng, T, nb, bs)
    skip = slots.copy()
    skip[1::5] = -1 - skip[1::5]
    fill = rng.integers(0, 256, (2,) + PA.q4_pool_shape(nb, hkv, bs, D)).astype(np.uint8)
    kc, vc = _t(fill[0], cuda), _t(fill[1], cuda)
    PA.reshape_and_cache_q4(_t(k, cuda), _t(v, cuda), kc, vc, _t(skip, cuda), KS, VS)
    for pool, rows, ps, is_key, was in ((kc, k, KS, True, fill[0]), (vc, v, VS, False, fill[1])):
        codes, sb = R.unpack(was, is_key)
        codes, sb = codes.astype(np.uint8), sb.copy()
        c, s = R.encode(rows, ps)
        for t in range(T):
            if skip[t] >= 0:
                codes[skip[t] // bs, :, skip[t] % bs] = c[t]
                sb[skip[t] // bs, :, skip[t] % bs] = s[t]
        got = pool.cpu().numpy()
        gc, gs = R.unpack(got, is_key)
        np.testing.assert_array_equal(gs, sb)
        np.testing.assert_array_equal(gc, codes)  # what no token was written to stays
    at = np.concatenate([skip, skip[:3], [nb * bs, 2 ** 40]])
    rk, rv = PA.read_cache_q4(kc, vc, _t(at, cuda), KS, VS)
    for got, rows, ps in ((rk, k, KS), (rv, v, VS)):
        got = got.cpu().numpy()
        want = _expected(rows, ps)[1]
        want[skip < 0] = 0
        want = np.concatenate([want, want[:3], np.zeros((2,) + want.shape[1:], want.dtype)])
        # one fp32 rounding before the fp16 one: at most one fp16 step apart
        np.testing.assert_allclose(got.astype(np.float64), want.astype(np.float64),
                                   rtol=2.0 ** -10, atol=2.0 ** -24)
        assert np.mean(got != want) < 1e-3
    torch.cuda.synchronize()


@pytest.mark.parametrize("ps", [1.0, 0.37, 2.0 ** -9, 0.0119, 7.7, float.fromhex("0x1.fffffep-7"),
                                1e-30, 1e25])
def test_every_fp16_value_is_encoded_as_the_format_says(cuda, ps):
    """All finite fp16 bit patterns, infinities and a NaN, in groups whose largest element varies."""
    bits = np.arange(65536).astype(np.uint16)
    rng = np.random.default_rng(5)
    x = rng.permutation(bits).view(np.float16).reshape(-1, 1, 256)
    kc = _t(np.zeros(PA.q4_pool_shape(16, 1, 16, 256), np.uint8), cuda)
    vc = kc.clone()
    x2 = np.sort(bits.view(np.float16)).reshape(-1, 1, 256)  # neighbours share a group
    PA.reshape_and_cache_q4(_t(x, cuda), _t(x2, cuda), kc, vc, _t(np.arange(256), cuda), ps, ps)
    for pool, rows, is_key in ((kc, x, True), (vc, x2, False)):
        c, s = R.encode(rows, ps)
        gc, gs = R.unpack(pool.cpu().numpy(), is_key)
        gc = gc.transpose(0, 2, 1, 3).reshape(c.shape)
        gs = gs.transpose(0, 2, 1, 3).reshape(s.shape)
        np.testing.assert_array_equal(gs, s)
        # a NaN's code is a zero of either sign
        np.testing.assert_array_equal(np.where(gc == 8, 0, gc), np.where(c == 8, 0, c))


def test_rows_inside_a_fused_projection_and_off_alignment(cuda):
    """Strided rows, and rows that start off a 16-byte boundary, store the same bytes."""
    import torch
    T, hkv, D, bs = 40, 2, 80, 16
    rng = np.random.default_rng(3)
    k, v = _rows(rng, T, hkv, D), _rows(rng, T, hkv, D)
    slots = _t(_slots(rng, T, 4, bs), cuda)
    pools = [torch.zeros(PA.q4_pool_shape(4, hkv, bs, D), dtype=torch.uint8, device=cuda)
             for _ in range(4)]
    PA.reshape_and_cache_q4(_t(k, cuda), _t(v, cuda), pools[0], pools[1], slots, KS, VS)
    for lead in (0, 8, 3):
        fused = torch.zeros(T, lead + 2 * hkv * D + 5, dtype=torch.float16, device=cuda)
        kk = fused[:, lead:lead + hkv * D].view(T, hkv, D)
        vv = fused[:, lead + hkv * D:lead + 2 * hkv * D].view(T, hkv, D)
        kk.copy_(_t(k, cuda))
        vv.copy_(_t(v, cuda))
        pools[2].zero_(), pools[3].zero_()
        PA.reshape_and_cache_q4(kk, vv, pools[2], pools[3], slots, KS, VS)
        assert torch.equal(pools[0], pools[2]) and torch.equal(pools[1], pools[3])
        want = PA.read_cache_q4(*pools[:2], slots, KS, VS)
        kk.fill_(7), vv.fill_(7)
        PA.read_cache_q4(*pools[:2], slots, KS, VS, key=kk, value=vv)
        assert torch.equal(kk, want[0]) and torch.equal(vv, want[1])
        assert not fused[:, :lead].any() and not fused[:, lead + 2 * hkv * D:].any()


# ── attention ─────────────────────────────────────────────────────────────
def _case(seed, lens, hq, hkv, D, bs, mb=None, fill=None):
    """Pools of random codes and scales (a fraction of them zero), shuffled tables."""
    rng = np.random.default_rng(seed)
    lens = np.asarray(lens, np.int32)
    pages = -(-lens // bs)
    nb = int(pages.sum()) + 3
    mb = max(1, int(pages.max())) if mb is None else mb
    codes = rng.integers(0, 16, (2, nb, hkv, bs, D)).astype(np.uint8)
    sb = rng.integers(20, 70, (2, nb, hkv, bs, D // 16)).astype(np.uint8)
    sb[rng.random(sb.shape) < 0.02] = 0
    pools = [R.pack(codes[0], sb[0], True), R.pack(codes[1], sb[1], False)]
    table = np.full((len(lens), mb), -1, np.int32)
    ids = rng.permutation(nb)[:pages.sum()].astype(np.int32)
    table[np.arange(mb)[None] < pages[:, None]] = ids
    if fill is not None:  # slots past each length, and pages no one holds, hold `fill`
        for i, (p, is_key) in enumerate(zip(pools, (True, False))):
            c, s = R.unpack(p, is_key)
            c, s = c.astype(np.uint8), s.copy()
            used = np.zeros((nb, bs), bool)
            for b, n in enumerate(lens):
                at = np.arange(n)
                used[table[b, at // bs], at % bs] = True
            w = np.broadcast_to(used[:, None], (nb, hkv, bs))
            c[~w], s[~w] = fill & 15, fill
            pools[i] = R.pack(c, s, is_key)
    q = rng.standard_normal((len(lens), hq, D)).astype(np.float16)
    return q, pools, table, lens


def _reference(q, pools, table, lens, scale, num_blocks=None):
    k = R.values(*R.unpack(pools[0], True), KS)
    v = R.values(*R.unpack(pools[1], False), VS)
    return R.attention(q, k, v, table, lens, scale, num_blocks)


def _close(out, ref, bound):
    x = out.double().cpu().numpy()
    assert np.isfinite(x).all()
    worst = np.max(np.abs(x - ref) / bound)
    assert worst <= 1.0, worst
    return worst


SHAPES = [
    # hq, hkv, D, bs
    (1, 1, 64, 16), (8, 8, 128, 16), (32, 8, 128, 16), (16, 2, 128, 32), (32, 2, 128, 16),
    (40, 1, 128, 16), (12, 12, 64, 16), (16, 1, 64, 48), (10, 2, 256, 16), (20, 2, 256, 32),
    (6, 2, 16, 16), (6, 3, 32, 16), (5, 1, 48, 16), (20, 4, 96, 32), (9, 1, 80, 16),
    (4, 2, 144, 16), (34, 2, 192, 64), (3, 3, 208, 16), (7, 1, 240, 16),
    (12, 1, 112, 16), (2, 1, 160, 16), (11, 1, 176, 32), (24, 2, 224, 16), (18, 2, 48, 16),
    (9, 1, 16, 16), (16, 1, 96, 16), (30, 2, 80, 16), (10, 1, 32, 16),
]
LENS = [[1], [0, 1, 15, 16, 17, 33], [127, 700, 5, 2049, 0, 64]]


@pytest.mark.parametrize("lens", LENS, ids=lambda x: "x".join(map(str, x)))
@pytest.mark.parametrize("hq,hkv,D,bs", SHAPES)
def test_attention_is_within_its_bound(cuda, hq, hkv, D, bs, lens):
    import torch
    # bytes past the lengths decode to NaN: none may reach an output
    q, pools, table, lens = _case(hq * D + len(lens), lens, hq, hkv, D, bs, fill=0x7f)
    ref, bound = _reference(q, pools, table, lens, 1 / math.sqrt(D))
    args = (_t(q, cuda), _t(pools[0], cuda), _t(pools[1], cuda), _t(table, cuda), _t(lens, cuda))
    out = torch.full_like(args[0], float("nan"))
    PA.device_status(clear=True)
    PA.paged_attention_q4(*args, KS, VS, out=out)
    torch.cuda.synchronize()
    _close(out, ref, bound)
    assert not out[torch.from_numpy(lens == 0).to(cuda)].any()
    assert PA.device_status(clear=True) == 0


def test_masked_pages_clamped_lengths_and_status(cuda):
    import torch
    q, pools, table, lens = _case(5, [200, 90, 64, 500], 8, 2, 128, 16)
    table[0, 3] = -1
    table[0, 12] = -7            # the last, partial page
    table[1, :] = -1             # nothing left
    table[3, 5] = len(pools[0])  # past the pool
    table[3, 9] = 2 ** 31 - 1
    lens = lens.copy()
    lens[2] = 10 ** 9            # clamped to the table
    table[2, 4:] = -1
    ref, bound = _reference(q, pools, table, lens, 0.1)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    out = PA.paged_attention_q4(_t(q, cuda), _t(pools[0], cuda), _t(pools[1], cuda),
                                _t(table, cuda), _t(lens, cuda), KS, VS, scale=0.1,
                                device_status=status)
    _close(out, ref, bound)
    assert not out[1].any()
    assert int(status) == _native.NXT_PA_DEV_BAD_PAGE | _native.NXT_PA_DEV_SEQ_CLAMPED
    out = PA.paged_attention_q4(_t(q[2:3], cuda), _t(pools[0], cuda), _t(pools[1], cuda),
                                _t(table[2:3], cuda), _t(np.array([-5], np.int32), cuda), KS, VS,
                                device_status=status.zero_())
    assert not out.any() and int(status) == _native.NXT_PA_DEV_SEQ_CLAMPED


@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
def test_other_score_scales(cuda, scale):
    """Uniform, reversed and very peaked weights (scores hundreds of units apart)."""
    q, pools, table, lens = _case(11, [333, 64], 8, 2, 128, 16)
    ref, bound = _reference(q, pools, table, lens, scale)
    out = PA.paged_attention_q4(_t(q, cuda), _t(pools[0], cuda), _t(pools[1], cuda),
                                _t(table, cuda), _t(lens, cuda), KS, VS, scale=scale)
    _close(out, ref, bound)


def _c_call(q, kc, vc, bt, sl, out, hkv, D, bs, kbs, khs, ws=None, ws_bytes=0, stream=None):
    import torch
    st = torch.cuda.current_stream().cuda_stream if stream is None else stream
    p = lambda x: None if x is None else x.data_ptr()
    return _native.xpa().nxt_paged_attention_q4_ex(
        p(out), p(q), p(kc), p(vc), p(bt), p(sl), q.shape[0], q.shape[1], D, hkv,
        1 / math.sqrt(D), bt.shape[1], bs, KS, VS, kbs, khs, -1, p(ws), ws_bytes, None, st)


def test_strided_pools_unaligned_query_and_own_workspace(cuda):
    """Pools whose pages are padded, heads outermost; rows off every wide
    boundary; a workspace of exactly the size asked for, none of it past its end."""
    import torch
    hq, hkv, D, bs = 8, 2, 128, 16
    q, pools, table, lens = _case(21, [3000, 17, 900], hq, hkv, D, bs)
    ref, bound = _reference(q, pools, table, lens, 1 / math.sqrt(D))
    nb = len(pools[0])
    tile = 9 * D
    big = torch.full((2, hkv, nb, tile + 48), 0xff, dtype=torch.uint8, device=cuda)
    for i in (0, 1):
        big[i, :, :, :tile] = _t(pools[i].reshape(nb, hkv, tile).transpose(1, 0, 2), cuda)
    need = PA.q4_workspace_size(3, hq, D, hkv, table.shape[1], bs)
    assert need > 0
    qq = torch.zeros(q.size + 1, dtype=torch.float16, device=cuda)[1:].view(q.shape)
    qq.copy_(_t(q, cuda))
    oo = torch.zeros(q.size + 1, dtype=torch.float16, device=cuda)[1:].view(q.shape)
    ws = torch.full((need + 64,), 0x5a, dtype=torch.uint8, device=cuda)
    args = (qq, big[0], big[1], _t(table, cuda), _t(lens, cuda), oo, hkv, D, bs, tile + 48,
            nb * (tile + 48))
    assert _c_call(*args, ws=ws, ws_bytes=need - 1) == _native.NXT_PA_EWORKSPACE
    assert _c_call(*args, ws=ws, ws_bytes=need) == _native.NXT_PA_OK
    _close(oo, ref, bound)
    assert (ws[need:] == 0x5a).all()


def test_append_step_equals_write_then_attention(cuda):
    import torch
    for hq, hkv, D, bs in ((8, 2, 128, 16), (6, 3, 96, 32)):
        q, pools, table, lens = _case(31, [40, 1, 700, 2049], hq, hkv, D, bs)
        rng = np.random.default_rng(1)
        nk, nv = _rows(rng, 4, hkv, D), _rows(rng, 4, hkv, D)
        last = lens - 1
        slots = (table[np.arange(4), last // bs].astype(np.int64) * bs + last % bs)
        a = [_t(p, cuda) for p in pools]
        b = [_t(p, cuda) for p in pools]
        PA.reshape_and_cache_q4(_t(nk, cuda), _t(nv, cuda), *a, _t(slots, cuda), KS, VS)
        want = PA.paged_attention_q4(_t(q, cuda), *a, _t(table, cuda), _t(lens, cuda), KS, VS)
        got = PA.paged_attention_q4_append(_t(q, cuda), *b, _t(table, cuda), _t(lens, cuda),
                                           _t(nk, cuda), _t(nv, cuda), _t(slots, cuda), KS, VS)
        assert torch.equal(got, want) and torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        ref, bound = _reference(q, [x.cpu().numpy() for x in a], table, lens, 1 / math.sqrt(D))
        _close(got, ref, bound)


def test_offsets_past_32_bits(cuda):
    """A pool of over 4 GiB whose pages in use lie at its end."""
    import torch
    hkv, D, bs = 8, 128, 16
    nb = 2 ** 32 // (hkv * 9 * D) + 40
    q, pools, table, lens = _case(41, [70, 33], 8, hkv, D, bs)
    used = len(pools[0])
    big = torch.zeros(PA.q4_pool_shape(nb, hkv, bs, D), dtype=torch.uint8, device=cuda)
    big[nb - used:] = _t(pools[0], cuda)
    far = np.where(table >= 0, table + nb - used, -1).astype(np.int32)
    vfar = big.clone()
    vfar[nb - used:] = _t(pools[1], cuda)
    out = PA.paged_attention_q4(_t(q, cuda), big, vfar, _t(far, cuda), _t(lens, cuda), KS, VS)
    ref, bound = _reference(q, pools, table, lens, 1 / math.sqrt(D))
    _close(out, ref, bound)
    slots = _t(np.array([nb * bs - 1, nb * bs - 17], np.int64), cuda)
    rng = np.random.default_rng(2)
    k = _rows(rng, 2, hkv, D)
    PA.reshape_and_cache_q4(_t(k, cuda), _t(k, cuda), big, vfar, slots, KS, VS)
    rk, _ = PA.read_cache_q4(big, vfar, slots, KS, VS)
    np.testing.assert_allclose(rk.double().cpu().numpy(),
                               _expected(k, KS)[1].astype(np.float64), rtol=2.0 ** -10, atol=2.0 ** -24)


def test_streams_graphs_and_threads_give_the_same_bits(cuda):
    import torch
    q, pools, table, lens = _case(51, [3000, 100, 1700], 32, 8, 128, 16)
    args = (_t(q, cuda), _t(pools[0], cuda), _t(pools[1], cuda), _t(table, cuda), _t(lens, cuda))
    want = PA.paged_attention_q4(*args, KS, VS)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        out = torch.empty_like(want)
        PA.paged_attention_q4(*args, KS, VS, out=out)  # the stream's scratch exists from here on
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            PA.paged_attention_q4(*args, KS, VS, out=out)
    # a larger eager call on the same stream replaces the scratch; the graph keeps its own
    wide = _case(52, [3000] * 24, 32, 8, 128, 16)
    wargs = (_t(wide[0], cuda), _t(wide[1][0], cuda), _t(wide[1][1], cuda), _t(wide[2], cuda),
             _t(wide[3], cuda))
    PA.paged_attention_q4(*wargs, KS, VS, stream=side)
    torch.cuda.synchronize()
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    got = [None] * 4

    def work(i):
        st = torch.cuda.Stream()
        for _ in range(5):
            got[i] = PA.paged_attention_q4(*args, KS, VS, stream=st)
        st.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert all(torch.equal(g, want) for g in got)


def test_release_frees_the_scratch_and_later_calls_work(cuda):
    import torch
    q, pools, table, lens = _case(61, [3000], 8, 2, 128, 16)
    args = (_t(q, cuda), _t(pools[0], cuda), _t(pools[1], cuda), _t(table, cuda), _t(lens, cuda))
    want = PA.paged_attention_q4(*args, KS, VS)
    torch.cuda.synchronize()
    assert _native.xpa().nxt_paged_attention_release_workspaces() == _native.NXT_PA_OK
    assert torch.equal(PA.paged_attention_q4(*args, KS, VS), want)


def test_a_run_as_it_is_used(cuda):
    """A prompt is stored, five decode steps follow; the cache read back is the
    one that attention saw, and the step's output that of the rows read back."""
    import torch
    hq, hkv, D, bs, n0 = 8, 2, 128, 16, 45
    rng = np.random.default_rng(9)
    nb = 6
    kc = torch.zeros(PA.q4_pool_shape(nb, hkv, bs, D), dtype=torch.uint8, device=cuda)
    vc = torch.zeros_like(kc)
    bt = PA.build_block_tables([[4, 1, 0, 5]], [n0], 4, block_size=bs, device=cuda)
    order = np.array([4, 1, 0, 5])
    pos = np.arange(n0 + 5)
    slot_of = order[pos // bs] * bs + pos % bs
    prompt = _t(rng.standard_normal((2, n0, hkv, D)).astype(np.float16), cuda)
    PA.reshape_and_cache_q4(prompt[0], prompt[1], kc, vc, _t(slot_of[:n0], cuda), KS, VS)
    for step in range(5):
        n = n0 + step + 1
        bt = PA.build_block_tables([order[:-(-n // bs)].tolist()], [n], 4, block_size=bs,
                                   device=cuda)
        assert int(bt.slots[0]) == slot_of[n - 1]
        new = _t(rng.standard_normal((2, 1, hkv, D)).astype(np.float16), cuda)
        q = _t(rng.standard_normal((1, hq, D)).astype(np.float16), cuda)
        out = PA.paged_attention_q4_append(q, kc, vc, bt.tables, bt.seq_lens, new[0], new[1],
                                           bt.slots, KS, VS)
        pools = [kc.cpu().numpy(), vc.cpu().numpy()]
        ref, bound = _reference(q.cpu().numpy(), pools, bt.tables.cpu().numpy(), [n],
                                1 / math.sqrt(D))
        _close(out, ref, bound)
    k, v = PA.read_cache_q4(kc, vc, _t(slot_of, cuda), KS, VS)
    np.testing.assert_allclose(k[:n0].double().cpu().numpy(),
                               _expected(prompt[0].cpu().numpy(), KS)[1].astype(np.float64),
                               rtol=2.0 ** -10)
    assert v.shape == (n0 + 5, hkv, D)


def test_graphs_replayed_at_the_same_time_have_scratch_of_their_own(cuda):
    """Two graphs captured on one stream and an eager call, each with partials
    to merge, run side by side again and again."""
    import torch
    side, streams = torch.cuda.Stream(), [torch.cuda.Stream() for _ in range(2)]
    runs = []
    for seed in (71, 72, 73):
        q, pools, table, lens = _case(seed, [6000, 5000, 4000, 7000], 32, 8, 128, 16)
        args = [_t(x, cuda) for x in (q, pools[0], pools[1], table, lens)]
        want = PA.paged_attention_q4(*args, KS, VS)
        runs.append((args, want, torch.empty_like(want)))
    assert PA.q4_workspace_size(4, 32, 128, 8, table.shape[1]) > 0
    torch.cuda.synchronize()
    graphs = []
    for args, _, out in runs[:2]:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=side):
            for _ in range(4):
                PA.paged_attention_q4(*args, KS, VS, out=out)
    for _ in range(20):
        for _, _, out in runs:
            out.zero_()
        torch.cuda.synchronize()
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        for _ in range(4):
            PA.paged_attention_q4(*runs[2][0], KS, VS, out=runs[2][2], stream=side)
        torch.cuda.synchronize()
        for _, want, out in runs:
            assert torch.equal(out, want)
    assert _native.xpa().nxt_paged_attention_release_workspaces() == _native.NXT_PA_OK
    runs[0][2].zero_()  # a graph keeps its scratch
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(runs[0][2], runs[0][1])


def test_graphs_that_are_gone_give_their_scratch_back(cuda):
    import torch
    q, pools, table, lens = _case(74, [6000] * 24, 32, 8, 128, 16)
    args = [_t(x, cuda) for x in (q, pools[0], pools[1], table, lens)]
    out = PA.paged_attention_q4(*args, KS, VS)
    need = PA.q4_workspace_size(24, 32, 128, 8, table.shape[1])
    assert need > 2 ** 20
    side = torch.cuda.Stream()
    free = []
    for _ in range(40):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            PA.paged_attention_q4(*args, KS, VS, out=out)
        graph.replay()
        torch.cuda.synchronize()
        del graph
        torch.cuda.synchronize()
        free.append(torch.cuda.mem_get_info()[0])
    # the driver's thread may lag some captures behind
    assert free[0] - free[-1] < 20 * need


def test_more_blocks_than_the_pools_have_are_refused(cuda):
    q, pools, table, lens = _case(75, [100], 8, 2, 128, 16)
    args = [_t(x, cuda) for x in (q, pools[0], pools[1], table, lens)]
    nb = pools[0].shape[0]
    want = PA.paged_attention_q4(*args, KS, VS)
    for few in (nb, -1):
        assert (PA.paged_attention_q4(*args, KS, VS, num_blocks=few) == want).all()
    with pytest.raises(PA.PagedAttentionError):
        PA.paged_attention_q4(*args, KS, VS, num_blocks=nb + 1)


def test_read_back_into_either_or_both_rows(cuda):
    import torch
    hkv, D, T = 2, 64, 21
    rng = np.random.default_rng(76)
    pool = _t(rng.integers(0, 0x70, PA.q4_pool_shape(3, hkv, 16, D)).astype(np.uint8), cuda)
    slots = _t(_slots(rng, T, 3, 16), cuda)
    want = PA.read_cache_q4(pool, pool, slots, KS, VS)
    for given in (("key",), ("value",), ("key", "value")):
        wide = torch.zeros(T, hkv * D + 8, dtype=torch.float16, device=cuda)
        rows = {name: wide.clone()[:, :hkv * D].view(T, hkv, D) for name in given}
        got = PA.read_cache_q4(pool, pool, slots, KS, VS, **rows)
        assert all(torch.equal(g, w) for g, w in zip(got, want))
        assert all(got["key value".split().index(n)] is r for n, r in rows.items())
        assert got[0].stride() == got[1].stride()
    with pytest.raises(PA.PagedAttentionError):
        PA.read_cache_q4(pool, pool, slots, KS, VS, key=want[0], value=wide[:, 8:].view(T, hkv, D))
