"""The 4-bit cache, and attention over fp16 pages, at the ends of their range
and in narrow calls, against statements in 64 bits."""
import math
import os
import subprocess
import sys
import threading

import numpy as np
import pytest

import _q4ref as R
from xllms_b200 import _native
from xllms_b200 import operator_api as PA

pytestmark = pytest.mark.gpu


def _t(x, dev):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x)).to(dev)


def _paged(rng, lens, bs):
    """(table, number of blocks): shuffled pages for these lengths."""
    lens = np.asarray(lens)
    pages = -(-lens // bs)
    nb = int(pages.sum()) + 2
    table = np.full((len(lens), max(1, int(pages.max()))), -1, np.int32)
    table[np.arange(table.shape[1])[None] < pages[:, None]] = rng.permutation(nb)[:pages.sum()]
    return table, nb


def _rows_of(pool, table, n, h, bs):
    """Rows [n, D] of one sequence and KV head from values [nb, Hkv, bs, D]."""
    at = np.arange(n)
    return pool[table[at // bs], h, at % bs]


def _softmax_av(s, v, extra=0.0):
    """(out, bound) of exact scores s [n] and values v [n, D]. The kernels hold a
    weight as two fp16 terms: 2^-22 of it, and where the second is subnormal
    half of 2^-24, 2^-32 of the largest weight, which is at least 2^7. Its
    exponent is a difference of scores times a factor of three roundings, in
    one fused step: 2^-22 of the difference, and the exponential's 2^-22.
    Products and sums are fp32, a matrix step or a merge off by 2^-22 of the sum
    of magnitudes, and the output is rounded to fp16 once."""
    d = s - s.max()
    p = np.exp(d)
    p /= p.sum()
    out = p @ v
    ds = 2.0 ** -22 + 1.5 * 2.0 ** -22 * np.abs(d)
    bound = (p * (np.expm1(2 * ds) + 2.0 ** -21 + (len(s) / 16 + 16) * 2.0 ** -22 + extra)) @ np.abs(v)
    bound += 2.0 ** -32 * p.max() * np.abs(v).sum(0)
    return out, bound + 2.0 ** -11 * np.abs(out) + 2.0 ** -25


def _worst(out, ref, bound):
    x = out.double().cpu().numpy()
    assert np.isfinite(x).all()
    worst = np.max(np.abs(x - ref) / bound)
    assert worst <= 1.0, worst


# ── 4-bit pools with chosen keys ──────────────────────────────────────────
def _q4_pools(rng, k_codes, k_scale_byte):
    """(pools, values) of these key codes, one scale byte for all, random values."""
    nb, hkv, bs, D = k_codes.shape
    kb = np.full((nb, hkv, bs, D // 16), k_scale_byte, np.uint8)
    vc = rng.integers(0, 16, k_codes.shape).astype(np.uint8)
    vb = rng.integers(40, 60, kb.shape).astype(np.uint8)
    pools = R.pack(k_codes, kb, True), R.pack(vc, vb, False)
    return pools, (R.values(k_codes, kb, 1.0), R.values(vc, vb, 0.5))


def _q4_call(cuda, q, pools, table, lens, scale):
    return PA.paged_attention_q4(_t(q, cuda), _t(pools[0], cuda), _t(pools[1], cuda),
                                 _t(table, cuda), _t(np.asarray(lens, np.int32), cuda), 1.0, 0.5,
                                 scale=scale)


def _check_rows(out, q, k, v, table, lens, scale, bs, exact=True):
    hkv = k.shape[1]
    group = q.shape[1] // hkv
    ref, bound = np.zeros(q.shape), np.zeros(q.shape)
    for b, n in enumerate(lens):
        for x in range(q.shape[1]):
            kk, vv = (_rows_of(y, table[b], n, x // group, bs) for y in (k, v))
            s = kk @ q[b, x].astype(np.float64) * scale
            # equal keys have equal scores, whatever the sums round to
            s = s if exact else np.zeros(n)
            ref[b, x], bound[b, x] = _softmax_av(s, vv)
    _worst(out, ref, bound)


HUGE = [65504.0, -65504.0, 30000.0]
Q4_SHAPES = [(8, 2, 128, 16), (3, 1, 112, 16), (16, 1, 64, 32), (2, 1, 256, 16), (9, 1, 80, 16)]


@pytest.mark.parametrize("value", HUGE)
@pytest.mark.parametrize("hq,hkv,D,bs", Q4_SHAPES)
def test_q4_equal_keys_weigh_the_same_at_any_score(cuda, hq, hkv, D, bs, value):
    """The largest queries against the largest keys: one token's weight is 1,
    many tokens of one key get equal weights."""
    rng = np.random.default_rng(D)
    lens = [1, 40, 700, 5000]
    table, nb = _paged(rng, lens, bs)
    codes = np.broadcast_to(rng.integers(0, 16, (1, hkv, 1, D)), (nb, hkv, bs, D)).astype(np.uint8)
    for scale_byte in (0x7e, 0x38):  # 448 and 1
        pools, (k, v) = _q4_pools(rng, codes, scale_byte)
        q = np.full((len(lens), hq, D), value, np.float16)
        q[:, ::2, ::3] *= np.float16(0.5)
        for scale in (1 / math.sqrt(D), -3.0):
            out = _q4_call(cuda, q, pools, table, lens, scale)
            _check_rows(out, q, k, v, table, lens, scale, bs, exact=False)


def _rising(rng, n, steps):
    """Offsets of n tokens: some runs of rising ones, then any."""
    d = rng.integers(0, len(steps), n)
    d[:n // 2] = np.sort(d[:n // 2])
    return d


@pytest.mark.parametrize("scale", [1.0, -1.0, 0.25])
@pytest.mark.parametrize("D", [64, 128, 112, 256])
def test_q4_differences_of_large_scores(cuda, D, scale):
    """Scores of 12.6 million whose differences of a few units decide the
    weights; every sum is a whole number below 2^24, so fp32 holds it exactly."""
    rng = np.random.default_rng(D)
    hq, hkv, bs, lens = 2, 1, 16, [3, 64, 700, 5000]
    table, nb = _paged(rng, lens, bs)
    codes = np.zeros((nb, hkv, bs, D), np.uint8)
    codes[..., 0] = 7  # 6 * 64 * 32768
    for b, n in enumerate(lens):
        at = np.arange(n)
        codes[table[b, at // bs], 0, at % bs, 1] = _rising(rng, n, R.LEVELS)
    pools, (k, v) = _q4_pools(rng, codes, 0x68)  # 64
    q = np.zeros((len(lens), hq, D), np.float16)
    q[:, :, 0] = 32768 * np.sign(scale)
    q[:, 0, 1] = 1 / 32  # 32 code units / 32: whole numbers
    q[:, 1, 1] = -1 / 32
    out = _q4_call(cuda, q, pools, table, lens, scale)
    _check_rows(out, q, k, v, table, lens, scale, bs)


def _pages_case(rng, lens, hkv, D, bs):
    table, nb = _paged(rng, lens, bs)
    return table, nb, rng.standard_normal((nb, hkv, bs, D)).astype(np.float16)


def _keep_all(cuda, q, k, v, table, lens, scale, **kw):
    """Sparse attention that keeps every page (bounds are not read)."""
    bnd = np.zeros((len(k), k.shape[1], 2, k.shape[3]), np.float16)
    return PA.paged_attention_sparse(*(_t(x, cuda) for x in (q, k, v, bnd, table)),
                                     _t(np.asarray(lens, np.int32), cuda), table.shape[1],
                                     scale=scale, **kw)


# shapes of the kernel of plain page copies: its head sizes, a group of 13
PAGE_SHAPES = [(20, 5, 112, 16), (3, 1, 80, 32), (13, 1, 256, 16), (2, 2, 208, 48)]


@pytest.mark.parametrize("value", HUGE)
@pytest.mark.parametrize("hq,hkv,D,bs", PAGE_SHAPES)
def test_pages_equal_keys_weigh_the_same_at_any_score(cuda, hq, hkv, D, bs, value):
    rng = np.random.default_rng(D)
    lens = [1, 40, 900, 3000]
    table, nb, v = _pages_case(rng, lens, hkv, D, bs)
    k = np.broadcast_to(rng.choice([65504.0, 30000.0, -9.5], (1, hkv, 1, D)), v.shape).astype(np.float16)
    q = np.full((len(lens), hq, D), value, np.float16)
    q[:, ::2, ::3] *= np.float16(0.5)
    for scale in (1 / math.sqrt(D), -3.0):
        out = _keep_all(cuda, q, k, v, table, lens, scale)
        _check_rows(out, q, k.astype(np.float64), v.astype(np.float64), table, lens, scale, bs,
                    exact=False)


@pytest.mark.parametrize("scale", [1.0, -1.0, 0.25])
@pytest.mark.parametrize("hq,hkv,D,bs", PAGE_SHAPES)
def test_pages_differences_of_large_scores(cuda, hq, hkv, D, bs, scale):
    """As for 4-bit pools: scores of 2^23 and whole differences."""
    rng = np.random.default_rng(D)
    lens = [3, 64, 900, 3000]
    table, nb, v = _pages_case(rng, lens, hkv, D, bs)
    k = np.zeros(v.shape, np.float16)
    k[..., 0] = 2048
    for b, n in enumerate(lens):
        at = np.arange(n)
        k[table[b, at // bs], :, at % bs, 1] = _rising(rng, n, range(13))[:, None]
    q = np.zeros((len(lens), hq, D), np.float16)
    q[:, :, 0] = 4096 * np.sign(scale)
    q[:, :, 1] = rng.choice([1, -1], hq)
    out = _keep_all(cuda, q, k, v, table, lens, scale)
    _check_rows(out, q, k.astype(np.float64), v.astype(np.float64), table, lens, scale, bs)


@pytest.mark.parametrize("hq,hkv,D,bs", Q4_SHAPES + [(20, 2, 128, 16), (10, 1, 240, 16)])
def test_q4_weights_keep_22_bits(cuda, hq, hkv, D, bs):
    """Whole-number queries and keys of half units, whose scores are exact: what
    is off is the weights' and the sums' own rounding, and it stays within the
    bound of two fp16 terms a weight."""
    rng = np.random.default_rng(hq * D)
    lens = [1, 17, 300, 2500]
    table, nb = _paged(rng, lens, bs)
    pools, (k, v) = _q4_pools(rng, rng.integers(0, 16, (nb, hkv, bs, D)).astype(np.uint8), 0x38)
    q = rng.integers(-2, 3, (len(lens), hq, D)).astype(np.float16)
    for scale in (1 / 16, 1 / 64):
        out = _q4_call(cuda, q, pools, table, lens, scale)
        _check_rows(out, q, k, v, table, lens, scale, bs)


# ── NaN ───────────────────────────────────────────────────────────────────
def test_a_nan_query_gives_zeros_however_a_row_is_split(cuda):
    """As in the framework's other decode calls: a head whose scores are NaN has
    no sum above 0 and its output is 0, in one partition or many; the others'
    outputs are off by no more than their rounding (the reference points of a
    warp's heads move together, so not every bit need be the same)."""
    rng = np.random.default_rng(6)
    hq, hkv, D, bs, lens = 8, 2, 128, 16, [40, 1, 6000, 4097]
    table, nb = _paged(rng, lens, bs)
    q = rng.standard_normal((len(lens), hq, D)).astype(np.float16)
    bad = q.copy()
    bad[:, 1, 5] = np.nan
    bad[:, 6] = np.nan
    others = [0, 2, 3, 4, 5, 7]
    kv = rng.standard_normal((2, nb, hkv, bs, D)).astype(np.float16)
    pools, (_, v4) = _q4_pools(rng, rng.integers(0, 16, (nb, hkv, bs, D)).astype(np.uint8), 0x38)
    lt = _t(np.asarray(lens, np.int32), cuda)
    calls = {
        "fp16": lambda x: PA.paged_attention(_t(x, cuda), _t(kv[0], cuda), _t(kv[1], cuda),
                                             _t(table, cuda), lt),
        "q4": lambda x: _q4_call(cuda, x, pools, table, lens, 0.1),
    }
    def check(good, out, top, name):
        assert not out[:, [1, 6]].any(), name
        # one fp16 step, and twice the sums' bound
        tol = good.abs().double() * 2.0 ** -10 + top * 2 * 2.0 ** -22 * (
            _t(np.asarray(lens) / 16 + 20.0, cuda))[:, None, None]
        assert ((out.double() - good.double()).abs() <= tol)[:, others].all(), name

    for name, call in calls.items():
        check(call(q), call(bad), 8.0 if name == "fp16" else float(abs(v4).max()), name)
    k = rng.standard_normal((nb, hkv, bs, 112)).astype(np.float16)
    q, bad = q[..., :112], bad[..., :112]
    check(*(_keep_all(cuda, x, k, k, table, lens, 0.1) for x in (q, bad)), 8.0, "pages")


@pytest.mark.parametrize("at", [0, 33, "last"])
@pytest.mark.parametrize("hq,hkv,D,bs", PAGE_SHAPES)
def test_a_nan_key_gives_zeros_however_a_row_is_split(cuda, hq, hkv, D, bs, at):
    """Also where the NaN is the only token of the row's last partition."""
    rng = np.random.default_rng(7)
    lens = [64, 500, 2049, 4097]
    table, nb, v = _pages_case(rng, lens, hkv, D, bs)
    k = rng.standard_normal(v.shape).astype(np.float16)
    for b, n in enumerate(lens):
        tok = n - 1 if at == "last" else at
        k[table[b, tok // bs], 0, tok % bs, 2] = np.nan
    q = rng.standard_normal((len(lens), hq, D)).astype(np.float16)
    out = _keep_all(cuda, q, k, v, table, lens, 0.1)
    group = hq // hkv
    assert not out[:, :group].any()
    if hkv > 1:
        clean = np.nan_to_num(k)
        assert (out[:, group:] == _keep_all(cuda, q, clean, v, table, lens, 0.1)[:, group:]).all()


# ── narrow calls ──────────────────────────────────────────────────────────
def test_one_tokens_rows_of_any_outer_strides(cuda):
    """With one token, or one head, the strides that no address uses may differ:
    a view of a fused projection's row beside a dense one."""
    import torch
    D, bs = 64, 16
    rng = np.random.default_rng(3)
    for T, hkv in ((1, 2), (1, 1), (5, 1)):
        width = 3 * hkv * D + 8
        fused = _t(rng.standard_normal((T, width)).astype(np.float16), cuda)
        if T > 1:  # rows of one head: any head stride beside the same token stride
            key = fused.as_strided((T, 1, D), (width, 7, 1), 8)
            value = fused.as_strided((T, 1, D), (width, D, 1), 8 + D)
        else:
            key = fused.as_strided((1, hkv, D), (width, D, 1), 8)
            value = _t(rng.standard_normal((1, hkv, D)).astype(np.float16), cuda)
        assert key.stride() != value.stride()
        slots = _t(rng.permutation(32)[:T].astype(np.int64), cuda)
        pools = torch.zeros((4,) + PA.q4_pool_shape(2, hkv, bs, D), dtype=torch.uint8, device=cuda)
        PA.reshape_and_cache_q4(key, value, pools[0], pools[1], slots, 0.01, 0.02)
        PA.reshape_and_cache_q4(key.clone(memory_format=torch.contiguous_format),
                                value.clone(memory_format=torch.contiguous_format), pools[2],
                                pools[3], slots, 0.01, 0.02)
        assert torch.equal(pools[:2], pools[2:]) and pools[0].any()
        want = PA.read_cache_q4(pools[0], pools[1], slots, 0.01, 0.02)
        got = PA.read_cache_q4(pools[0], pools[1], slots, 0.01, 0.02, key=key, value=value)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_rows_of_two_tokens_still_need_one_stride(cuda):
    import torch
    rows = torch.zeros(2, 300, dtype=torch.float16, device=cuda)
    key, dense = rows[:, :128].view(2, 2, 64), torch.zeros(2, 2, 64, dtype=torch.float16, device=cuda)
    pool = torch.zeros(PA.q4_pool_shape(2, 2, 16, 64), dtype=torch.uint8, device=cuda)
    slots = torch.arange(2, device=cuda)
    with pytest.raises(PA.PagedAttentionError):
        PA.reshape_and_cache_q4(key, dense, pool, pool.clone(), slots, 1.0, 1.0)


# ── another thread's capture ──────────────────────────────────────────────
def test_an_eager_call_on_a_new_stream_leaves_another_threads_capture_alone(cuda):
    """While one thread captures, another makes its stream's first call (which
    allocates that stream's scratch) and a larger one (which replaces it)."""
    import torch
    rng = np.random.default_rng(5)
    cases = []
    for lens in ([6000, 5000], [9000] * 6):
        table, nb = _paged(rng, lens, 16)
        pools, _ = _q4_pools(rng, rng.integers(0, 16, (nb, 8, 16, 128)).astype(np.uint8), 0x38)
        q = rng.standard_normal((len(lens), 32, 128)).astype(np.float16)
        args = [_t(x, cuda) for x in (q, *pools, table, np.asarray(lens, np.int32))]
        want = PA.paged_attention_q4(*args, 1.0, 0.5)
        cases.append((args, want, torch.empty_like(want), torch.empty_like(want)))
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    # every stream's scratch is gone: the next call on each is its first
    assert _native.xpa().nxt_paged_attention_release_workspaces() == _native.NXT_PA_OK
    failed = []

    def eager():
        try:
            for args, _, out, _ in cases:
                PA.paged_attention_q4(*args, 1.0, 0.5, out=out, stream=other)
        except Exception as exc:  # looked at by the test's own thread
            failed.append(exc)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        PA.paged_attention_q4(*cases[0][0], 1.0, 0.5, out=cases[0][3])
        thread = threading.Thread(target=eager)
        thread.start()
        thread.join()
        PA.paged_attention_q4(*cases[1][0], 1.0, 0.5, out=cases[1][3])
    assert not failed, failed
    graph.replay()
    torch.cuda.synchronize()
    for _, want, out, captured in cases:
        assert torch.equal(out, want) and torch.equal(captured, want)


FIRST_CALL = """
import sys, threading
import torch
from xllms_b200 import operator_api as PA
dev = torch.device("cuda:0")
q = torch.randn(2, 8, 128, device=dev).half()
pool = torch.zeros(PA.q4_pool_shape(200, 2, 16, 128), dtype=torch.uint8, device=dev)
pool.view(-1)[::5] = 0x31
table = torch.arange(200, dtype=torch.int32, device=dev).view(2, 100)
lens = torch.tensor([1600, 1500], dtype=torch.int32, device=dev)
outs = [torch.zeros_like(q) for _ in range(2)]
side, other = torch.cuda.Stream(), torch.cuda.Stream()
call = lambda out, st: PA.paged_attention_q4(q, pool, pool, table, lens, 1.0, 1.0, out=out, stream=st)
x = torch.zeros(4, device=dev)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=side):
    x.add_(1)
    if sys.argv[1] == "beside":
        thread = threading.Thread(target=call, args=(outs[0], other))
        thread.start()
        thread.join()
    else:
        call(outs[0], None)
graph.replay()
torch.cuda.synchronize()
call(outs[1], None)
torch.cuda.synchronize()
assert outs[1].any() and torch.equal(*outs) and (x == 1).all() and PA.device_status() == 0
print("first call ok")
"""


@pytest.mark.parametrize("where", ["beside", "inside"])
def test_the_devices_first_call_beside_or_inside_a_capture(cuda, where):
    """A process of its own, whose first library call allocates the status word."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST_CALL, where], cwd=root, capture_output=True,
                       text=True, timeout=300)
    assert r.returncode == 0 and "first call ok" in r.stdout, r.stderr[-2000:]
