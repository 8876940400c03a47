"""The 64-bit statement of the 4-bit KV format, and the refusals of the 4-bit
entry points, without a GPU."""
import ctypes

import numpy as np
import pytest
import torch

import _q4ref as R
from xllms_b200 import _native
from xllms_b200 import operator_api as PA


def test_scale_bytes_are_torchs_e4m3():
    t = torch.arange(256).to(torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(t, R.E4M3)


@pytest.mark.parametrize("x,level", [(0.25, 0.0), (0.2500001, 0.5), (0.75, 1.0), (1.25, 1.0),
                                     (1.75, 2.0), (2.5, 2.0), (2.500001, 3.0), (3.5, 4.0),
                                     (5.0, 4.0), (5.1, 6.0), (100.0, 6.0)])
def test_codes_round_to_the_nearest_level_ties_to_even(x, level):
    assert R.LEVELS[R._nearest(np.array(min(x, 6.0)), R.LEVELS)] == level


def test_encoding_keeps_what_the_format_holds():
    rng = np.random.default_rng(0)
    codes = rng.integers(0, 16, (3, 2, 16, 96)).astype(np.uint8)
    codes[..., ::16] = 7  # every group holds its largest level, so its scale is found again
    sb = rng.integers(8, 127, (3, 2, 16, 6)).astype(np.uint8)
    x = R.values(codes, sb, 1.0)
    c2, s2 = R.encode(x.astype(np.float32), 1.0)
    np.testing.assert_array_equal(s2, sb)
    np.testing.assert_array_equal(R.values(c2, s2, 1.0), x)


@pytest.mark.parametrize("D", [16, 48, 64, 80, 128, 256])
@pytest.mark.parametrize("is_key", [True, False])
def test_tiles_hold_every_code_and_scale_once(D, is_key):
    byte, shift, sc = R.tile_index(D, is_key)
    cells = sorted((byte * 2 + shift // 4).ravel().tolist())
    assert cells == list(range(16 * D))
    assert sorted(sc.ravel().tolist()) == list(range(8 * D, 9 * D))
    rng = np.random.default_rng(D)
    codes = rng.integers(0, 16, (2, 3, 32, D)).astype(np.uint8)
    sb = rng.integers(0, 127, (2, 3, 32, D // 16)).astype(np.uint8)
    c2, s2 = R.unpack(R.pack(codes, sb, is_key), is_key)
    np.testing.assert_array_equal(c2, codes)
    np.testing.assert_array_equal(s2, sb)


def test_nan_infinity_zero_and_saturation():
    x = np.zeros((1, 64), np.float16)
    x[0, 0] = np.nan
    x[0, 16] = np.inf
    x[0, 17] = 100.0
    x[0, 32] = 65504.0
    x[0, 48] = 2.0 ** -24
    c, s = R.encode(x, 1.0)
    v = R.values(c, s, 1.0)
    assert not v[0, :16].any()
    assert v[0, 16] == 6 * 448 and v[0, 17] == 0.0
    assert v[0, 32] == 6 * 448
    assert not v[0, 48:].any()  # below the smallest scale


# ── refusals (nothing is launched: the addresses are never read) ─────────
F = 1 << 20  # an aligned address


def _write(lib, key=F, value=F, kc=F, vc=F, slots=F, T=4, hkv=2, d=64, bs=16, ks=1.0, vs=1.0,
           kbs=2 * 576, khs=576, ts=128, read=False):
    fn = lib.nxt_read_cache_q4 if read else lib.nxt_reshape_and_cache_q4
    return fn(key, value, kc, vc, slots, T, hkv, d, bs, ks, vs, kbs, khs, ts, 8, None)


BAD_ROWS = [dict(key=None), dict(value=None), dict(kc=None), dict(vc=None), dict(slots=None),
            dict(T=-1), dict(hkv=0), dict(d=0), dict(d=24), dict(d=272), dict(bs=8), dict(bs=0),
            dict(ks=0.0), dict(vs=float("inf")), dict(ks=float("nan")), dict(ks=-1.0),
            dict(kc=F + 8), dict(vc=F + 1), dict(kbs=1160), dict(khs=584), dict(kbs=-16),
            dict(ts=127), dict(key=F + 1), dict(T=2 ** 31 - 1, hkv=2)]


@pytest.mark.parametrize("read", [False, True])
@pytest.mark.parametrize("bad", BAD_ROWS, ids=str)
def test_row_calls_refuse(bad, read):
    assert _write(_native.xpa(), read=read, **bad) == _native.NXT_PA_EINVAL


@pytest.mark.parametrize("read", [False, True])
def test_row_calls_without_tokens_do_nothing(read):
    assert _write(_native.xpa(), read=read, T=0, key=None) == _native.NXT_PA_OK


def _attend(lib, append=False, out=F, q=F, kc=F, vc=F, bt=F, sl=F, B=2, hq=4, d=64, hkv=2, mb=4,
            bs=16, ks=1.0, vs=1.0, kbs=2 * 576, khs=576, ws=None, nk=F, nv=F, slots=F):
    if append:
        return lib.nxt_paged_attention_q4_append_ex(out, q, kc, vc, bt, sl, nk, nv, slots, B, hq, d,
                                                    hkv, 0.1, mb, bs, ks, vs, kbs, khs, 8, None, None)
    return lib.nxt_paged_attention_q4_ex(out, q, kc, vc, bt, sl, B, hq, d, hkv, 0.1, mb, bs, ks, vs,
                                         kbs, khs, 8, ws, 0, None, None)


BAD_CALLS = [dict(out=None), dict(q=None), dict(kc=None), dict(vc=None), dict(bt=None),
             dict(sl=None), dict(B=-1), dict(hq=3), dict(hkv=0), dict(d=72), dict(d=272),
             dict(mb=-1), dict(bs=24), dict(ks=0.0), dict(vs=float("nan")), dict(kc=F + 4),
             dict(kbs=1153), dict(khs=8), dict(q=F + 1), dict(out=F + 1)]


@pytest.mark.parametrize("append", [False, True])
@pytest.mark.parametrize("bad", BAD_CALLS, ids=str)
def test_attention_refuses(bad, append):
    assert _attend(_native.xpa(), append=append, **bad) == _native.NXT_PA_EINVAL


def test_attention_refuses_a_misaligned_workspace():
    assert _attend(_native.xpa(), ws=F + 8) == _native.NXT_PA_EINVAL


@pytest.mark.parametrize("append", [False, True])
def test_attention_over_no_sequences_does_nothing(append):
    assert _attend(_native.xpa(), append=append, B=0, q=None) == _native.NXT_PA_OK


def test_workspace_query_of_nonsense_is_zero():
    lib = _native.xpa()
    assert lib.nxt_paged_attention_q4_workspace_size(0, 1, 64, 1, 1, 16) == 0
    assert lib.nxt_paged_attention_q4_workspace_size(1, 1, 64, 1, 1, 0) == 0


def test_python_wrappers_refuse_host_and_misshapen_tensors():
    pool = torch.zeros(PA.q4_pool_shape(4, 2, 16, 64), dtype=torch.uint8)
    row = torch.zeros(3, 2, 64, dtype=torch.float16)
    slots = torch.zeros(3, dtype=torch.int64)
    with pytest.raises(PA.PagedAttentionError):
        PA.reshape_and_cache_q4(row, row, pool, pool, slots, 1.0, 1.0)
    with pytest.raises(PA.PagedAttentionError):
        PA.read_cache_q4(pool, pool, slots, 1.0, 1.0)
    q = torch.zeros(1, 4, 64, dtype=torch.float16)
    t, n = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(PA.PagedAttentionError):
        PA.paged_attention_q4(q, pool, pool, t, n, 1.0, 1.0)
    for shape in ((4, 2, 8, 64), (4, 2, 16, 40), (4, 2, 16, 272)):
        with pytest.raises(PA.PagedAttentionError):
            PA.q4_pool_shape(*shape)


def test_argument_lists_match_the_header():
    for name in ("nxt_reshape_and_cache_q4", "nxt_read_cache_q4", "nxt_paged_attention_q4_ex",
                 "nxt_paged_attention_q4_append_ex"):
        assert name in _native.SIGNATURES
        assert isinstance(getattr(_native.xpa(), name), ctypes._CFuncPtr)
