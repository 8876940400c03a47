"""Refusals of calls over 4-bit pools that depend on several sizes, without a GPU."""
import pytest

from xllms_b200 import _native

F = 1 << 20  # an aligned address; nothing is launched, so it is never read


def _sparse(nb, hkv=2, d=64, kbs=1184, khs=592):
    return _native.xpa().nxt_paged_attention_q4_sparse_ex(
        F, F, F, F, F, F, F, None, 2, 4, d, hkv, 0.1, 40, 16, 1.0, 1.0, kbs, khs, nb, 8, 1, 2, None, 0,
        F, None)


def _dense(nb, hkv=2, d=64, kbs=1168, khs=576):
    return _native.xpa().nxt_paged_attention_q4_ex(
        F, F, F, F, F, F, 2, 4, d, hkv, 0.1, 40, 16, 1.0, 1.0, kbs, khs, nb, None, 0, F, None)


# A page of 1184 bytes in units of 16, the most that divides 576 too: two heads of 37
# units each. Ids of the 2^26 pages' heads and of their tiles stay below 2^32 units.
LAST = (2 ** 32 - 2 - 36) // 37 // 2


@pytest.mark.parametrize("nb", [LAST + 1, 2 ** 30, 2 ** 31, 2 ** 40])
def test_sparse_calls_refuse_pools_past_their_addresses_before_any_launch(nb):
    assert _sparse(nb) == _native.NXT_PA_EINVAL


def test_pools_within_the_addresses_are_not_refused():
    """They get as far as the device, which is not there or not asked for memory."""
    import torch
    if torch.cuda.is_available():
        pytest.skip("would launch over addresses that are not there")
    assert _sparse(LAST) == _native.NXT_PA_ECUDA
    assert _sparse(2 ** 31 - 1, kbs=1152, khs=576) == _native.NXT_PA_ECUDA  # whole tiles
    assert _sparse(-1) == _native.NXT_PA_ECUDA
    assert _dense((2 ** 32 - 2 - 36) // 73 + 1) == _native.NXT_PA_ECUDA


@pytest.mark.parametrize("nb", [(2 ** 32 - 2 - 36) // 73 + 2, 2 ** 40, 2 ** 62])
def test_dense_calls_refuse_the_same(nb):
    assert _dense(nb) == _native.NXT_PA_EINVAL


@pytest.mark.parametrize("rows,heads,D,tiles,split", [
    (1, 8, 128, 24, False), (1, 8, 128, 25, True), (1, 8, 128, 32, True), (6, 8, 128, 32, True),
    (6, 8, 64, 48, False), (1, 1, 64, 49, True), (1, 8, 256, 24, False), (1, 8, 256, 32, True),
    (1, 8, 16, 48, False), (16, 8, 128, 32, False), (16, 8, 128, 48, False), (16, 8, 128, 49, True),
    (48, 8, 256, 48, False)])
def test_short_rows_are_split_only_where_they_are_few(rows, heads, D, tiles, split):
    """A call whose rows all stay whole asks for no workspace."""
    need = _native.xpa().nxt_paged_attention_q4_workspace_size(rows, heads, D, heads, tiles, 16)
    assert (need > 0) == split
