"""CPU checks of the batch step's entry points at the edges of their arguments (a call without a context reaches the checks)."""
import ctypes as C

import pytest

from rabbit_amd import abi
from rabbit_amd.abi import RBT_E_INVALID
from test_batch import _rows
from test_drafts import A, _refused


@pytest.mark.parametrize("off", [1, 2, 3])
@pytest.mark.parametrize("which", ["plen", "first", "len", "n", "parent"])
def test_prefix_refuses_misaligned_numbers(rbt_lib, which, off):
    d = abi.RbtGqaPrefixDesc(8, 4, 64, 0.125, 0, 100, 0, 50, 0, 0, 0)
    r = C.byref(_rows())
    a = dict(B=2, T=3, G=2, q=A, prefix=r, cache=r, draft=r, plen=A, first=A, len=A, n=A, parent=A, gate=None, out=A)
    _refused(rbt_lib, rbt_lib.rbt_gqa_prefix_d(None, C.byref(d), *{**a, which: A + off}.values()), RBT_E_INVALID, "aligned")
    rc = rbt_lib.rbt_gqa_prefix_d(None, C.byref(d), *{**a, which: A + 4}.values())
    _refused(rbt_lib, rc, RBT_E_INVALID, "null context")
    if which in ("plen", "first"):  # not used without prefixes
        rc = rbt_lib.rbt_gqa_prefix_d(None, C.byref(d), *{**a, which: A + off, "G": 0, "prefix": None}.values())
        _refused(rbt_lib, rc, RBT_E_INVALID, "null context")


@pytest.mark.parametrize("rows,row,seq", [((1 << 25) + 1, 1 << 39, 1 << 40), ((1 << 24) + 1, 1 << 40, 1 << 40), ((1 << 30) + 1, 1 << 36, 1 << 37)])
def test_read_back_spans_past_64_bits(rbt_lib, rows, row, seq):
    """Rows whose span is 2^64 entries and a few: the next sequence begins inside it."""
    d, r = abi.RbtKvQuantDesc(1, 64, (1 << 31) - 1, 0, seq, row, 64), _rows()
    _refused(rbt_lib, rbt_lib.rbt_kv_dequant_d(None, C.byref(d), 2, rows, C.byref(r), A, A, A, 2 * A), RBT_E_INVALID, "result rows overlap")
    _refused(rbt_lib, rbt_lib.rbt_kv_dequant_d(None, C.byref(d), 1, rows, C.byref(r), A, A, A, 2 * A), RBT_E_INVALID, "null context")
