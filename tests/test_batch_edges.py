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
