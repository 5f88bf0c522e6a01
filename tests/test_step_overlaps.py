"""Tensors of a step that share memory: what is written twice, or read by one workgroup after another has written it, has
no one result.  Refused before anything touches a GPU."""

import ctypes

import pytest
import torch

from axonn_amd import _native as nv

# A call that is not refused here is one that has no GPU to launch on.
pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are made up")

A = 0x100000000   # addresses that are never dereferenced: without a GPU nothing is launched
SIZES = (600, 40)
LISTS = {"g": 0, "p": 1, "m": 2, "v": 3, "low": 4}


def call(name, change=None, sizes=SIZES, gdt=nv.BF16):
    """The status, and the error's text, of a step over lists that are far apart but for `change`: {(list, index): address}."""
    lib = nv.load()
    at = [[A * (1 + 2 * i), A * (1 + 2 * i) + (1 << 24)] for i in range(5)]
    for (which, i), address in (change or {}).items():
        at[LISTS[which]][i] = address
    hp = nv.AdamWHParams()
    tail = (0, None, hp, None) if name.endswith("8") else (None, hp, None)
    rc = getattr(lib, name)(*((ctypes.c_void_p * 2)(*p) for p in at), (ctypes.c_int64 * 2)(*sizes), 2, gdt, nv.BF16, 1.0, *tail)
    return rc, lib.axn_last_error().decode()


def place(which, i=0):
    return A * (1 + 2 * LISTS[which]) + i * (1 << 24)


def nbytes(name, which, i, gdt=nv.BF16):
    n = SIZES[i]
    if which in "mv" and name.endswith("8"):
        return -(-n // 256) * (512 if which == "m" else 2)
    return n * (2 if which == "low" or (which == "g" and gdt == nv.BF16) else 4)


PAIRS = [(a, b) for a in LISTS for b in LISTS if a < b]


def refused(rc, text):
    return rc == nv.AXN_EINVAL and "overlap" in text


@pytest.mark.parametrize("a,b", PAIRS)
@pytest.mark.parametrize("name", ["axn_mt_adamw", "axn_mt_adamw8"])
def test_lists_that_overlap_are_refused(name, a, b):
    """By their first or last bytes, one inside the other, and the same place for two different tensors."""
    names = {"m": "codes", "v": "exponents", "low": "p_lowp"} if name.endswith("8") else {"low": "p_lowp"}
    for i, j in ((0, 0), (0, 1), (1, 0), (1, 1)):
        for first, second, k, l in ((a, b, i, j), (b, a, i, j)):
            here, size, other = place(first, k), nbytes(name, first, k), nbytes(name, second, l)
            inside = [here + size - 8, here - other + 8] + ([here + 16] if size > 16 + other else [])
            if k != l:
                inside.append(here)
            for address in inside:
                address -= address % 8       # (as every list's alignment asks, and still inside)
                if not here - other < address < here + size:
                    continue
                rc, text = call(name, {(second, l): address})
                assert refused(rc, text) and names.get(a, a) in text and names.get(b, b) in text, (first, second, k, l, rc, text)
            # end to end
            rc, text = call(name, {(second, l): here + -(-size // 8) * 8})
            assert not refused(rc, text), text


def test_a_gradient_may_be_where_its_own_copy_is():
    """Element for element in one place: a lane reads its gradient before it writes the copy there, or the weight."""
    for name in ("axn_mt_adamw", "axn_mt_adamw8"):
        assert not refused(*call(name, {("low", i): place("g", i) for i in (0, 1)}))
        assert not refused(*call(name, {("p", i): place("g", i) for i in (0, 1)}, gdt=nv.F32))
        assert refused(*call(name, {("low", 0): place("g", 1), ("low", 1): place("g", 0)}, sizes=(40, 40)))
        assert refused(*call(name, {("p", i): place("g", i) for i in (0, 1)}))                  # (of another width)
        assert refused(*call(name, {("m", i): place("g", i) for i in (0, 1)}, gdt=nv.F32))
        assert refused(*call(name, {("low", 0): place("p", 0)}))


def test_empty_tensors_overlap_nothing():
    for name in ("axn_mt_adamw", "axn_mt_adamw8"):
        assert not refused(*call(name, {(w, 1): place("p") + 64 for w in LISTS}, sizes=(600, 0)))
