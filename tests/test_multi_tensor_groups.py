"""How a list of tensors is cut into launches (csrc/multi_tensor.h), on the host: a dimension of a launch takes fewer
than 2^32 threads, and more of them wrap without an error, so that a part of the elements would be left as it was."""

import ctypes
import os
import subprocess

import pytest

from axonn_amd import _native as nv

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
A = 1 << 50   # addresses that are never dereferenced

SOURCE = r"""
#include "multi_tensor.h"
namespace axn { void set_error(const char*, ...) {} }
// first[i], count[i]: of launch i its first tensor's size and its workgroups; the number of launches, or the status
extern "C" int groups(const long long* at, const int64_t* sizes, int64_t n, int chunk, int threads, int64_t* first, int64_t* count) {
  const void* const* sets[1] = {(const void* const*)at};
  const int es[1] = {4};
  int used = 0;
  const int rc = axn::for_each_group(sets, es, 1, sizes, n, chunk, threads, [&](const axn::Group& g) {
    first[used] = g.tab.size[0];
    count[used++] = g.blocks;
    return 0;
  });
  return rc ? rc : used;
}
"""


@pytest.fixture(scope="module")
def groups(tmp_path_factory):
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not available")
    folder = tmp_path_factory.mktemp("groups")
    (folder / "groups.hip").write_text(SOURCE)
    subprocess.run([HIPCC, "--cuda-host-only", "-O1", "-std=c++17", "-fPIC", "-shared", "-I" + os.path.join(ROOT, "include"),
                    "-I" + os.path.join(ROOT, "axonn_amd", "csrc"), str(folder / "groups.hip"), "-o", str(folder / "groups.so")],
                   check=True, capture_output=True, timeout=600)
    lib = ctypes.CDLL(str(folder / "groups.so"))

    def call(sizes, chunk, threads):
        n = len(sizes)
        at = (ctypes.c_longlong * n)(*(A + (i << 40) for i in range(n)))
        first, count = (ctypes.c_int64 * n)(), (ctypes.c_int64 * n)()
        rc = lib.groups(at, (ctypes.c_int64 * n)(*sizes), ctypes.c_int64(n), chunk, threads, first, count)
        return rc if rc < 0 else list(zip(first[:rc], count[:rc]))

    return call


@pytest.mark.parametrize("chunk,threads", [(256, 64), (65536, 256), (16384, 256)])
def test_launches_stay_below_2_to_the_32_threads(groups, chunk, threads):
    most = ((1 << 32) - 1) // threads          # workgroups
    quarter = (most // 4 + 1) * chunk          # elements: three of them fit, four do not
    assert groups([quarter] * 3, chunk, threads) == [(quarter, 3 * (most // 4 + 1))]
    found = groups([quarter + i for i in range(-6, 0)], chunk, threads)
    assert [f for f, _ in found] == [quarter - 6, quarter - 3] and all(c * threads < 1 << 32 for _, c in found)
    assert sum(c for _, c in found) == 6 * (most // 4 + 1)
    assert groups([most * chunk], chunk, threads) == [(most * chunk, most)]
    assert groups([5, most * chunk], chunk, threads) == [(5, 1), (most * chunk, most)]
    assert groups([most * chunk + 1], chunk, threads) == nv.AXN_ELIMIT
    assert groups([7] * 64, chunk, threads) == [(7, 64)] and groups([7] * 65, chunk, threads) == [(7, 64), (7, 1)]


@pytest.mark.parametrize("name", ["axn_mt_adam", "axn_mt_adamw"])
def test_a_tensor_beyond_a_launch_is_refused(name):
    """Before anything touches a GPU."""
    lib, hp = nv.load(), (nv.AdamWHParams if name.endswith("w") else nv.AdamHParams)()
    lists = [(ctypes.c_void_p * 1)(A + (i << 40)) for i in range(4)]
    rc = getattr(lib, name)(*lists, None, (ctypes.c_int64 * 1)(1 << 34), 1, nv.BF16, nv.BF16, 1.0, None, hp, None)
    assert rc == nv.AXN_ELIMIT and "too many elements" in lib.axn_last_error().decode()
