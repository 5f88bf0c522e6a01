"""Generated gfx950 code of the layer norm and AdamW kernels: registers, memory accesses and their
order, as the measured figures beside the kernels rest on them."""

import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "axonn_amd", "csrc")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not available")
    found = {}
    for name in ("adamw", "layer_norm"):
        out = tmp_path_factory.mktemp("asm") / (name + ".s")
        subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang", "-target-feature", "-Xclang",
                        "-packed-fp32-ops", "-I" + os.path.join(ROOT, "include"), "-I" + CSRC, "--cuda-device-only", "-S",
                        os.path.join(CSRC, name + ".hip"), "-o", str(out)], check=True, capture_output=True, timeout=900)
        text = out.read_text()
        for m in re.finditer(r"^(_ZN\S+):\s", text, re.M):
            end = text.find(".end_amdhsa_kernel", m.end())
            if end > 0 and ".amdhsa_kernel" in text[m.end():end]:
                found[m.group(1)] = text[m.end():end]
    return found


def instructions(body):
    return [s for s in (line.split(";")[0].strip() for line in body.split("\n")) if s and not s.startswith(".")]


def number(body, what):
    return int(re.search(r"\.amdhsa_%s (\d+)" % what, body).group(1))


def test_no_packed_arithmetic(kernels):
    assert len(kernels) > 50
    for name, body in kernels.items():
        assert not re.search(r"\bv_pk_(add|mul|fma)_f32", body), name


def test_update_of_8_bit_moments(kernels):
    """No spills, 32 registers at most, the streams by buffer accesses past the caches, all of their loads in front of the first
    store."""
    mine = {k: v for k, v in kernels.items() if "mt_adamw8_kernel" in k}
    assert len(mine) == 18   # 3 gradient types x (no copy, bf16, fp16) x with/without scan result
    for name, body in mine.items():
        assert number(body, "private_segment_fixed_size") == 0 and number(body, "next_free_vgpr") <= 32, name
        ins = instructions(body)
        loads = [i for i, s in enumerate(ins) if s.startswith("buffer_load_dwordx")]
        stores = [i for i, s in enumerate(ins) if s.startswith("buffer_store_dwordx")]
        assert len(loads) == 3 and len(stores) in (2, 3) and max(loads) < min(stores), name
        assert all(ins[i].endswith(" nt") for i in loads) and all(ins[i].endswith(" nt sc1") for i in stores), name


def test_update_in_fp32_is_the_shared_one(kernels):
    mine = {k: v for k, v in kernels.items() if "mt_adamw_kernel" in k}
    assert len(mine) == 18
    for name, body in mine.items():
        ins = instructions(body)
        loads = [i for i, s in enumerate(ins) if s.startswith("buffer_load_dwordx")]
        stores = [i for i, s in enumerate(ins) if s.startswith("buffer_store_dwordx")]
        assert number(body, "private_segment_fixed_size") == 0 and len(loads) == 4 and max(loads) < min(stores), name


def test_norm_kernels_hold_their_rows_in_registers(kernels):
    """Rows in 16-byte accesses wherever they start; no spills but where a lane has four vectors of 16-bit elements, a
    workgroup of 16 waves 128 registers each."""
    for which, template in (("norm_rows_kernel", r"norm_rows_kernelI(\w+?)Li(\d)E"), ("norm_grad_rows_kernel", r"norm_grad_rows_kernelI(\w+?)Li(\d)E")):
        mine = {k: v for k, v in kernels.items() if re.search(r"\d" + which, k)}
        assert len(mine) >= 12
        for name, body in mine.items():
            k = int(re.search(template, name).group(2))
            assert number(body, "next_free_vgpr") <= 128, name
            spilled = number(body, "private_segment_fixed_size")
            assert spilled == 0 or k == 4 or (spilled <= 32 and k == 2), (name, spilled)
            assert not re.search(r"global_load_(u|s)(short|byte)", body), name
