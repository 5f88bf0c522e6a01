"""The entry points of include/axn_ext.h: declared, bound and exported alike, and their
refusals, which come before anything touches a GPU (so all of this runs without one)."""

import ctypes
import os
import re
import zlib

import pytest
import torch

from axonn_amd import _native as nv
from axonn_amd import ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
A = 0x10000000   # addresses that are never dereferenced: the checks fail first


def header():
    return open(os.path.join(ROOT, "include", "axn_ext.h")).read()


def err():
    return nv.load().axn_last_error().decode()


def test_header_binding_and_library_agree():
    names = set(re.findall(r"AXN_API\s+[\w\s\*]+?\b(axn_[a-z0-9_]+)\s*\(", header()))
    assert names == set(nv.EXT_SYMBOLS) and not names & set(nv.SYMBOLS)
    lib = ctypes.CDLL(nv.lib_path())
    assert all(hasattr(lib, name) for name in names)
    assert nv.load().axn_ext_abi_version() == nv.EXT_ABI_VERSION
    assert int(re.search(r"AXN_ADAMW8_BLOCK (\d+)", header()).group(1)) == nv.ADAMW8_BLOCK
    assert ctypes.sizeof(nv.AdamWHParams) == 28


def test_the_version_goes_with_the_declarations():
    text = re.sub(r"#define AXN_EXT_ABI_VERSION[^\n]*", "", re.sub(r"/\*.*?\*/", " ", header(), flags=re.S))
    assert (nv.EXT_ABI_VERSION, "%08x" % zlib.crc32(" ".join(text.split()).encode())) == (1, "2647fe52")


def test_norm_refusals():
    f = nv.load().axn_layer_norm_fwd

    def call(x=A, r=None, w=A, b=A, y=A, h=None, mean=A, rstd=A, dt=nv.BF16, pdt=nv.BF16, M=4, N=16, ldx=16, ldr=16,
             eps=1e-5):
        return f(x, r, w, b, y, h, mean, rstd, dt, pdt, M, N, ldx, ldr, eps, None)

    assert call(x=None) == nv.AXN_EINVAL and "x is null" in err()
    assert call(y=None) == nv.AXN_EINVAL
    assert call(dt=7) == nv.AXN_EINVAL
    assert call(pdt=nv.F16) == nv.AXN_EINVAL and "parameters" in err()
    assert call(dt=nv.F32, pdt=nv.BF16) == nv.AXN_EINVAL
    assert call(M=-1) == nv.AXN_EINVAL and call(N=0) == nv.AXN_EINVAL
    assert call(M=1 << 31) == nv.AXN_ELIMIT and call(N=1 << 31, ldx=1 << 31) == nv.AXN_ELIMIT
    assert call(ldx=15) == nv.AXN_EINVAL and "stride" in err()
    assert call(r=A) == nv.AXN_EINVAL and call(h=A) == nv.AXN_EINVAL and "together" in err()
    assert call(r=A, h=A, ldr=15) == nv.AXN_EINVAL and "residual" in err()
    assert call(mean=None) == nv.AXN_EINVAL and call(rstd=None) == nv.AXN_EINVAL
    assert call(eps=-1.0) == nv.AXN_EINVAL and call(eps=float("nan")) == nv.AXN_EINVAL
    for what in ("x", "y"):
        assert call(**{what: A + 1}) == nv.AXN_EALIGN and what in err()
    for what in ("w", "b", "mean", "rstd"):
        assert call(pdt=nv.F32, **{what: A + 2}) == nv.AXN_EALIGN
    assert call(M=0, x=None, y=None) == nv.AXN_OK   # nothing to do


def test_norm_gradient_refusals():
    f = nv.load().axn_layer_norm_bwd
    need = nv.load().axn_layer_norm_bwd_workspace_bytes(600, 16)
    assert need >= 2 * 16 * 4

    def call(dy=A, h=A, w=A, mean=A, rstd=A, dsum=None, dx=A, dw=A, db=A, dt=nv.BF16, pdt=nv.BF16, M=600, N=16, lddy=16,
             ldh=16, ldsum=16, ws=A, nbytes=need):
        return f(dy, h, w, mean, rstd, dsum, dx, dw, db, dt, pdt, M, N, lddy, ldh, ldsum, ws, nbytes, None)

    assert call(dy=None) == nv.AXN_EINVAL and call(h=None) == nv.AXN_EINVAL
    assert call(mean=None) == nv.AXN_EINVAL and call(rstd=None) == nv.AXN_EINVAL
    assert call(dx=None, dw=None, db=None) == nv.AXN_EINVAL and "nothing" in err()
    assert call(lddy=8) == nv.AXN_EINVAL and call(ldh=8) == nv.AXN_EINVAL and call(dsum=A, ldsum=8) == nv.AXN_EINVAL
    assert call(ws=None) == nv.AXN_EINVAL and call(nbytes=need - 1) == nv.AXN_EINVAL and "workspace" in err()
    assert call(ws=A + 8) == nv.AXN_EALIGN
    assert call(dy=A + 1) == nv.AXN_EALIGN and call(dx=A + 1) == nv.AXN_EALIGN and call(dw=A + 1) == nv.AXN_EALIGN
    assert call(dt=nv.F16, pdt=nv.BF16) == nv.AXN_EINVAL and call(N=0) == nv.AXN_EINVAL and call(M=-1) == nv.AXN_EINVAL
    assert call(M=0, dw=None, db=None) == nv.AXN_OK
    q = nv.load().axn_layer_norm_bwd_workspace_bytes
    assert q(0, 16) == q(4, 0) == q(-1, 16) == q(1 << 31, 16) == q(512, 16) == 0 < q(513, 16)   # (few rows need none)


@pytest.mark.parametrize("name", ["axn_mt_adamw", "axn_mt_adamw8"])
def test_step_refusals(name):
    f, eight = getattr(nv.load(), name), name.endswith("8")

    def arr(*p):
        return (ctypes.c_void_p * len(p))(*p)

    def call(g=None, p=None, m=None, v=None, low=None, sizes=(4, 600), n=2, gdt=nv.BF16, pdt=nv.BF16, hp=nv.AdamWHParams()):
        far = [arr(A * i, A * i + (1 << 24)) for i in range(1, 5)]
        tail = (0, None, hp, None) if eight else (None, hp, None)
        return f(g or far[0], p or far[1], m or far[2], v or far[3], low, (ctypes.c_int64 * 2)(*sizes), n, gdt, pdt, 1.0,
                 *tail)

    assert call(hp=None) == nv.AXN_EINVAL and "hyper" in err()
    assert call(gdt=9) == nv.AXN_EINVAL and call(n=-1) == nv.AXN_EINVAL and call(sizes=(-1, 4)) == nv.AXN_EINVAL
    assert call(low=arr(A, 2 * A), pdt=nv.F32) == nv.AXN_EINVAL
    assert call(g=arr(A, None)) == nv.AXN_EINVAL and "g[1] is null" in err()
    assert call(p=arr(A + 2, 2 * A)) == nv.AXN_EALIGN and call(g=arr(A + 1, 2 * A)) == nv.AXN_EALIGN
    # tensors that share elements, in either order, and one that is there twice
    for second in (A, A + 12, A - 2396):
        assert call(p=arr(A, second)) == nv.AXN_EINVAL and "overlap" in err(), second
    assert call(low=arr(A, A + 6)) == nv.AXN_EINVAL and "p_lowp overlap" in err()
    if eight:
        assert call(m=arr(A + 4, 2 * A)) == nv.AXN_EALIGN and call(v=arr(A + 1, 2 * A)) == nv.AXN_EALIGN
        assert call(m=arr(A, A + 504)) == nv.AXN_EINVAL and "codes overlap" in err()
        assert call(v=arr(A, A - 4)) == nv.AXN_EINVAL and "exponents overlap" in err()
        assert call(sizes=(4, 1 << 34)) == nv.AXN_ELIMIT
    else:
        assert call(m=arr(A, A + 12)) == nv.AXN_EINVAL and call(v=arr(A, A + 12)) == nv.AXN_EINVAL
    # an empty tensor may carry any pointer, and the same as another
    assert call(p=arr(None, None), sizes=(0, 0)) == nv.AXN_OK
    assert call(n=0) == nv.AXN_OK


def test_moments_refusals():
    f = nv.load().axn_adamw8_moments
    assert f(A, A, A, A, nv.F16, 8, None) == nv.AXN_EINVAL
    assert f(A, A, None, None, nv.F32, 8, None) == nv.AXN_EINVAL
    assert f(None, A, A, A, nv.F32, 8, None) == nv.AXN_EINVAL
    assert f(A, A, A, A, nv.F32, -1, None) == nv.AXN_EINVAL
    assert f(A + 4, A, A, A, nv.F32, 8, None) == nv.AXN_EALIGN and f(A, A, A + 2, A, nv.F32, 8, None) == nv.AXN_EALIGN
    assert f(A, A, A, A, nv.F32, 1 << 40, None) == nv.AXN_ELIMIT
    assert f(None, None, A, A, nv.F32, 0, None) == nv.AXN_OK


def test_cpu_tensors_are_refused():
    from axonn_amd.intra_layer import LayerNorm
    from axonn_amd.optim import AdamW

    x = torch.zeros(2, 8)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.layer_norm_fwd(x)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.layer_norm_bwd(x, x, None, x[:, 0], x[:, 0])
    with pytest.raises(RuntimeError, match="GPU"):
        LayerNorm(8)(x)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.mt_adamw([x], [x], [x], [x], None, ops.adamw_hparams(1, 1e-3, 0.9, 0.999, 1e-8, 0.0))
    codes, exponents = ops.adamw8_state(16, "cpu")
    with pytest.raises(RuntimeError, match="GPU"):
        ops.mt_adamw8([x], [x], [codes], [exponents], None, ops.adamw_hparams(1, 1e-3, 0.9, 0.999, 1e-8, 0.0), 0)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.adamw8_moments(codes, exponents)
    with pytest.raises(RuntimeError, match="GPU"):
        AdamW([torch.nn.Parameter(torch.zeros(8))])


def test_optimizer_arguments():
    from axonn_amd.optim import AdamW

    p = [torch.nn.Parameter(torch.zeros(8))]
    for bad in (dict(state_bits=16), dict(state_bits=8, eps=0.0), dict(lr=-1.0), dict(eps=-1.0), dict(betas=(1.0, 0.9)),
                dict(betas=(0.9, 1.0)), dict(weight_decay=-0.1)):
        with pytest.raises(ValueError, match="[Ii]nvalid|positive"):
            AdamW(p, **bad)


def test_module_arguments():
    from axonn_amd.intra_layer import LayerNorm, layer_norm

    a, b = LayerNorm((3, 4)), torch.nn.LayerNorm((3, 4))
    assert {k: v.shape for k, v in a.state_dict().items()} == {k: v.shape for k, v in b.state_dict().items()}
    a.load_state_dict(b.state_dict())
    assert LayerNorm(4, bias=False).bias is None and not list(LayerNorm(4, elementwise_affine=False).parameters())
    with pytest.raises(ValueError, match="last dimensions"):
        a(torch.zeros(2, 4, 3))
    with pytest.raises(ValueError, match="residual"):
        a(torch.zeros(2, 3, 4), torch.zeros(1, 3, 4))
    with pytest.raises(ValueError, match="parameter"):
        layer_norm(torch.zeros(2, 4), 4, torch.ones(3))
