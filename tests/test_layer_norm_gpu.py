"""Layer norm on the GPU against the formulas in 64 bits (oracle/layer_norm.py).

Tolerances.  A value computed in fp32 and rounded to T is off by half a step of T, eps(T) / 2 of
itself, and by the fp32 arithmetic: sums of n terms added in chains of c are off by at most
c 2^-24 of the sum of magnitudes, everything else is a handful of roundings of its operands.
"""

import numpy as np
import pytest
import torch

from oracle import layer_norm as ol

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
U = 2.0 ** -24
EPS = 1e-5


def f64(t):
    return None if t is None else t.detach().double().cpu().numpy()


def half_step(t):
    """Half a step of type t, relative (nothing for what the comparison holds in 64 bits), and its smallest."""
    return torch.finfo(t).eps / 2, torch.finfo(t).tiny * torch.finfo(t).eps / 2


def chain(n):
    """Additions one after another in a row's sums: at most n / 64 + 32 in a lane, and 16 to join lanes and waves."""
    return n / 64 + 48


def check(got, want, dtype, work, what):
    """|got - want| <= half a step of dtype + work, elementwise."""
    rel, least = half_step(dtype)
    got = f64(got)
    # the rounding is of the computed value, which `work` may take further than want
    bound = work + rel * (np.abs(want) + work) + least
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (what, int(bad.sum()), got[bad][:3], want[bad][:3], bound[bad][:3])


def make(M, N, dtype, params="same", seed=0, residual=False, x_offset=0.3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    param = torch.float32 if params == "fp32" else dtype
    x = (torch.randn(M, N, generator=g, device="cuda") * 2 + x_offset).to(dtype)
    r = torch.randn(M, N, generator=g, device="cuda").to(dtype) if residual else None
    w = b = None
    if params != "none":
        w = (1 + 0.2 * torch.randn(N, generator=g, device="cuda")).to(param)
        b = (0.2 * torch.randn(N, generator=g, device="cuda")).to(param)
    dy = torch.randn(M, N, generator=g, device="cuda").to(dtype)
    ds = torch.randn(M, N, generator=g, device="cuda").to(dtype) if residual else None
    return x, r, w, b, dy, ds


def check_forward(y, mean, rstd, h, w, b, dtype, eps=EPS):
    hn, wn, bn = f64(h), f64(w), f64(b)
    N = hn.shape[1]
    want, m64, s64 = ol.forward(hn, wn, bn, eps)
    c = chain(N)
    size = np.abs(hn).mean(1)
    spread = ((hn - m64[:, None]) ** 2).mean(1)
    off_mean = (c + 2) * U * size
    # var: chains over squares, a few roundings each, and the mean's error, which counts squared
    off_var = (c + 6) * U * spread + 4 * off_mean * U * size + off_mean ** 2
    off_rstd = s64 * (off_var / (2 * (spread + eps)) + 4 * U)
    if mean is not None:
        check(mean, m64, torch.float32, off_mean, "mean")
        check(rstd, s64, torch.float32, off_rstd, "rstd")
    a = np.abs(wn) if wn is not None else 1.0
    d = np.abs(hn - m64[:, None])
    work = a * (s64[:, None] * off_mean[:, None] + d * off_rstd[:, None] + 4 * U * d * s64[:, None])
    work += 2 * U * (np.abs(want) + (0 if bn is None else np.abs(bn)))
    check(y, want, dtype, work, "y")


def check_backward(got, dy, h, w, mean, rstd, ds, dtype):
    dx, dw, db = got
    M, N = dy.shape
    d64, h64, w64, m64, s64, e64 = (f64(t) for t in (dy, h, w, mean, rstd, ds))
    wx, ww, wb = ol.backward(d64, h64, w64, m64, s64, e64)
    xhat = np.abs((h64 - m64[:, None]) * s64[:, None])
    a = np.abs(d64 if w64 is None else d64 * w64)
    c = chain(N)
    if dx is not None:
        work = s64[:, None] * ((c + 8) * U * (a.mean(1) [:, None] + xhat * (a * xhat).mean(1)[:, None]) + 8 * U * a)
        work = work + (0 if e64 is None else 2 * U * np.abs(e64)) + 2 * U * np.abs(wx)
        check(dx, wx, dtype, work, "dx")
    # rows per workgroup one after another (16 at least, or M / 256 where that is more), at most 256 parts, 16 to join
    rows = max(16, -(-M // 256)) + min(256, M) + 16
    for got_, want, terms, what in ((dw, ww, np.abs(d64) * xhat, "dweight"), (db, wb, np.abs(d64), "dbias")):
        if got_ is not None:
            check(got_, want, got_.dtype, (rows + 4) * U * terms.sum(0), what)


SIZES = [(1, 1), (3, 2), (2, 7), (5, 8), (7, 63), (16, 64), (9, 100), (4, 129), (33, 256), (3, 1000), (17, 1025),
         (64, 1024), (5, 2049), (3, 4096), (2, 4099), (3, 5120), (2, 8192), (3, 8200), (1, 16384), (2, 16387), (2, 32768),
         (2, 32776), (2, 40001), (300, 520), (1030, 96), (4097, 24), (512, 1000), (513, 1000), (513, 40001), (600, 15), (520, 8),
         (700, 9000), (530, 16388), (515, 32768), (3, (1 << 20) + 7), (2000, 7), (70000, 3), ((1 << 20) + 300, 2)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N", SIZES)
def test_forward_and_backward(M, N, dtype):
    from axonn_amd import ops

    for params, residual in (("same", False), ("fp32", True), ("none", False)):
        x, r, w, b, dy, ds = make(M, N, dtype, params, seed=M * 7 + N, residual=residual)
        y, h, mean, rstd = ops.layer_norm_fwd(x, w, b, EPS, residual=r)
        if residual:
            assert torch.equal(h, (x.float() + r.float()).to(dtype))
        else:
            assert h is None
            h = x
        check_forward(y, mean, rstd, h, w, b, dtype)
        again, _, none, _ = ops.layer_norm_fwd(x, w, b, EPS, residual=r, save=False)
        assert none is None and torch.equal(again, y)
        got = ops.layer_norm_bwd(dy, h, w, mean, rstd, ds)
        assert got[1].dtype == got[2].dtype == (dtype if w is None else w.dtype)
        check_backward(got, dy, h, w, mean, rstd, ds, dtype)
        for a, c in zip(got, ops.layer_norm_bwd(dy, h, w, mean, rstd, ds)):
            assert torch.equal(a, c)      # the sums have one order


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_other_strides_and_alignments(dtype):
    """Views of wider buffers, at odd places, with odd strides; what is around them is left alone."""
    from axonn_amd import ops

    for M, N in ((5, 64), (5, 100), (5, 1024), (5, 1027), (5, 4096), (5, 8200), (600, 64), (600, 1027), (515, 8200), (600, 3),
                 (5, 40001), (515, 33000)):
        for skip, ld in ((1, N + 3), (8, N + 16), (5, N + 8)):
            x, r, w, b, dy, ds = make(M, N, dtype, "same", seed=N, residual=True)
            wide = []
            for t in (x, r, dy, ds):
                big = torch.full((M, ld + skip), 777.0, device="cuda").to(dtype)
                big[:, skip:skip + N] = t
                wide.append(big[:, skip:skip + N])
            apart = torch.cat([torch.zeros(1, device="cuda", dtype=dtype), w])[1:]   # (a parameter at an odd place too)
            want = ops.layer_norm_fwd(x, w, b, EPS, residual=r)
            got = ops.layer_norm_fwd(wide[0], apart, b, EPS, residual=wide[1])
            check_forward(got[0], got[2], got[3], got[1], apart, b, dtype)
            assert torch.equal(got[1], want[1])
            grads = ops.layer_norm_bwd(wide[2], got[1], apart, got[2], got[3], wide[3])
            check_backward(grads, dy, got[1], w, got[2], got[3], ds, dtype)
    # one row repeated, columns apart, a transposed matrix: made dense first
    x = torch.randn(1, 96, device="cuda").to(dtype).expand(6, 96)
    check_forward(*[ops.layer_norm_fwd(x)[i] for i in (0, 2, 3)], x, None, None, dtype)
    x = torch.randn(96, 6, device="cuda").to(dtype).t()
    check_forward(*[ops.layer_norm_fwd(x)[i] for i in (0, 2, 3)], x, None, None, dtype)
    x = torch.randn(6, 192, device="cuda").to(dtype)[:, ::2]
    check_forward(*[ops.layer_norm_fwd(x)[i] for i in (0, 2, 3)], x, None, None, dtype)


@pytest.mark.parametrize("M,N", [(3, 3), (600, 2), (520, 33001), (3, 63), (3, 64), (3, 1024), (3, 4096), (3, 8200), (3, 40001), (517, 63), (517, 64), (517, 1030),
                                 (517, 8200), (517, 40001)])
def test_outputs_end_where_their_rows_do(M, N):
    """Through the C ABI into buffers with something behind them (and in front), M rows of them."""
    from axonn_amd import _native as nv

    for dtype in DTYPES:
        x, r, w, b, dy, ds = make(M, N, dtype, "fp32", seed=N, residual=True)
        guard, n = 64, M * N
        buf = {k: torch.full((n + 2 * guard,), 55.0, device="cuda").to(dtype) for k in ("y", "h", "dx")}
        par = {k: torch.full((N + 2 * guard,), 55.0, device="cuda") for k in ("dw", "db")}
        st = {k: torch.full((M + 2 * guard,), 55.0, device="cuda") for k in ("mean", "rstd")}
        at = lambda t: t.data_ptr() + guard * t.element_size()  # noqa: E731
        lib = nv.load()
        code = nv.dtype_code(dtype)
        nbytes = lib.axn_layer_norm_bwd_workspace_bytes(M, N)
        ws = torch.full((nbytes + 256,), 77, dtype=torch.uint8, device="cuda")
        nv.check(lib.axn_layer_norm_fwd(x.data_ptr(), r.data_ptr(), w.data_ptr(), b.data_ptr(), at(buf["y"]), at(buf["h"]),
                                        at(st["mean"]), at(st["rstd"]), code, nv.F32, M, N, N, N, EPS, nv.current_stream()))
        nv.check(lib.axn_layer_norm_bwd(dy.data_ptr(), at(buf["h"]), w.data_ptr(), at(st["mean"]), at(st["rstd"]),
                                        ds.data_ptr(), at(buf["dx"]), at(par["dw"]), at(par["db"]), code, nv.F32, M, N, N, N,
                                        N, ws.data_ptr(), nbytes, nv.current_stream()))
        torch.cuda.synchronize()
        for t in (*buf.values(), *par.values(), *st.values()):
            assert (t[:guard] == 55).all() and (t[-guard:] == 55).all()
        assert (ws[nbytes:] == 77).all()
        h = buf["h"][guard:guard + n].view(M, N)
        mean, rstd = (st[k][guard:guard + M] for k in ("mean", "rstd"))
        check_forward(buf["y"][guard:guard + n].view(M, N), mean, rstd, h, w, b, dtype)
        check_backward((buf["dx"][guard:guard + n].view(M, N), par["dw"][guard:guard + N], par["db"][guard:guard + N]), dy, h,
                       w, mean, rstd, ds, dtype)


@pytest.mark.parametrize("N", [5, 64, 1000, 4096, 40000])
def test_rows_far_from_zero_and_without_spread(N):
    """The variance is that of the deviations: rows around 1000 keep theirs, equal rows have none."""
    from axonn_amd import ops

    x, *_ = make(4, N, torch.float32, x_offset=1000.0)
    y, _, mean, rstd = ops.layer_norm_fwd(x)
    check_forward(y, mean, rstd, x, None, None, torch.float32)
    x = torch.full((3, N), 7.0, device="cuda")
    y, _, mean, rstd = ops.layer_norm_fwd(x, eps=1e-4)
    assert (mean == 7).all() and torch.allclose(rstd, torch.full((3,), 100.0, device="cuda"), rtol=1e-6) and not y.any()
    dx, dw, db = ops.layer_norm_bwd(torch.ones_like(x), x, None, mean, rstd)
    assert not dx.any() and not dw.any() and (db == 3).all()
    # without eps a row without spread is 0 / 0, as by the formula
    assert torch.isnan(ops.layer_norm_fwd(x, eps=0.0)[0]).all()


@pytest.mark.parametrize("N", [3, 40, 1024, 8192, 40000])
def test_values_that_are_not_finite_stay_in_their_row(N):
    from axonn_amd import ops

    for dtype in DTYPES:
        x, _, w, b, dy, _ = make(5, N, dtype)
        x[1, N - 1], x[3, 0] = float("nan"), float("inf")
        y, _, mean, rstd = ops.layer_norm_fwd(x, w, b)
        assert torch.isnan(y[1]).all() and torch.isnan(y[3]).all() and torch.isfinite(y[[0, 2, 4]]).all()
        check_forward(y[[0, 2, 4]], mean[[0, 2, 4]], rstd[[0, 2, 4]], x[[0, 2, 4]], w, b, dtype)
        dx, dw, db = ops.layer_norm_bwd(dy, x, w, mean, rstd)
        assert torch.isnan(dx[1]).all() and torch.isfinite(dx[[0, 2, 4]]).all()
        assert torch.isnan(dw).all() and torch.isfinite(db).all()


def test_largest_magnitudes_of_fp16():
    """Rows at the end of fp16's range: sums in fp32 hold them, results that fp16 cannot hold are infinite."""
    from axonn_amd import ops

    x = torch.full((2, 512), 65504.0, device="cuda").half()
    x[:, ::2] = -65504.0
    y, _, mean, rstd = ops.layer_norm_fwd(x)
    check_forward(y, mean, rstd, x, None, None, torch.float16)
    y, h, *_ = ops.layer_norm_fwd(x, residual=x)
    assert torch.isinf(h).all() and torch.isnan(y).all()


def test_no_rows():
    from axonn_amd import ops

    for dtype in DTYPES:
        x, w = torch.zeros(0, 24, device="cuda", dtype=dtype), torch.ones(24, device="cuda", dtype=dtype)
        y, h, mean, rstd = ops.layer_norm_fwd(x, w, w, residual=x)
        assert y.shape == h.shape == (0, 24) and mean.shape == rstd.shape == (0,)
        dx, dw, db = ops.layer_norm_bwd(y, h, w, mean, rstd, y)
        assert dx.shape == (0, 24) and not dw.any() and not db.any() and dw.shape == db.shape == (24,)
        assert ops.layer_norm_bwd(y, h, w, mean, rstd, want_dweight=False, want_dbias=False)[0].shape == (0, 24)


@pytest.mark.parametrize("want", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1), (1, 1, 0), (0, 0, 0)])
def test_gradients_one_by_one(want):
    from axonn_amd import ops

    for M, N in ((37, 72), (37, 1001), (37, 4096), (37, 40000), (600, 72), (600, 1001), (530, 4096), (515, 40000)):
        x, _, w, _, dy, _ = make(M, N, torch.bfloat16)
        _, _, mean, rstd = ops.layer_norm_fwd(x, w)
        every = ops.layer_norm_bwd(dy, x, w, mean, rstd)
        some = ops.layer_norm_bwd(dy, x, w, mean, rstd, None, *map(bool, want))
        for a, b, wanted in zip(some, every, want):
            assert (a is not None and torch.equal(a, b)) if wanted else a is None


def test_operands_that_do_not_fit_are_refused():
    from axonn_amd import ops

    x, r, w, b, dy, ds = make(4, 32, torch.bfloat16, residual=True)
    _, h, mean, rstd = ops.layer_norm_fwd(x, w, b, residual=r)
    for bad in (dict(weight=w[:31]), dict(bias=b.view(4, 8)), dict(residual=r[:3]), dict(residual=r.float())):
        with pytest.raises(ValueError):
            ops.layer_norm_fwd(x, **bad)
    for bad in (dict(weight=w.half()), dict(weight=w.float(), bias=b), dict(bias=b.double())):
        with pytest.raises(TypeError):
            ops.layer_norm_fwd(x, **bad)
    with pytest.raises(TypeError):
        ops.layer_norm_fwd(x.double())
    with pytest.raises(ValueError):
        ops.layer_norm_fwd(x.view(2, 2, 32))
    with pytest.raises(ValueError):
        ops.layer_norm_fwd(x[:, :0])
    with pytest.raises(RuntimeError, match="eps"):
        ops.layer_norm_fwd(x, eps=-1.0)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.layer_norm_fwd(x, w.cpu())
    for args in ((dy, h[:3], w, mean, rstd), (dy, h.float(), w, mean, rstd), (dy, h, w, mean[:3], rstd),
                 (dy, h, w, mean, rstd.double()), (dy, h, w, mean, rstd, ds[:, :31]), (dy, h, w[:8], mean, rstd)):
        with pytest.raises(ValueError):
            ops.layer_norm_bwd(*args)
    with pytest.raises(TypeError):
        ops.layer_norm_bwd(dy, h, None, mean, rstd, param_dtype=torch.float16)


# ---------------------------------------------------------------- the layer --
@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_against_autograd_in_64_bits(dtype):
    """LayerNorm in a graph where the sum goes on by itself, as in a pre-norm block, on a padded batch."""
    from axonn_amd.intra_layer import LayerNorm

    torch.manual_seed(1)
    for shape, norm in (((2, 9, 96), 96), ((3, 4, 5, 8), (5, 8)), ((7, 1040), 1040)):
        layer = LayerNorm(norm, eps=1e-3).cuda().to(dtype)
        with torch.no_grad():
            layer.weight.add_(torch.randn_like(layer.weight) * 0.1)
            layer.bias.add_(torch.randn_like(layer.bias) * 0.1)
        x, r = (torch.randn(shape, device="cuda").to(dtype).requires_grad_() for _ in range(2))
        dy, ds = (torch.randn(shape, device="cuda").to(dtype) for _ in range(2))
        y, h = layer(x, r)
        torch.autograd.backward((y, h), (dy, ds))
        n = layer.weight.numel()
        rows = lambda t: t.detach().reshape(-1, n)  # noqa: E731
        _, m64, s64 = ol.forward(f64(rows(h)), eps=1e-3)
        mean, rstd = torch.tensor(m64).float(), torch.tensor(s64).float()
        check_forward(rows(y), None, None, rows(h), layer.weight.reshape(-1), layer.bias.reshape(-1), dtype, 1e-3)
        assert torch.equal(x.grad, r.grad)
        # (statistics rounded to fp32 here, and the kernel's own: a few steps of fp32 more than `check_backward` counts)
        got = (rows(x.grad), layer.weight.grad.reshape(-1), layer.bias.grad.reshape(-1))
        check_backward(got, rows(dy), rows(h), layer.weight.reshape(-1), mean, rstd, rows(ds), dtype)
        # the sum alone, the norm alone, and a gradient that autograd hands over expanded
        for t in (x, r, layer.weight, layer.bias):
            t.grad = None
        layer(x, r)[1].backward(ds)
        assert torch.equal(x.grad, ds) and layer.weight.grad is None
        x.grad = None
        layer(x, r)[0].sum().backward()
        check_backward((rows(x.grad), None, None), torch.ones_like(rows(x)), rows(h), layer.weight.reshape(-1), mean, rstd,
                       None, dtype)


def test_layer_without_parameters_or_gradients():
    from axonn_amd.intra_layer import LayerNorm, layer_norm

    x = torch.randn(6, 64, device="cuda")
    want = torch.nn.functional.layer_norm(x.double(), (64,)).float()
    plain, no_bias = LayerNorm(64, elementwise_affine=False).cuda(), LayerNorm(64, bias=False).cuda()
    for layer in (plain, no_bias):
        assert torch.allclose(layer(x), want, atol=1e-5)
        with torch.no_grad():
            assert torch.equal(layer(x), layer(x))
    no_bias(x).sum().backward()
    assert no_bias.weight.grad is not None
    xg = x.clone().requires_grad_()
    bias = torch.zeros(64, device="cuda", requires_grad=True)
    layer_norm(xg, 64, None, bias).backward(torch.ones_like(x))
    assert (bias.grad == 6).all() and xg.grad.abs().max() < 1e-5
    frozen = LayerNorm(64).cuda().requires_grad_(False)
    frozen(xg).sum().backward()
    assert frozen.weight.grad is None
    # second derivatives are refused, not wrong
    y = LayerNorm(64).cuda()(xg)
    (gx,) = torch.autograd.grad(y.square().sum(), xg, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable|differentiate twice"):
        gx.sum().backward()


def test_layer_under_autocast_is_fp32_as_torchs():
    from axonn_amd.intra_layer import LayerNorm

    torch.manual_seed(2)
    layer, ref = LayerNorm(128).cuda(), torch.nn.LayerNorm(128).cuda()
    x = torch.randn(5, 128, device="cuda").half()
    outs = []
    for module in (layer, ref):
        leaf = x.clone().requires_grad_()
        with torch.autocast("cuda", dtype=torch.float16):
            y = module(leaf)
        y.square().sum().backward()
        outs.append((y, leaf.grad, module.weight.grad, module.bias.grad))
    for a, b in zip(*outs):
        assert a.dtype == b.dtype and torch.allclose(a.float(), b.float(), rtol=1e-3, atol=1e-4)


def test_gradients_against_differences():
    """Directional derivatives of the 64-bit formula by central differences against the kernel's fp32 gradients:
    differences with step 1e-5 are off by some 1e-9 of the loss's scale, the kernel by the bound of `check_backward`."""
    from axonn_amd import ops

    for M, N in ((3, 17), (4, 320), (2, 1100)):
        x, _, w, b, dy, _ = make(M, N, torch.float32, seed=N)
        _, _, mean, rstd = ops.layer_norm_fwd(x, w, b)
        got = ops.layer_norm_bwd(dy, x, w, mean, rstd)
        base = [f64(t) for t in (x, w, b)]
        rng = np.random.default_rng(N)
        for i, grad in enumerate(got):
            u = rng.normal(0, 1, base[i].shape)
            loss = []
            for s in (1e-5, -1e-5):
                moved = list(base)
                moved[i] = base[i] + s * u
                loss.append((ol.forward(moved[0], moved[1], moved[2])[0] * f64(dy)).sum())
            want = (loss[0] - loss[1]) / 2e-5
            terms = np.abs(f64(grad) * u).sum() + np.sqrt(M * N) * 8
            assert abs((f64(grad) * u).sum() - want) < (chain(N) + 64) * U * terms + 1e-7 * terms


@pytest.mark.parametrize("rows", [200, 2000])
def test_replayed_norm_equals_the_eager_one(rows):
    """Forward and backward captured once, replayed with other inputs between eager calls of the same sizes."""
    from axonn_amd import ops

    x, r, w, b, dy, ds = make(rows, 1000, torch.bfloat16, "fp32", residual=True)

    def both():
        y, h, mean, rstd = ops.layer_norm_fwd(x, w, b, residual=r)
        return (y, h) + ops.layer_norm_bwd(dy, h, w, mean, rstd, ds)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):   # two graphs, each with workspaces of its own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = both()
        graphs.append((graph, out))
    for i in range(3):
        for t, s in zip((x, r, dy, ds), range(4)):
            t.normal_(generator=torch.Generator(device="cuda").manual_seed(10 * i + s))
        want = both()
        for graph, out in graphs:
            graph.replay()
            torch.cuda.synchronize()
            for a, c in zip(out, want):
                assert torch.equal(a, c)


def test_other_stream():
    from axonn_amd import ops

    x, r, w, b, dy, ds = make(64, 2048, torch.float16, residual=True)
    want = ops.layer_norm_fwd(x, w, b, residual=r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.layer_norm_fwd(x, w, b, residual=r)
        grads = ops.layer_norm_bwd(dy, got[1], w, got[2], got[3], ds)
    side.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    check_backward(grads, dy, got[1], w, got[2], got[3], ds, torch.float16)


@pytest.mark.parametrize("N", [64, 1024, 1027, 4160, 20000])
def test_sums_larger_than_the_cache(N):
    """With a residual, from 256 MB on: rows from all over the matrix, the last ones among them."""
    from axonn_amd import ops

    M = (300 << 20) // (8 * N) + 5
    for params in ("same", "fp32"):
        x, r, w, b, _, _ = make(M, N, torch.float16, params, seed=N, residual=True)
        y, h, mean, rstd = ops.layer_norm_fwd(x, w, b, residual=r)
        assert torch.equal(h, x + r)
        rows = torch.cat([torch.arange(0, M, max(1, M // 50)), torch.arange(M - 5, M)]).cuda()
        check_forward(y[rows], mean[rows], rstd[rows], h[rows], w, b, torch.float16)
        z, _, _, _ = ops.layer_norm_fwd(h, w, b)      # without: the other kernel, of the same sums
        assert torch.equal(z, y)


def test_rows_beyond_32_bits():
    """The last rows of a matrix of more than 2^31 elements, and of one whose stride takes them there."""
    from axonn_amd import ops

    N, M = 8192, (1 << 18) + 3
    x = torch.zeros(M, N, device="cuda", dtype=torch.bfloat16)
    x[-3:] = torch.randn(3, N, device="cuda").bfloat16()
    y, _, mean, rstd = ops.layer_norm_fwd(x)
    check_forward(y[-3:], mean[-3:], rstd[-3:], x[-3:], None, None, torch.bfloat16)
    dx, dw, db = ops.layer_norm_bwd(x, x, None, mean, rstd)
    check_backward((dx[-3:], None, None), x[-3:], x[-3:], None, mean[-3:], rstd[-3:], None, torch.bfloat16)
    assert torch.equal(db, x[-3:].float().sum(0).bfloat16()) or (db.float() - x[-3:].double().sum(0).float()).abs().max() < 0.05
    del x, y, dx
    flat = torch.randn(3 * (1 << 30), device="cuda", dtype=torch.bfloat16)[:2 * 1500000000 + 64]
    far = flat.as_strided((3, 64), (1500000000, 1))
    y, _, mean, rstd = ops.layer_norm_fwd(far)
    check_forward(y, mean, rstd, far, None, None, torch.bfloat16)
