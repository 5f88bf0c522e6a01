"""The layer norm's backward pass where a workgroup holds several rows and goes on to others: rows in turn in two sets of
registers, their sums over turns joined in LDS, and a last turn that is not full.  Against the formulas in 64 bits, with
the tolerances of test_layer_norm_gpu.py."""

import pytest
import torch
from launches import launches
from test_layer_norm_gpu import EPS, check_backward, check_forward, make

pytestmark = pytest.mark.gpu


def plan(M, N, size):
    """(vectors of a lane, waves of a row or 0 for 16 lanes, rows at a time, workgroups, turns of a workgroup)."""
    vectors = -(-N // (16 // size))
    if vectors <= 32:
        k, waves, fit = 1 + (vectors > 16), 0, 64
    else:
        k = 1 if vectors <= 1024 else 2 if vectors <= 2048 else 4
        waves = -(-vectors // (64 * k))
        fit = 16 // waves
    rows = min(-(-M // 256), fit)
    if waves == 0:
        rows = -(-rows // 4) * 4
    parts = min(-(-M // rows), 256)
    return k, waves, rows, parts, -(-M // (rows * parts))


# rows, and elements of a row in vectors of 16 bytes (the last one cut short by 0, 1 or 2 elements), with what they reach
CASES = [(20011, 8, 0, (1, 0, 64)), (16401, 16, 1, (1, 0, 64)), (17003, 25, 0, (2, 0, 64)), (17003, 32, 2, (2, 0, 64)),
         (5003, 63, 1, (1, 1, 16)), (5003, 33, 0, (1, 1, 16)), (4099, 125, 0, (1, 2, 8)), (2999, 300, 1, (1, 5, 3)),
         (2999, 512, 0, (1, 8, 2)), (1500, 513, 1, (1, 9, 1)), (777, 1030, 2, (2, 9, 1))]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M,vectors,short,reached", CASES)
def test_rows_in_turns(M, vectors, short, reached, dtype):
    from axonn_amd import ops

    N = vectors * 16 // dtype.itemsize - short
    k, waves, rows, parts, turns = plan(M, N, dtype.itemsize)
    assert (k, waves, rows) == reached and turns > 1 and M % (rows * parts) != 0
    for params, residual in (("same", False), ("fp32", True), ("none", True), ("fp32", False)):
        x, r, w, b, dy, ds = make(M, N, dtype, params, seed=M + N, residual=residual)
        y, h, mean, rstd = ops.layer_norm_fwd(x, w, b, EPS, residual=r)
        h = x if h is None else h
        check_forward(y, mean, rstd, h, w, b, dtype)
        got = ops.layer_norm_bwd(dy, h, w, mean, rstd, ds)
        check_backward(got, dy, h, w, mean, rstd, ds, dtype)
    # the launch that this was
    name, groups, threads = next(found for found in launches(lambda: ops.layer_norm_bwd(dy, h, w, mean, rstd, ds), threads=True)
                                 if "norm_grad_rows_kernel" in found[0])
    assert (groups, threads) == (parts, rows * (16 if waves == 0 else waves * 64)), name


@pytest.mark.parametrize("M,N", [((1 << 18) + 3, 8192), ((1 << 25) + 5, 64), ((1 << 16) + 3, 33000)])
def test_gradients_of_rows_beyond_32_bits(M, N):
    """The last rows of more than 2^31 elements: all three gradients.  The rows before them are zero and so is their
    gradient, so that the sums over rows are those of the last ones."""
    from axonn_amd import ops

    last = 3
    x, _, w, b, dy, _ = make(last, N, torch.bfloat16, "fp32", seed=N)
    rows, grads = (torch.zeros(M, N, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    rows[-last:], grads[-last:] = x, dy
    y, _, mean, rstd = ops.layer_norm_fwd(rows, w, b)
    check_forward(y[-last:], mean[-last:], rstd[-last:], x, w, b, torch.bfloat16)
    dx, dw, db = ops.layer_norm_bwd(grads, rows, w, mean, rstd)
    check_backward((dx[-last:], dw, db), dy, x, w, mean[-last:], rstd[-last:], None, torch.bfloat16)
    assert not dx[:-last].any()
