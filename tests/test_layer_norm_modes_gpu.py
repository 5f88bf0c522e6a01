"""The layer in autograd's modes: tangents and traces, with and without gradients, and AdamW and the norm from several
host threads."""

import threading

import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("gradients", [True, False])
def test_tangents_are_refused(gradients):
    from axonn_amd.intra_layer import LayerNorm

    layer, x = LayerNorm(64).cuda(), torch.randn(5, 64, device="cuda")
    with torch.set_grad_enabled(gradients), forward_ad.dual_level():
        assert torch.equal(layer(x), layer(x, torch.zeros_like(x))[0])
        with pytest.raises(NotImplementedError, match="jvp"):
            layer(forward_ad.make_dual(x, torch.ones_like(x)))


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("gradients", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_traces_compute(gradients, dtype):
    from axonn_amd.intra_layer import LayerNorm

    layer = LayerNorm(1040).cuda().to(dtype)
    draw = lambda: (torch.randn(7, 1040, device="cuda").to(dtype), torch.randn(7, 1040, device="cuda").to(dtype))  # noqa: E731
    with torch.set_grad_enabled(gradients):
        traced = torch.jit.trace(layer, draw(), check_trace=False)
    for _ in range(3):
        args = draw()
        for again in (False, True):
            with torch.set_grad_enabled(again):
                assert all(torch.equal(a, b) for a, b in zip(traced(*args), layer(*args)))


def _inputs(seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    draw = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    return {"x": draw(300, 520).bfloat16(), "r": draw(300, 520).bfloat16(), "dy": draw(300, 520).bfloat16(), "w": draw(520),
            "many": draw(1030, 96), "g": draw(5001).bfloat16(), "p": draw(5001)}


def _work(s, rounds):
    from axonn_amd import ops

    w = s["w"].clone()
    dw = torch.zeros_like(w)
    state = [s["p"].clone(), torch.zeros_like(s["p"]), torch.zeros_like(s["p"])]
    p8, eight = s["p"].clone(), ops.adamw8_state(5001)
    low = torch.zeros_like(s["g"])
    for t in range(1, rounds + 1):
        y, h, mean, rstd = ops.layer_norm_fwd(s["x"], w, None, residual=s["r"])
        dx, grad, _ = ops.layer_norm_bwd(s["dy"], h, w, mean, rstd, s["r"])
        dw += grad
        _, _, mean, rstd = ops.layer_norm_fwd(s["many"])
        wide = ops.layer_norm_bwd(s["many"], s["many"], None, mean, rstd)      # (two launches and a workspace)
        hp = ops.adamw_hparams(t, 1e-3, 0.9, 0.999, 1e-8, 0.1)
        scan = ops.mt_scan([s["g"]], 1.0, 1.0)
        ops.mt_adamw([s["g"]], [state[0]], [state[1]], [state[2]], [low], hp, scan=scan)
        ops.mt_adamw8([s["g"]], [p8], [eight[0]], [eight[1]], None, hp, t, scan=scan)
        moments = ops.adamw8_moments(*eight, 5001)
    torch.cuda.current_stream().synchronize()
    return [t.clone() for t in (y, h, dx, dw, *wide, *state, low, p8, *eight, *moments)]


def test_concurrent_callers_match_a_lone_caller():
    n, rounds = 4, 12
    inputs = [_inputs(100 + i) for i in range(n)]
    want = [_work(s, rounds) for s in inputs]
    torch.cuda.synchronize()
    got, errors, start = [None] * n, [], threading.Barrier(n)

    def run(i):
        try:
            stream = torch.cuda.Stream()
            stream.wait_stream(torch.cuda.default_stream())
            with torch.cuda.stream(stream):
                start.wait()
                got[i] = _work(inputs[i], rounds)
        except Exception as e:  # noqa: BLE001 - reported by the asserting thread
            errors.append((i, repr(e)))

    threads = [threading.Thread(target=run, args=(i,)) for i in range(n)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    for i in range(n):
        assert all(torch.equal(a, b) for a, b in zip(got[i], want[i])), i
