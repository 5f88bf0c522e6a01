"""AdamW's state dict: a run that is saved, and goes on in another process's model and optimizer, is the run that was
never interrupted, bit by bit."""

import pytest
import torch

pytestmark = pytest.mark.gpu

SHAPES = ((3,), (17, 31), (256,), (40, 64), (1,))


def fresh(dtype, bits, seed, seed8=7):
    from axonn_amd.optim import AdamW

    gen = torch.Generator(device="cuda").manual_seed(seed)
    params = [torch.nn.Parameter((torch.randn(*s, generator=gen, device="cuda") * 0.1).to(dtype)) for s in SHAPES]
    opt = AdamW([dict(params=params[:2], lr=1e-2), dict(params=params[2:], weight_decay=0.3)], lr=3e-3, max_grad_norm=1.0,
                state_bits=bits, seed=seed8)
    return params, opt


def train(params, opt, steps):
    for t in steps:
        gen = torch.Generator(device="cuda").manual_seed(t)
        for p in params:
            p.grad.copy_(torch.randn(p.shape, generator=gen, device="cuda") * 0.01 * min(opt.loss_scale, 1024.0))
        if t == 4 and opt.dynamic_loss_scale:
            params[1].grad[0, 0] = float("inf")      # a skipped step, which halves the scale
        opt.param_groups[0]["lr"] *= 0.9
        opt.step()


def everything(params, opt):
    flat = [opt.codes, opt.exponents] if opt.state_bits == 8 else [opt.exp_avg, opt.exp_avg_sq]
    return [p.detach() for p in params] + [opt.model_params_fp32] + flat


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("bits", [32, 8])
def test_a_run_goes_on_where_it_was_saved(bits, dtype, tmp_path):
    from axonn_amd import checkpoint

    params, opt = fresh(dtype, bits, 0)
    train(params, opt, range(1, 6))
    checkpoint.save({"opt": opt.state_dict()}, str(tmp_path), "state")
    at = opt.step_count, opt.loss_scale, opt.scaler.no_overflow_iters, opt.param_groups[0]["lr"]
    train(params, opt, range(6, 9))

    twin, other = fresh(dtype, bits, 1, seed8=8)       # other weights, another seed
    train(twin, other, range(1, 3))
    other.load_state_dict(checkpoint.load(None, str(tmp_path), "state", map_location="cpu")["opt"])
    assert at == (other.step_count, other.loss_scale, other.scaler.no_overflow_iters, other.param_groups[0]["lr"])
    assert at[0] == (4 if dtype == torch.float16 else 5)
    train(twin, other, range(6, 9))
    for a, b in zip(everything(params, opt), everything(twin, other)):
        assert torch.equal(a, b)
    assert (opt.step_count, opt.loss_scale) == (other.step_count, other.loss_scale)


@pytest.mark.parametrize("bits", [32, 8])
def test_weights_come_back_with_the_state(bits):
    """Before the next step too, and into the memory that the parameters have."""
    params, opt = fresh(torch.bfloat16, bits, 0)
    train(params, opt, (1, 2))
    twin, other = fresh(torch.bfloat16, bits, 1)
    places = [p.data_ptr() for p in twin]
    other.load_state_dict(opt.state_dict())
    assert [p.data_ptr() for p in twin] == places
    for a, b in zip(everything(params, opt), everything(twin, other)):
        assert torch.equal(a, b)
    train(params, opt, (3,))
    for a, b in zip(params, twin):
        assert not torch.equal(a, b)               # (a copy, not the other's memory)


@pytest.mark.parametrize("bits", [32, 8])
def test_states_that_do_not_fit_are_refused(bits):
    """And leave the optimizer as it was."""
    from axonn_amd.optim import AdamW

    params, opt = fresh(torch.bfloat16, bits, 0)
    train(params, opt, (1,))
    before = [t.clone() for t in everything(params, opt)]
    moments = {k: v for k, v in opt.state_dict().items() if k in ("state", "param_groups")}     # as torch's class keeps it: no moments
    shapes = [(3,), (17, 31), (256,), (64, 40), (2,)]
    other = AdamW([dict(params=[torch.nn.Parameter(torch.zeros(s, device="cuda", dtype=torch.bfloat16)) for s in ss])
                   for ss in (shapes[:2], shapes[2:])], state_bits=bits).state_dict()
    for bad in (moments, fresh(torch.bfloat16, 40 - bits, 0)[1].state_dict(), other):
        with pytest.raises(ValueError, match="AdamW"):
            opt.load_state_dict(bad)
    assert opt.step_count == 1 and opt.param_groups[0]["lr"] == 1e-2 * 0.9
    assert all(torch.equal(a, b) for a, b in zip(before, everything(params, opt)))


def test_a_saved_group_without_eps_is_refused_by_8_bit_moments():
    params, opt = fresh(torch.bfloat16, 8, 0)
    state = opt.state_dict()
    state["param_groups"][1]["eps"] = 0.0
    with pytest.raises(ValueError, match="positive"):
        opt.load_state_dict(state)
    assert opt.param_groups[1]["eps"] == 1e-8
