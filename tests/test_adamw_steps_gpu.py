"""The AdamW optimizer step by step against the oracle: every step of two groups from the state in front of it, scaled,
clipped, with moments in 32 and in 8 bits."""

import numpy as np
import pytest
import torch

from oracle import adamw as oa

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
SHAPES = ((3,), (17, 31), (256,), (40, 64), (1,))


def n64(t):
    return t.detach().double().cpu().numpy()


def check_step(before, after, g, t, lr, beta1, beta2, eps, decay, what):
    """Moments and weights (p, m, v) of a step whose gradients are g, rounded once to fp32 by the clip's product.

    m + (g - m) c: g's rounding, the difference's, the product's and c's, at most of |m| + |g| each, and the sum's: 5.
    v b + (1 - b) g g: of the second term the constant, two products and twice g's rounding, of the first the constant and
    the product, and the sum: 6.
    p keep - rate (m / denom): m's error divided by denom; of the rest of the update half of v's 6, the constants, the root
    and quotient (two steps each where they are instructions of 1 ulp) and the products: 16; p's own constant, product and
    difference: 3."""
    p0, m0, v0 = before
    p, m, v = oa.step(g, p0, m0, v0, t, lr, beta1, beta2, eps, decay)
    off_m = 5 * U * (np.abs(m0) + np.abs(g))
    if after[1] is not None:
        assert (np.abs(n64(after[1]) - m) <= off_m + 1e-45).all(), what
        assert (np.abs(n64(after[2]) - v) <= 6 * U * v + 1e-45).all(), what
    slope = lr / (1 - beta1 ** t) / (np.sqrt(v / (1 - beta2 ** t)) + eps)
    bound = slope * off_m + 16 * U * slope * np.abs(m) + 3 * U * (np.abs(p0) + np.abs(p)) + 1e-45
    assert (np.abs(n64(after[0]) - p) <= bound).all(), what


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bits", [32, 8])
def test_every_step_of_the_optimizer(bits, dtype):
    from axonn_amd.optim import AdamW

    gen = torch.Generator(device="cuda").manual_seed(5)
    params = [torch.nn.Parameter((torch.randn(*s, generator=gen, device="cuda") * 0.1).to(dtype)) for s in SHAPES]
    opt = AdamW([dict(params=params[:2], lr=1e-2, betas=(0.8, 0.99)), dict(params=params[2:], weight_decay=0.3, eps=1e-6)],
                lr=3e-3, weight_decay=0.05, max_grad_norm=2.0, state_bits=bits, seed=11)
    for t in range(1, 6):
        scale = opt.loss_scale
        for p in params:
            p.grad.copy_(torch.randn(p.shape, generator=gen, device="cuda") * (0.02 * t * min(scale, 256.0)))
        flat = [opt.model_grads_fp16, opt.model_params_fp32] + ([opt.exp_avg, opt.exp_avg_sq] if bits == 32 else [])
        before = [n64(f) for f in flat]
        state = [x.cpu().numpy().copy() for x in (opt.codes, opt.exponents)] if bits == 8 else None
        opt.step()
        assert opt.step_count == t and not opt.last_step_skipped
        clip = float(opt._scan.clip_coef)
        g = before[0] / scale * clip
        for no, group in enumerate(opt.param_groups):
            lo, hi = opt.group_offsets[no], opt.group_offsets[no + 1]
            part = slice(lo, hi)
            hp = (group["lr"], *group["betas"], group["eps"], group["weight_decay"])
            if bits == 32:
                check_step([x[part] for x in before[1:]], (opt.model_params_fp32[part], opt.exp_avg[part], opt.exp_avg_sq[part]),
                           g[part], t, *hp, (t, no))
                continue
            blocks = slice(lo // 256, hi // 256)
            old = [x[blocks] for x in state]
            _, codes, exponents = oa.step8(before[0][part], before[1][part], *old, opt._step_seed(t, no), t, *hp,
                                           inv_scale=1.0 / scale, clip=clip)
            assert np.array_equal(opt.codes[blocks].cpu().numpy(), codes), (t, no)
            assert np.array_equal(opt.exponents[blocks].cpu().numpy(), exponents), (t, no)
            m, v = (x.reshape(-1) for x in oa.decode(*old))
            check_step((before[1][part], m, v), (opt.model_params_fp32[part], None, None), g[part], t, *hp, (t, no))
        # what the parameters, the copies and the read-back moments are
        for p, (m, v), (offset, n) in zip(params, opt.moments(), opt._views):
            assert torch.equal(p.detach().view(-1), opt.model_params_fp32[offset:offset + n].to(dtype))
            if bits == 8:
                wm, wv = (x.reshape(-1)[offset:offset + n].astype(np.float32) for x in
                          oa.decode(opt.codes.cpu().numpy(), opt.exponents.cpu().numpy()))
                assert np.array_equal(m.view(-1).cpu().numpy(), wm) and np.array_equal(v.view(-1).cpu().numpy(), wv)
