"""What a step writes, and only that: tensors that share their memory until the first write."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("as_list", [list, tuple])
def test_lazy_clones_of_what_a_step_writes_stay(bits, as_list):
    """`torch._lazy_clone` gives a tensor that has its twin's memory until one of them is written; the step is such a
    write, through its one native call and (for lists that are none) the general way."""
    from axonn_amd import ops

    n, gen = 700, torch.Generator(device="cuda").manual_seed(bits)
    draw = lambda: torch.randn(n, generator=gen, device="cuda")  # noqa: E731
    g, p, m = draw().bfloat16(), draw(), draw()
    v, low = draw().square(), torch.zeros_like(p, dtype=torch.bfloat16)
    if bits == 8:
        m, v = ops.adamw8_state(p.numel())
    hp = ops.adamw_hparams(1, 1e-2, 0.9, 0.999, 1e-8, 0.1)

    def step(*tensors):
        lists = [as_list([t]) for t in tensors]
        if bits == 32:
            ops.mt_adamw(*lists, hp)
        else:
            ops.mt_adamw8(*lists, hp, 5)
        return tensors[1:]

    start = [t.clone() for t in (g, p, m, v, low)]
    want = step(*(t.clone() for t in start))
    for which in range(5):
        twins = [t.clone() for t in start]
        lazy = [torch._lazy_clone(t) if i == which else t for i, t in enumerate(twins)]
        for a, b in zip(step(*lazy), want):
            assert torch.equal(a, b), which
        assert torch.equal(twins[which], start[which]), which
