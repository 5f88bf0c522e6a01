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


def test_lists_that_share_memory_are_refused():
    """And nothing of them is written."""
    from axonn_amd import ops

    hp = ops.adamw_hparams(1, 1e-2, 0.9, 0.999, 1e-8, 0.1)
    flat = torch.randn(4096, device="cuda")
    g, p, m, v = flat[:1000], flat[1000:2000], flat[2000:3000], flat[3000:4000]
    spare = torch.zeros(4096, device="cuda", dtype=torch.uint8)
    codes, exponents = spare[:2048], torch.zeros(8, device="cuda", dtype=torch.uint8)
    before = flat.clone()
    for lists in (([g], [p], [m], [m]), ([g], [p], [p], [v]), ([g], [p], [m], [flat[2999:3999]]),
                  ([flat[1:1001]], [g], [m], [v]), ([m], [p], [m], [v])):
        with pytest.raises(RuntimeError, match="overlap"):
            ops.mt_adamw(*lists, None, hp)
    for lists in (([p], [p], [codes], [codes[:8]]), ([g], [spare[96:].view(torch.float32)], [codes], [exponents])):
        with pytest.raises(RuntimeError, match="overlap"):
            ops.mt_adamw8(*lists, None, hp, 0)
    assert torch.equal(flat, before) and not spare.any()
    # the copy in the gradients' place, as apart from them
    low, apart = g.bfloat16(), torch.empty(1000, device="cuda", dtype=torch.bfloat16)
    args = [(low.clone(), p.clone(), m.clone(), v.abs()) for _ in range(2)]
    ops.mt_adamw(*([t] for t in args[0]), [apart], hp)
    ops.mt_adamw(*([t] for t in args[1]), [args[1][0]], hp)
    assert torch.equal(args[1][0], apart) and all(torch.equal(a, b) for a, b in zip(args[0][1:], args[1][1:]))
