"""AdamW on the GPU: the step with fp32 moments against the formulas in 64 bits, the one with
8-bit moments bit by bit against oracle/adamw.py, and the optimizer over both."""

import numpy as np
import pytest
import torch

from oracle import adamw as oa

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HP = dict(lr=1e-2, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.1)
SIZES = [1, 3, 255, 0, 256, 257, 1000, 4096, 5001, 2, 64]


def n64(t):
    return t.detach().double().cpu().numpy()


def views(flat, sizes, gap=0):
    out, off = [], 0
    for n in sizes:
        out.append(flat[off:off + n])
        off += n + gap
    return out


def lists(sizes, dtype, seed=0, gap=0, skip=0, low=None):
    """(g, p, m, v, low) as views of flat buffers, `gap` elements apart from element `skip` on; the buffers too."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    total = sum(sizes) + gap * len(sizes)
    flat = [torch.randn(total + skip, generator=gen, device="cuda") for _ in range(4)]
    flat[0] = (flat[0] * 4).to(dtype)
    flat[2] *= 0.1
    flat[3].square_()
    if low is not None:
        flat.append(torch.full((total + skip,), 9.0, device="cuda").to(low))
    return [views(f[skip:], sizes, gap) for f in flat], flat


def hparams(t, **kw):
    from axonn_amd import ops

    return ops.adamw_hparams(t, **{**HP, **kw})


def check_p(got, want, before, update, what=""):
    """p keep - rate m / denom in fp32: the constants, each of some ten operations and the quotient round once, each by
    2^-24 of its own term."""
    bound = 4 * U * np.abs(before) + 24 * U * np.abs(update) + U * np.abs(want) + 1e-45
    assert (np.abs(n64(got) - want) <= bound).all(), what


def update_of(p0, p1):
    return p1 - p0 * (1 - HP["lr"] * HP["weight_decay"])


@pytest.mark.parametrize("gdt,low", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
                                     (torch.float32, None), (torch.float32, torch.bfloat16), (torch.bfloat16, None)])
@pytest.mark.parametrize("gap,skip", [(0, 0), (0, 1), (7, 3)])
def test_step_in_fp32(gdt, low, gap, skip):
    from axonn_amd import ops

    (g, p, m, v, *lo), flat = lists(SIZES, gdt, gap=gap, skip=skip, low=low)
    before = [f.clone() for f in flat]
    old = [[n64(t) for t in ts] for ts in (g, p, m, v)]
    ops.mt_adamw(g, p, m, v, lo[0] if lo else None, hparams(3), inv_scale=0.25)
    for i in range(len(SIZES)):
        wp, wm, wv = oa.step(old[0][i], old[1][i], old[2][i], old[3][i], 3, *HP.values(), inv_scale=0.25)
        # m: the difference, its product and the sum; v: two products and their factors' roundings
        assert (np.abs(n64(m[i]) - wm) <= 4 * U * (np.abs(old[2][i]) + np.abs(old[0][i]))).all()
        assert (np.abs(n64(v[i]) - wv) <= 6 * U * wv + 1e-45).all()
        check_p(p[i], wp, old[1][i], update_of(old[1][i], wp))
        if lo:
            assert torch.equal(lo[0][i], p[i].to(low))
    inside = torch.zeros(flat[0].numel(), dtype=torch.bool, device="cuda")
    for view in views(inside[skip:], SIZES, gap):
        view.fill_(True)
    for f, b in zip(flat, before):
        assert torch.equal(f[~inside], b[~inside])
    assert torch.equal(flat[0], before[0])


def eight(sizes, seed=0):
    """Random valid codes for tensors of these sizes, zero behind their ends."""
    rng = np.random.default_rng(seed)
    out = []
    for n in sizes:
        blocks = -(-n // 256)
        m = rng.normal(0, 0.1, (blocks, 256)).astype(np.float32)
        v = (rng.normal(0, 1, (blocks, 256)) ** 2).astype(np.float32)
        behind = np.arange(blocks * 256).reshape(blocks, 256) >= n
        m[behind] = v[behind] = 0
        out.append(oa.quantize(m, v, oa.random_words(blocks, seed)) if blocks else
                   (np.zeros((0, 512), np.uint8), np.zeros((0, 2), np.uint8)))
    return [[torch.tensor(c, device="cuda") for c in cs] for cs in zip(*out)]


@pytest.mark.parametrize("gdt,low", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
                                     (torch.float32, None), (torch.float32, torch.bfloat16), (torch.bfloat16, None)])
@pytest.mark.parametrize("gap,skip", [(0, 0), (0, 1), (8, 4), (7, 3)])
def test_step_in_8_bits(gdt, low, gap, skip):
    """Codes and exponents equal to the oracle's bit by bit over three steps, weights within fp32's rounding."""
    from axonn_amd import ops

    (g, p, _, _, *lo), flat = lists(SIZES, gdt, gap=gap, skip=skip, low=low)
    codes, exps = eight(SIZES)
    for t in (5, 6, 7):
        old = [[n64(x) for x in xs] for xs in (g, p)]
        state = [[x.cpu().numpy().copy() for x in xs] for xs in (codes, exps)]
        seed = 0x123456789ABCDEF + (t << 33)
        ops.mt_adamw8(g, p, codes, exps, lo[0] if lo else None, hparams(t), seed, inv_scale=0.25)
        first = 0
        for i, n in enumerate(SIZES):
            wp, wc, we = oa.step8(old[0][i], old[1][i], state[0][i], state[1][i], seed, t, *HP.values(), inv_scale=0.25,
                                  first=first)
            first += len(we)
            assert np.array_equal(exps[i].cpu().numpy(), we), (t, i)
            assert np.array_equal(codes[i].cpu().numpy(), wc), (t, i)
            check_p(p[i], wp, old[1][i], update_of(old[1][i], wp), (t, i))
            if lo:
                assert torch.equal(lo[0][i], p[i].to(low))


@pytest.mark.parametrize("eightbit", [False, True])
def test_many_tensors_take_several_launches(eightbit):
    """150 tensors of sizes around a block: as one by one, and in the order given (the words are numbered through)."""
    from axonn_amd import ops

    sizes = [(i * 37) % 600 + 1 for i in range(150)]
    (g, p, m, v, lo), _ = lists(sizes, torch.bfloat16, low=torch.bfloat16)
    p2 = [t.clone() for t in p]
    if not eightbit:
        m2, v2 = [t.clone() for t in m], [t.clone() for t in v]
        ops.mt_adamw(g, p, m, v, lo, hparams(2))
        for i in range(150):
            ops.mt_adamw([g[i]], [p2[i]], [m2[i]], [v2[i]], None, hparams(2))
        assert all(torch.equal(a, b) for a, b in zip(p + m + v, p2 + m2 + v2))
        return
    codes, exps = eight(sizes)
    state = [[x.cpu().numpy().copy() for x in xs] for xs in (codes, exps)]
    old = [n64(t) for t in g], [n64(t) for t in p]
    ops.mt_adamw8(g, p, codes, exps, lo, hparams(2), 99)
    first = 0
    for i in range(150):
        _, wc, we = oa.step8(old[0][i], old[1][i], state[0][i], state[1][i], 99, 2, *HP.values(), first=first)
        first += len(we)
        assert np.array_equal(codes[i].cpu().numpy(), wc) and np.array_equal(exps[i].cpu().numpy(), we), i


@pytest.mark.parametrize("eightbit", [False, True])
def test_scan_result_clips_and_skips(eightbit):
    from axonn_amd import ops

    sizes = [300, 1025]

    def run(scale_g, max_norm, bad=None):
        (g, p, m, v, lo), _ = lists(sizes, torch.float16, low=torch.float16)
        for t in g:
            t.mul_(scale_g)
        if bad is not None:
            g[1][7] = bad
        codes, exps = eight(sizes)
        state = (codes, exps) if eightbit else (m, v)
        before = [t.clone() for ts in (p, lo, *state) for t in ts]
        scan = ops.mt_scan(g, 0.5, max_norm)
        if eightbit:
            ops.mt_adamw8(g, p, codes, exps, lo, hparams(4), 11, 0.5, scan)
        else:
            ops.mt_adamw(g, p, m, v, lo, hparams(4), 0.5, scan)
        return before, [t for ts in (p, lo, *state) for t in ts], scan, g

    for bad in (float("inf"), float("nan")):   # the step is skipped: nothing is written
        before, after, scan, _ = run(1.0, 1.0, bad)
        assert int(scan.found_inf) == 1 and all(torch.equal(a, b) for a, b in zip(before, after))
    before, after, scan, g = run(1.0, 1.0)
    clip = float(scan.clip_coef)
    assert clip < 0.1
    first = 0
    for i, n in enumerate(sizes):
        args = (n64(g[i]), n64(before[i]))
        if eightbit:
            wp, wc, we = oa.step8(*args, before[4 + i].cpu().numpy(), before[6 + i].cpu().numpy(), 11, 4, *HP.values(),
                                  inv_scale=0.5, clip=clip, first=first)
            first += len(we)
            assert np.array_equal(after[4 + i].cpu().numpy(), wc) and np.array_equal(after[6 + i].cpu().numpy(), we)
        else:
            wp, _, _ = oa.step(*args, n64(before[4 + i]), n64(before[6 + i]), 4, *HP.values(), inv_scale=0.5, clip=clip)
        check_p(after[i], wp, args[1], update_of(args[1], wp))


def test_moments_read_back():
    from axonn_amd import ops

    rng = np.random.default_rng(4)
    codes = rng.integers(0, 256, (9, 512)).astype(np.uint8)
    exps = rng.integers(30, 200, (9, 2)).astype(np.uint8)
    exps[3], exps[4] = (255, 100), (100, 255)
    exps[5], exps[6] = (0, 0), (254, 254)
    c, e = torch.tensor(codes, device="cuda"), torch.tensor(exps, device="cuda")
    wm, wv = (x.astype(np.float32).reshape(-1) for x in oa.decode(codes, exps))
    for n in (9 * 256, 9 * 256 - 1, 8 * 256 + 1):
        m, v = ops.adamw8_moments(c, e, n)
        assert m.shape == v.shape == (n,)
        assert np.array_equal(m.cpu().numpy(), wm[:n], equal_nan=True) and np.array_equal(v.cpu().numpy(), wv[:n], equal_nan=True)
        mb, vb = ops.adamw8_moments(c, e, n, torch.bfloat16)
        assert torch.equal(mb.float().nan_to_num(7), m.bfloat16().float().nan_to_num(7))
        assert torch.equal(vb.float().nan_to_num(7), v.bfloat16().float().nan_to_num(7))
    normal = np.abs(wm) >= 2.0 ** -126   # what bf16's own range holds it holds exactly
    assert np.array_equal(ops.adamw8_moments(c, e, dtype=torch.bfloat16)[0].float().cpu().numpy()[normal], wm[normal])
    m, v = ops.adamw8_moments(*ops.adamw8_state(0))
    assert m.numel() == v.numel() == 0
    for bad in (dict(dtype=torch.float16),):
        with pytest.raises(TypeError):
            ops.adamw8_moments(c, e, **bad)
    for bad in ((c, e, 8 * 256), (c.float(), e), (c[:8], e), (c, e[:, :1])):
        with pytest.raises(ValueError):
            ops.adamw8_moments(*bad)


def test_values_at_the_ends_of_the_codes():
    """Zero, denormal and huge gradients, and a second moment at its smallest code: as the oracle, and never 0 / eps."""
    from axonn_amd import ops

    for size in (0.0, 1e-30, 1e-22, 1e-10, 1e4, 1e12, 1e17):
        g = torch.randn(512, device="cuda") * size
        g[::3] = 0
        g[1] = size * 1e-6
        p = torch.randn(512, device="cuda")
        codes, exps = ops.adamw8_state(512)
        for t in (1, 2):
            state, old = (codes.cpu().numpy().copy(), exps.cpu().numpy().copy()), (n64(g), n64(p))
            ops.mt_adamw8([g], [p], [codes], [exps], None, hparams(t), t)
            _, wc, we = oa.step8(*old, *state, t, t, *HP.values())
            assert np.array_equal(exps.cpu().numpy(), we) and np.array_equal(codes.cpu().numpy(), wc), size
        m, v = ops.adamw8_moments(codes, exps)
        assert torch.isfinite(p).all() and ((v > 0) | (g == 0) | (size < 1e-15)).all()


def test_a_gradient_that_is_not_finite_marks_its_block():
    from axonn_amd import ops

    for bad in (float("nan"), float("inf"), -float("inf"), 1e25):   # (the last one's square overflows: v alone)
        g = torch.ones(700, device="cuda")
        g[300] = bad
        p = torch.ones(700, device="cuda")
        codes, exps = ops.adamw8_state(700)
        ops.mt_adamw8([g], [p], [codes], [exps], None, hparams(1), 0)
        e = exps.cpu().numpy()
        assert e[1, 1] == 255 and (e[1, 0] == 255) == (abs(bad) > 1e30 or bad != bad) and (e[[0, 2]] < 255).all()
        v = ops.adamw8_moments(codes, exps, 700)[1]
        assert torch.isnan(v[256:512]).all() and torch.isfinite(v[:256]).all() and torch.isfinite(v[512:]).all()
        ops.mt_adamw8([torch.ones_like(g)], [p], [codes], [exps], None, hparams(2), 0)
        assert torch.isnan(p[256:512]).all() and torch.isfinite(p[:256]).all() and torch.isfinite(p[512:]).all()


def test_equal_calls_are_equal_and_seeds_differ():
    from axonn_amd import ops

    out = []
    for seed in (1, 1, 2, 1 << 40):
        (g, p, _, _), _ = lists([5000], torch.float32)
        codes, exps = ops.adamw8_state(5000)
        ops.mt_adamw8(g, p, [codes], [exps], None, hparams(1), seed)
        out.append((p[0].clone(), codes, exps))
    assert all(torch.equal(a, b) for a, b in zip(out[0], out[1]))
    for other in out[2:]:
        assert torch.equal(out[0][0], other[0]) and torch.equal(out[0][2], other[2])
        assert (out[0][1] != other[1]).float().mean() > 0.1


def test_lists_that_do_not_fit_are_refused():
    from axonn_amd import ops

    (g, p, m, v, lo), _ = lists([40, 300], torch.bfloat16, low=torch.bfloat16)
    codes, exps = eight([40, 300])
    good = [g, p, m, v, lo]
    good8 = [g, p, codes, exps, lo]
    hp = hparams(1)
    for i in range(5):
        with pytest.raises(ValueError, match="lengths"):
            ops.mt_adamw(*[t[:1] if k == i else t for k, t in enumerate(good)], hp)
        with pytest.raises(ValueError, match="lengths"):
            ops.mt_adamw8(*[t[:1] if k == i else t for k, t in enumerate(good8)], hp, 0)
    short = lambda ts: [ts[0], ts[1][:-1]]  # noqa: E731
    for i in range(1, 5):
        with pytest.raises(ValueError, match="sizes"):
            ops.mt_adamw(*[short(t) if k == i else t for k, t in enumerate(good)], hp)
    for i in (1, 4):
        with pytest.raises(ValueError, match="sizes"):
            ops.mt_adamw8(*[short(t) if k == i else t for k, t in enumerate(good8)], hp, 0)
    for i in (2, 3):
        with pytest.raises(ValueError, match="bytes"):
            ops.mt_adamw8(*[short(t) if k == i else t for k, t in enumerate(good8)], hp, 0)
    with pytest.raises(ValueError, match="bytes"):
        ops.mt_adamw8(g, p, m, v, lo, hp, 0)
    for bad in ([g, m[:1] + [p[1].double()], m, v, lo], [g, [t.half() for t in p], m, v, lo], [[g[0], g[1].half()], p, m, v, lo],
                [g, p, [t.half() for t in m], v, lo], [g, p, m, [t.half() for t in v], lo],
                [[t.double() for t in g], p, m, v, lo]):
        with pytest.raises(TypeError):
            ops.mt_adamw(*bad, hp)
    with pytest.raises(ValueError, match="contiguous"):
        ops.mt_adamw([torch.ones(600, device="cuda")[::2]], [p[1]], [m[1]], [v[1]], None, hp)
    with pytest.raises(RuntimeError, match="overlap"):   # the same tensor twice
        ops.mt_adamw([g[1], g[1]], [p[1], p[1]], [m[1], m[1].clone()], [v[1], v[1].clone()], None, hp)
    with pytest.raises(RuntimeError, match="overlap"):
        ops.mt_adamw8([g[1], g[1]], [p[1], p[1].clone()], [codes[1], codes[1]], [exps[1], exps[1].clone()], None, hp, 0)
    with pytest.raises(RuntimeError, match="copy"):
        ops.mt_adamw(g, p, m, v, [t.float() for t in p], hp)
    ops.mt_adamw([], [], [], [], None, hp)
    ops.mt_adamw8([], [], [], [], None, hp, 0)


def test_replayed_step_equals_the_eager_one():
    from axonn_amd import ops

    sizes = [300, 5000, 257]
    (g, p, m, v, lo), flat = lists(sizes, torch.bfloat16, low=torch.bfloat16)
    codes, exps = eight(sizes)
    p8 = [t.clone() for t in p]
    live = [*p, *m, *v, *lo, *codes, *exps, *p8]

    def both():
        scan = ops.mt_scan(g, 1.0, 1.0)
        ops.mt_adamw(g, p, m, v, lo, hparams(2), scan=scan)
        ops.mt_adamw8(g, p8, codes, exps, None, hparams(2), 5, scan=scan)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    start = [t.clone() for t in live]
    with torch.cuda.graph(graph):
        both()
    for i in range(3):
        flat[0].normal_(generator=torch.Generator(device="cuda").manual_seed(i))
        before = [t.clone() for t in live]
        both()
        want = [t.clone() for t in live]
        for t, s in zip(live, before):
            t.copy_(s)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(live, want))
    assert not torch.equal(start[0], live[0])


def test_offsets_beyond_32_bits():
    """The last block of a tensor of 2^31 + 2^29 + 5 elements, whose codes end past 4 GiB and weights past 8."""
    from axonn_amd import ops

    n = (1 << 31) + (1 << 29) + 5
    p, g = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda", dtype=torch.bfloat16)
    g[-300:], p[-300:] = torch.randn(300, device="cuda").bfloat16(), torch.randn(300, device="cuda")
    codes, exps = ops.adamw8_state(n)
    first = (n - 300) // 256                       # a whole block in front of the last one, and that one
    lo = first * 256
    old = n64(g[lo:]), n64(p[lo:]), codes[first:].cpu().numpy(), exps[first:].cpu().numpy()
    ops.mt_adamw8([g], [p], [codes], [exps], None, hparams(1), 3)
    wp, wc, we = oa.step8(*old, 3, 1, *HP.values(), first=first)
    assert np.array_equal(codes[first:].cpu().numpy(), wc) and np.array_equal(exps[first:].cpu().numpy(), we)
    check_p(p[lo:], wp, old[1], update_of(old[1], wp))
    m, _ = ops.adamw8_moments(codes, exps, n)
    assert np.array_equal(m[lo:].cpu().numpy(), oa.decode(wc, we)[0].reshape(-1)[:n - lo].astype(np.float32))
    assert not codes[:first].any() and not exps[:first].any() and not m[:lo].any()


# ------------------------------------------------------------ the optimizer --
def small_params(dtype, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.nn.Parameter((torch.randn(*s, generator=gen, device="cuda") * 0.1).to(dtype))
            for s in ((3,), (17, 31), (256,), (40, 64), (1,))]


@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_against_torch(bits):
    """Four steps of two groups: fp32 moments as torch.optim.AdamW in 64 bits; with 8 bits the first step (from zero
    moments, whose update does not depend on codes) does, and later moments are within a step of their codes."""
    from axonn_amd.optim import AdamW

    params = small_params(torch.float32)
    twins = [torch.nn.Parameter(p.detach().double().cpu()) for p in params]
    groups = lambda ps: [dict(params=ps[:2], lr=1e-2), dict(params=ps[2:], weight_decay=0.3)]  # noqa: E731
    opt = AdamW(groups(params), lr=3e-3, weight_decay=0.05, state_bits=bits)
    ref = torch.optim.AdamW(groups(twins), lr=3e-3, weight_decay=0.05)
    for t in range(4):
        for p, q in zip(params, twins):
            g = torch.randn(p.shape, generator=torch.Generator().manual_seed(31 * t + p.numel()))
            p.grad.copy_(g)
            q.grad = g.double()
        opt.step()
        ref.step()
        if bits == 32 or t == 0:
            for p, q in zip(params, twins):
                # three constants and some twenty operations a step, updates of at most lr (and decay) each
                assert (p.detach().double().cpu() - q.detach()).abs().max() <= (t + 1) * 32 * U * (q.detach().abs().max() + 1e-2)
        if t == 0:
            for (m, v), p, q in zip(opt.moments(), params, twins):
                s = ref.state[q]
                for mine, theirs in ((m, s["exp_avg"]), (v, s["exp_avg_sq"])):
                    assert mine.shape == p.shape
                    off = (mine.double().cpu() - theirs).abs()
                    least = theirs.abs().max() * (2.0 ** -17 if mine is m else 2.0 ** -33)
                    rel = 4 * U if bits == 32 else 1 / 8 + 4 * U
                    assert (off <= rel * theirs.abs() + (least if bits == 8 else 0)).all()
    assert opt.step_count == 4 and not opt.last_step_skipped


@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_scales_clips_and_skips(bits):
    """fp16 parameters with dynamic loss scaling: an overflow leaves everything, the step that follows uses the halved
    scale; and `.grad`s that were rebound are found."""
    from axonn_amd.optim import AdamW

    params = small_params(torch.float16)
    opt = AdamW(params, lr=1e-2, max_grad_norm=1.0, state_bits=bits)
    assert opt.dynamic_loss_scale
    state = [opt.model_params_fp32, opt.model_params_fp16] + ([opt.codes, opt.exponents] if bits == 8 else
                                                             [opt.exp_avg, opt.exp_avg_sq])
    scale = opt.loss_scale
    for p in params:
        p.grad.copy_(torch.ones_like(p) * 0.01)
    params[1].grad[0, 0] = float("inf")
    before = [t.clone() for t in state]
    opt.step()
    assert opt.last_step_skipped and opt.step_count == 0 and opt.loss_scale == scale / 2
    assert all(torch.equal(a, b) for a, b in zip(before, state))
    opt.zero_grad()
    for p in params:
        p.grad = torch.full_like(p, 1e-3)      # rebound
    opt.step()
    assert not opt.last_step_skipped and opt.step_count == 1
    n = sum(p.numel() for p in params)
    assert abs(float(opt.grad_norm()) - 1e-3 / opt.loss_scale * n ** 0.5) < 1e-3 * float(opt.grad_norm())
    for p, old in zip(params, small_params(torch.float16)):
        want = old.detach().float() * (1 - 1e-2 * 1e-2) - 1e-2 * 1e-3 / opt.loss_scale / (1e-3 / opt.loss_scale + 1e-8)
        assert (p.detach().float() - want).abs().max() <= 2.0 ** -11 * want.abs().max() + 1e-4 * 1e-2


def test_optimizer_runs_with_equal_seeds_are_equal():
    from axonn_amd.optim import AdamW

    out = []
    for seed in (0, 0, 1):
        params = small_params(torch.bfloat16)
        opt = AdamW(params, state_bits=8, seed=seed)
        for t in range(3):
            opt.model_grads_fp16.normal_(generator=torch.Generator(device="cuda").manual_seed(t))
            opt.step()
        out.append((opt.model_params_fp32.clone(), opt.codes.clone(), opt.exponents.clone()))
    assert all(torch.equal(a, b) for a, b in zip(out[0], out[1]))
    assert not torch.equal(out[0][1], out[2][1])


@pytest.mark.parametrize("bits", [32, 8])
def test_a_block_trains(bits):
    """LayerNorm, Linear with GELU, Linear, and the residual's next norm, under AdamW: runs, gradients reach every
    parameter and equal autograd's over torch's own layers; weights move."""
    from axonn_amd.intra_layer import LayerNorm, Linear
    from axonn_amd.optim import AdamW

    torch.manual_seed(3)
    n1, n2 = LayerNorm(64).cuda(), LayerNorm(64).cuda()
    up, down = Linear(64, 256, fused_activation="gelu").cuda(), Linear(256, 64).cuda()
    modules = (n1, up, down, n2)
    params = [p for m in modules for p in m.parameters()]
    opt = AdamW(params, lr=1e-3, state_bits=bits, max_grad_norm=1.0)
    x = torch.randn(2, 33, 64, device="cuda")
    start = opt.model_params_fp32.clone()
    for _ in range(3):
        opt.zero_grad()
        y, h = n2(down(up(n1(x))), x)
        (y.square().mean() + h.mean()).backward()
        t1, t2 = (torch.nn.functional.layer_norm for _ in range(2))
        leaves = [p.detach().double().cpu().requires_grad_() for p in params]
        w1, b1, uw, ub, dw, db, w2, b2 = leaves
        xc = x.double().cpu()
        z = torch.nn.functional.gelu(t1(xc, (64,), w1, b1) @ uw.view(256, 64).t() + ub) @ dw.view(64, 256).t() + db
        (t2(z + xc, (64,), w2, b2).square().mean() + (z + xc).mean()).backward()
        for p, q in zip(params, leaves):
            # fp32 products of 64 and 256 terms, three layers deep: some hundred roundings of the largest terms
            scale = q.grad.abs().max() + 1e-3
            assert (p.grad.double().cpu().view(-1) - q.grad.view(-1)).abs().max() <= 2000 * U * scale * 4
        opt.step()
    moved = [(p.detach().view(-1) != s).any() for p, s in
             zip(params, (start[o:o + n] for o, n in opt._views))]
    assert all(moved)
