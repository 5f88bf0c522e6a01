"""The 8-bit moments' codes as oracle/adamw.py defines them (the kernels are compared with it bit by
bit): round trips, the octaves' borders, unbiased rounding, and what the rounding is for."""

import numpy as np
import pytest
import torch

from oracle import adamw as oa


def test_magnitudes_ascend_by_a_sixteenth_to_an_eighth():
    f = oa.magnitude(np.arange(256))
    assert f[0] == 0 and f[1] == 0.125 and f[127] == 1.875 * 2 ** 14 and f[255] == 1.875 * 2 ** 30
    step = np.diff(f)[8:] / f[8:-1]
    assert step.min() == 1 / 15 and step.max() == 1 / 8
    assert np.array_equal(f.astype(np.float32), f) and np.array_equal(torch.tensor(f).bfloat16().double().numpy(), f)


@pytest.mark.parametrize("bias,most", [(141, 127), (157, 255)])
def test_every_code_is_its_own_rounding(bias, most):
    c = np.arange(most + 1)
    for e in (40, 127, 200, 254):
        x = (oa.magnitude(c) * 2.0 ** (e - bias)).astype(np.float32)
        for u in (0.5 / 65536, 65535.5 / 65536):
            assert np.array_equal(oa.encode(x, e, bias, u, False), c), (e, u)


def test_exponent_borders():
    for k in (-100, -3, 0, 5, 120):
        one = np.float32(2.0 ** k)
        below, at = np.nextafter(np.float32(1.875) * one, np.float32(0)), np.float32(1.875) * one
        assert oa.exponent(one) == oa.exponent(below) == 127 + k and oa.exponent(at) == 128 + k
        for bias, most in ((141, 127), (157, 255)):   # rounded up, the largest still has a code
            assert oa.encode(below, 127 + k, bias, 65535.5 / 65536, False) == most
    assert oa.exponent(0.0) == 0 and oa.exponent(np.inf) == oa.exponent(np.nan) == 255
    # the same as the integer form that the kernels use
    bits = np.random.default_rng(0).integers(0, 0x7F800000, 20000).astype(np.uint32)
    bits = np.concatenate([bits, np.arange(0x700000 - 4, 0x700000 + 4, dtype=np.uint32), np.uint32([0, 1, 0x7F7FFFFF])])
    assert all(oa.exponent(x) == min(255, (int(b) + 0x100000) >> 23) for x, b in zip(bits.view(np.float32), bits))


def test_encoding_is_the_bits_of_a_float():
    """(bits of x 2^(bias - 126 - E) + 16 w + 8) >> 20, on magnitudes of all sizes."""
    rng = np.random.default_rng(1)
    x = np.exp2(rng.uniform(-60, 0.9, 40000)).astype(np.float32)
    w = rng.integers(0, 65536, x.size)
    for bias in (141, 157):
        y = np.ldexp(x, bias - 126 - 127).astype(np.float32)
        want = (y.view(np.uint32).astype(np.int64) + 16 * w + 8) >> 20
        assert np.array_equal(oa.encode(x, 127, bias, (w + 0.5) / 65536, False), want)


def test_rounding_is_unbiased():
    """Over all 2^16 words the mean of the codes' values is the value, to half a word's share of the step
    (and fp32's own spacing)."""
    u = (np.arange(65536) + 0.5) / 65536
    for x in np.float32([1.0, 1.03, 1.7, 0.2, 3e-4, 1e-5, 4e-10]):
        for bias in (141, 157):
            got = oa.magnitude(oa.encode(np.full(65536, x), 127, bias, u, False)) * 2.0 ** (127 - bias)
            step = max(x / 8, 2.0 ** (127 - bias - 3))
            assert abs(got.mean() - float(x)) <= step * (0.5 / 65536 + 2.0 ** -20), (x, bias)


def test_random_words_are_even():
    """Halves of the words over 2^16 elements: mean and variance of a uniform variable within 5 deviations of their
    estimates, no more correlation between places, halves or seeds than that."""
    n = 256
    sets = [oa.random_words(n, s) for s in (0, 1, 1 << 32)]
    halves = [(w & 0xFFFF).reshape(-1) / 65536 for w in sets] + [(w >> 16).reshape(-1) / 65536 for w in sets]
    halves += [halves[0].reshape(-1, 4)[:, i] for i in range(4)]
    sd = 1 / 12 ** 0.5
    for h in halves:
        assert abs(h.mean() - 0.5) < 5 * sd / h.size ** 0.5
        assert abs(h.var() - 1 / 12) < 5 * (1 / 180) ** 0.5 / h.size ** 0.5
    for group in (halves[:6], halves[6:]):
        corr = np.corrcoef(group) - np.eye(len(group))
        assert np.abs(corr).max() < 5 / group[0].size ** 0.5
    # the blocks of a list go on where the ones before end, also past 2^32 counters
    assert np.array_equal(oa.random_words(4, 9)[2:], oa.random_words(2, 9, first=2))
    assert len(np.unique(oa.random_words(2, 9, first=(1 << 26) - 1))) > 500


def test_a_second_moment_follows_its_gradients():
    """What nearest rounding cannot do: a hundred-fold larger gradient raises v, none lets it decay.  1024 elements
    follow their mean: after 1000 steps of beta2 = 0.999 the exact value, within five deviations of the mean of 1024
    roundings whose variance is at most what 1000 steps of an eighth each leave."""
    blocks, beta2 = 4, 0.999
    for grad, start in ((0.02, 1e-4), (0.0, 1e-4), (0.01, 1e-6)):
        v = np.full((blocks, 256), start, np.float32)
        m = np.zeros_like(v)
        codes, exps = oa.quantize(m, v, oa.random_words(blocks, 77))
        for t in range(1000):
            _, v = oa.moments_step(np.full((blocks, 256), grad), m, oa.decode(codes, exps)[1].astype(np.float32), 0.9, beta2)
            words = np.random.default_rng(t).integers(0, 1 << 32, (blocks, 256))
            codes, exps = oa.quantize(m, v, words)
        got = oa.decode(codes, exps)[1].mean()
        want = start * beta2 ** 1000 + grad ** 2 * (1 - beta2 ** 1000)
        # a step's rounding has variance at most step * |change|; the changes sum to |want - start| and more by 1/8
        largest = max(want, start) * 2
        deviation = (largest / 8 * (abs(want - start) * 2 + 1e-3 * largest * 1000 / 8)) ** 0.5
        assert abs(got - want) < 5 * deviation / 32, (grad, got, want)


def test_step_against_torch():
    """The 64-bit step against torch.optim.AdamW in 64 bits, four steps."""
    rng = np.random.default_rng(3)
    p = rng.normal(0, 0.1, 100)
    param = torch.nn.Parameter(torch.tensor(p))
    opt = torch.optim.AdamW([param], lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
    m = v = np.zeros(100)
    for t in range(1, 5):
        g = rng.normal(0, 1, 100)
        param.grad = torch.tensor(g)
        opt.step()
        p, m, v = oa.step(g, p, m, v, t, 1e-2, 0.9, 0.99, 1e-8, 0.1)
        assert np.abs(param.detach().numpy() - p).max() < 1e-14


def test_norm_oracle_against_torch_and_differences():
    from oracle import layer_norm as ol

    rng = np.random.default_rng(5)
    h, w, b = rng.normal(0.3, 1, (3, 10)), rng.normal(1, 0.1, 10), rng.normal(0, 0.1, 10)
    dy, dsum = rng.normal(0, 1, (3, 10)), rng.normal(0, 1, (3, 10))
    t = [torch.tensor(a, requires_grad=True) for a in (h, w, b)]
    out = torch.nn.functional.layer_norm(t[0], (10,), t[1], t[2], 1e-3)
    (out * torch.tensor(dy)).sum().backward()
    y, mean, rstd = ol.forward(h, w, b, 1e-3)
    got = ol.backward(dy, h, w, mean, rstd)
    assert np.abs(y - out.detach().numpy()).max() < 1e-13
    for a, x in zip(got, t):
        assert np.abs(a - x.grad.numpy()).max() < 1e-12
    assert np.abs(ol.backward(dy, h, w, mean, rstd, dsum)[0] - got[0] - dsum).max() < 1e-12
    # central differences of the loss sum(y dy), step 1e-5: off by some 1e-10 of their second order
    for i, a in enumerate((h, w, b)):
        for at in [(0,) * a.ndim, (a.shape[0] - 1,) * a.ndim]:
            loss = []
            for s in (1e-5, -1e-5):
                moved = [h.copy(), w.copy(), b.copy()]
                moved[i][at] += s
                loss.append((ol.forward(*moved, 1e-3)[0] * dy).sum())
            assert abs((loss[0] - loss[1]) / 2e-5 - got[i][at]) < 1e-7
