"""CPU tests of the 8-bit Adam step over many steps, on its numpy restatements (the device equals them bit for bit): where parameters and first moments go, against Adam in 64 bits.

Bounds. The first moment is right in the mean; the root of the second is held to one step of its grid, at most 1/16 of it, and the rounding of r adds up to 3.2 % to the mean of v = r^2
(1.6 % of r) once steps are many: a mean parameter change is within 3 % of the exact one. A single element's parameter may be off by some 16 % of its whole way, so a mean over n elements is
allowed 2 * 0.16 / sqrt(n) more."""
import numpy as np
import pytest

import adam8_ref as A8
import adam8_threshold_ref as T8

LR = 1e-3


def run(step, grads, steps, b1, n):
    """(p, m, r) of the 8-bit run, (p, m) of Adam in 64 bits"""
    p, codes = np.zeros(n, np.float32), (np.zeros(n, np.uint8), np.zeros(n, np.uint8), np.zeros((n // 64, 2), np.int8))
    x, m, v = np.zeros(n), np.zeros(n), np.zeros(n)
    for t in range(1, steps + 1):
        g = grads(t).astype(np.float32)
        p, codes = step(p, g, codes, t, LR, b1, 0.999, 1e-8)
        g = g.astype(np.float64)
        m, v = b1 * m + (1 - b1) * g, 0.999 * v + 0.001 * g * g
        x = x - LR / (1 - b1 ** t) * m / (np.sqrt(v / (1 - 0.999 ** t)) + 1e-8)
    return p.astype(np.float64), *A8.decode(*codes), x, m


def near(p, x):
    way = np.abs(x).mean()
    assert np.abs(p.mean() - x.mean()) <= (0.03 + 0.32 / np.sqrt(p.size)) * way, (p.mean(), x.mean())
    assert np.abs(p - x).max() <= way, (p.min(), p.max(), x.mean())


@pytest.mark.parametrize("b1", [0.9, 0.95, 0.99])
def test_constant_gradient(b1):
    p, m, _, x, exact = run(T8.step, lambda t: np.full(256, 0.01), 300, b1, 256)
    near(p, x)
    # With a = 1 - b1 and a grid step s <= g / 8, a step that should move m by a (g - m) moves it by s with probability a (g - m) / s: variance s a (g - m) at most, and every step after it
    # takes b1^2 of what there is. m(t) = g (1 - e^-at), so the variance is s g a * integral of e^-2a(t-u) e^-au du = s g (e^-at - e^-2at) <= s g / 4 = (0.177 g)^2. Once m has arrived it
    # sits on one of two neighbours: s / 2 = 0.0625 g more at most. 5 of these deviations for an element among 256, 4 over 16 for their mean.
    dev = (0.177 + 0.0625) * 0.01
    assert np.sqrt(np.mean((m - exact) ** 2)) <= dev and np.abs(m - exact).max() <= 5 * dev and abs(m.mean() - exact[0]) <= 4 * dev / 16


@pytest.mark.parametrize("b1", [0.9, 0.95, 0.99])
def test_gradient_that_stops(b1):
    p, m, _, x, _ = run(T8.step, lambda t: np.full(256, 1.0 if t <= 100 else 0.0), 2000, b1, 256)
    near(p, x)
    assert np.abs(m).max() <= 1e-6


@pytest.mark.parametrize("b1", [0.9, 0.95, 0.99])
def test_gradient_that_stops_in_half_of_a_block(b1):
    """the others of the block keep its scale up, the root decays to its smallest code: nothing may be left of the first moment"""
    g = np.random.RandomState(0)
    dead = np.arange(128) % 64 < 32
    p, m, _, x, _ = run(T8.step, lambda t: np.where(dead, 1.0 if t <= 100 else 0.0, g.randn(128)), 20000, b1, 128)
    near(p[dead], x[dead])
    assert not m[dead].any()
    # The others (gradients of mean 0, deviation 1) walk at random. A rounding of m is off by a deviation of s / 2 at most, s <= |m| / 8, m^2 = a / 2 in the mean; over the steps it moves p by
    # lr / a times that, independently at every step: variance lr^2 N (a / 2 / 64 / 4) / a^2 = lr^2 N / (512 a). 5 deviations for an element among 64.
    assert np.abs(p[~dead] - x[~dead]).max() <= 5 * LR * np.sqrt(20000.0 / (512 * (1 - b1)))


def test_rounding_to_nearest_does_not_follow():
    """what the thresholds are for: a constant gradient is held too small, and a stopped one drives its parameter on"""
    p, m, _, x, exact = run(A8.step, lambda t: np.full(64, 0.01), 300, 0.9, 64)
    assert m.max() < 0.8 * exact[0] and p.mean() > 0.85 * x.mean()                # (both negative)
    p, m, _, x, _ = run(A8.step, lambda t: np.full(64, 1.0 if t <= 100 else 0.0), 2000, 0.95, 64)
    assert m.min() > 0.3 and p.max() < 10 * x.mean()


def test_threshold_rounding_of_a_first_moment():
    """every value lands on one of its two neighbours on the grid, with the mean of many thresholds on the value; signs and what is not finite are kept; grid points stay"""
    g = np.random.RandomState(3)
    y = np.concatenate([g.randn(4096) * np.exp(2 * g.randn(4096)), [0.0, -0.0, 2.0 ** -9, -(2.0 ** -6), 256.0, 2.0 ** -20]]).astype(np.float32)
    y = np.clip(y, -256, 256)
    total = np.zeros(y.size)
    grid = np.unique(A8.E4M3[np.isfinite(A8.E4M3)]).astype(np.float64)
    below = grid[np.searchsorted(grid, y, side="right") - 1]
    above = grid[np.searchsorted(grid, y, side="left")]
    for t in range(400):
        v = A8.E4M3[T8.encode_e4m3(y, T8.m_thresholds(y.size, t))].astype(np.float64)
        assert np.all((v == below) | (v == above)) and np.array_equal(np.signbit(v), np.signbit(y))
        total += v
    # standard deviation of one rounding at most half a step; 6 of them over sqrt(400) for every element, 6 over sqrt(400 n) for all
    step = np.maximum(above - below, 1e-30)
    off = (total / 400 - y) / step
    assert np.abs(off).max() <= 6 * 0.5 / 20 and abs(off.mean()) <= 6 * 0.5 / 20 / np.sqrt(y.size)
    bad = T8.encode_e4m3(np.array([np.nan, np.inf, -np.inf], np.float32), np.array([8, 8, 8], np.uint32))
    assert (bad == 0x7F).all()


def test_adam8_step_refuses_another_rounding():
    import torch

    from med_ts_llm_amd.hip import _native as N
    from med_ts_llm_amd.hip import optim
    p, g = torch.zeros(10, 7), torch.zeros(10, 7)
    with pytest.raises(ValueError):
        optim.adam8_step([p], [g], [optim.adam8_state(p)], 1, first_moment="up")
    assert N.lib().mtl_adam8_step(None, 0, 1e-3, 0.9, 0.999, 1e-8, 0.0, 4, 1, None) == -1 and N.lib().mtl_adam8_step(None, 0, 1e-3, 0.9, 0.999, 1e-8, 0.0, 3, 1, None) == 0


def test_gradient_whose_square_overflows():
    """one finite gradient beyond 1.8e19: the second moment is infinite from there on and the parameter stands still (as with 32-bit moments); its neighbours go on"""
    g = np.random.RandomState(5)
    p, codes = np.zeros(128, np.float32), (np.zeros(128, np.uint8), np.zeros(128, np.uint8), np.zeros((2, 2), np.int8))
    for t in range(1, 31):
        x = g.randn(128).astype(np.float32)
        if t == 10:
            x[3], x[70], held = 1e20, -3e38, p[[3, 70]]
        p, codes = T8.step(p, x, codes, t, LR, 0.9, 0.999, 1e-8)
        if t >= 10:
            assert np.array_equal(p[[3, 70]], held) and codes[1][3] == 254 and codes[1][70] == 254
    assert np.isfinite(p).all()
    old = (np.zeros(64, np.uint8), np.zeros(64, np.uint8), np.zeros((1, 2), np.int8))           # with every root that is not finite as NaN the parameter is lost
    q = np.zeros(64, np.float32)
    for x in (np.full(64, 1e20, np.float32), np.ones(64, np.float32)):
        q, old = A8.step(q, x, old, 1, LR, 0.9, 0.999, 1e-8)
    assert np.isnan(q).all()
