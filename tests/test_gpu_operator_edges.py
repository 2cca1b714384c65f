"""GPU tests of the token table, the query / key norm and the 8-bit Adam step where a call's effect reaches beyond the call: runs of many steps, values at the ends of their range, state read
beside a running update, views and versions of what is written."""
import numpy as np
import pytest
import torch

import adam8_ref as A8
import adam8_threshold_ref as T8
from test_gpu_operators import codes_of, gen, np_of, randn

pytestmark = pytest.mark.gpu
F32, BF16, F64 = torch.float32, torch.bfloat16, torch.float64


@pytest.fixture(scope="module")
def ops():
    from med_ts_llm_amd.hip import ops
    return ops


@pytest.fixture(scope="module")
def optim():
    from med_ts_llm_amd.hip import optim
    return optim


# ================================================================================================ first moment against thresholds
@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("wd,decoupled", [(0.0, False), (0.01, False), (0.01, True)])
def test_adam8_threshold_step_bit_for_bit(optim, dt, wd, decoupled):
    """parameters, codes and exponents equal the numpy restatement's bits over six steps: odd sizes, unaligned views, gradients of every magnitude, zeros, NaN and infinities"""
    g = gen(3)
    sizes = [1, 3, 63, 64, 65, 1000, 4097, 70001]
    base = [randn(g, n + 1, dtype=dt, std=0.1) for n in sizes]
    ps = [b[1:] if i % 2 else b[:-1] for i, b in enumerate(base)]
    sts = [optim.adam8_state(p) for p in ps]
    want = [(np_of(p), codes_of(st)) for p, st in zip(ps, sts)]
    for t in range(1, 7):
        gs = [(randn(g, p.numel()) * torch.exp(3 * randn(g, p.numel()))).to(dt) * 10.0 ** (t - 4) for p in ps]
        if t > 1:
            gs[5][100:300] = 0
        if t == 4:
            gs[5][10], gs[5][11], gs[6][64] = np.nan, np.inf, -np.inf
        optim.adam8_step(ps, gs, sts, t, lr=1e-2, weight_decay=wd, decoupled_weight_decay=decoupled, first_moment="threshold")
        for i, (p, gr, st) in enumerate(zip(ps, gs, sts)):
            wp, wc = T8.step(want[i][0], np_of(gr), want[i][1], t, 1e-2, 0.9, 0.999, 1e-8, wd, decoupled)
            if dt == BF16:
                wp = torch.from_numpy(wp).to(BF16).float().numpy()
            want[i] = (wp, wc)
            assert np.array_equal(np_of(p), wp, equal_nan=True), (t, sizes[i])
            for a, b, what in zip(codes_of(st), wc, "mre"):
                assert np.array_equal(a, b), (t, sizes[i], what, np.flatnonzero(a != b)[:5])


def test_adam8_threshold_step_of_a_large_tensor(optim):
    """elements behind 2^31 get thresholds of their own index"""
    n = (1 << 31) + 4097
    big, gr = torch.zeros(n, dtype=BF16, device="cuda"), torch.full((n,), 1e-3, dtype=BF16, device="cuda")
    lo = (n - 1) // 64 * 64 - 4096
    gr[lo:] = randn(gen(1), n - lo, dtype=BF16, std=1e-3)
    st = optim.adam8_state(big)
    optim.adam8_step([big], [gr], [st], 1, lr=1e-2, first_moment="threshold")
    k = n - lo
    zero = (np.zeros(k, np.uint8), np.zeros(k, np.uint8), np.zeros(((k + 63) // 64, 2), np.int8))
    wp, wc = T8.step(np.zeros(k, np.float32), np_of(gr[lo:]), zero, 1, 1e-2, 0.9, 0.999, 1e-8, first=lo)
    assert np.array_equal(np_of(big[lo:]), torch.from_numpy(wp).to(BF16).float().numpy())
    assert np.array_equal(st.exp_avg[lo:].cpu().numpy(), wc[0]) and np.array_equal(st.exp_avg_sq[lo:].cpu().numpy(), wc[1])


@pytest.mark.parametrize("b1", [0.9, 0.95])
def test_hip_adam_8_follows_gradients_over_many_steps(optim, b1):
    """a constant gradient moves its parameters as exact Adam does; one that stops in half of every block stops moving them (bounds: tests/test_adam8_trajectory.py)"""
    p = torch.zeros(4096, device="cuda", requires_grad=True)
    opt = optim.HipAdam([p], lr=1e-3, betas=(b1, 0.999), state_bits=8)
    for _ in range(300):
        p.grad = torch.full_like(p, 0.01)
        opt.step()
    assert abs(p.mean().item() + 0.3) <= (0.03 + 0.32 / 64) * 0.3 and (p + 0.3).abs().max() <= 0.3
    g = gen(4)
    q = torch.zeros(4096, device="cuda", requires_grad=True)
    opt = optim.HipAdam([q], lr=1e-3, betas=(b1, 0.999), state_bits=8)
    dead = torch.arange(4096, device="cuda") % 64 < 32
    x = m = v = 0.0
    for t in range(1, 10001):
        one = 1.0 if t <= 100 else 0.0
        q.grad = torch.where(dead, one, randn(g, 4096))
        opt.step()
        m, v = b1 * m + (1 - b1) * one, 0.999 * v + 0.001 * one
        x -= 1e-3 / (1 - b1 ** t) * m / ((v / (1 - 0.999 ** t)) ** 0.5 + 1e-8)
    off = (q.detach()[dead] - x).abs()
    assert off.mean().item() <= 0.16 * abs(x) and off.max().item() <= abs(x) and not opt.moments()[q][0][dead].any()


def test_hip_adam_8_takes_thresholds(optim):
    """HipAdam(state_bits=8) is adam8_step(first_moment="threshold"); without an answer adam8_step rounds to nearest and says so"""
    g = gen(5)
    p = randn(g, 33, 70).requires_grad_()
    ref, st = p.detach().clone(), optim.adam8_state(p)
    other, so = p.detach().clone(), optim.adam8_state(p)
    opt = optim.HipAdam([p], lr=1e-2, state_bits=8)
    optim._said_nearest = False
    for t in range(1, 4):
        p.grad = randn(g, 33, 70, std=1e-2)
        opt.step()
        optim.adam8_step([ref], [p.grad], [st], t, lr=1e-2, first_moment="threshold")
        if t == 1:
            with pytest.warns(UserWarning, match="nearest"):
                optim.adam8_step([other], [p.grad], [so], t, lr=1e-2)
        else:
            optim.adam8_step([other], [p.grad], [so], t, lr=1e-2, first_moment="nearest")
    assert torch.equal(p, ref) and torch.equal(opt.state[p]["exp_avg_q"], st.exp_avg) and not torch.equal(other, ref)


# ================================================================================================ ends of the range
@pytest.mark.parametrize("dt", [F32, BF16])
def test_adam8_gradient_whose_square_overflows(optim, dt):
    """finite gradients beyond 1.8e19: parameters finite and where torch's Adam leaves them, codes as the restatement's; infinities and NaN still make their own element NaN"""
    g = gen(6)
    n = 4099
    p = randn(g, n, dtype=dt)
    q = p.float().clone().requires_grad_()
    wide = torch.optim.Adam([q], lr=1e-2)
    st = optim.adam8_state(p)
    huge = torch.tensor([0, 5, 64, 1000, 1001, n - 1], device="cuda")
    wp, wc = np_of(p), codes_of(st)
    for t in range(1, 9):
        gr = randn(g, n, dtype=dt)
        if t == 3:
            gr[huge] = torch.tensor([1e20, -1e20, 3e38, -3e38, 2e19, 1e30], device="cuda").to(dt)
            held = p[huge].clone()
        if t == 6:
            gr[7], gr[900] = float("inf"), float("nan")
        q.grad = gr.float()
        wide.step()
        optim.adam8_step([p], [gr], [st], t, lr=1e-2, first_moment="threshold")
        wp, wc = T8.step(wp, np_of(gr), wc, t, 1e-2, 0.9, 0.999, 1e-8)
        if dt == BF16:
            wp = torch.from_numpy(wp).to(BF16).float().numpy()
        assert np.array_equal(np_of(p), wp, equal_nan=True) and all(np.array_equal(a, b) for a, b in zip(codes_of(st), wc)), t
        if t >= 3:
            assert torch.equal(p[huge], held) and bool((st.exp_avg_sq[huge] == 254).all()), t
            if dt == F32:
                fixed = q.detach()[huge] if t == 3 else fixed
                assert torch.equal(q.detach()[huge], fixed)
    assert p.isnan().nonzero().view(-1).tolist() == [7, 900] == q.isnan().nonzero().view(-1).tolist()
    (m, v), = optim.adam8_moments([st])
    assert bool(v[huge].isposinf().all()) and bool(m[huge].isfinite().all())
    back = optim.adam8_quantize(m, v, 8)
    assert torch.equal(back.exp_avg_sq[huge], st.exp_avg_sq[huge])


# ================================================================================================ state read beside a running update
@pytest.mark.parametrize("bits", [8, 32])
def test_moments_read_behind_a_deferred_step(optim, bits):
    """moments() and state_dict() right after a step whose update still waits on the side stream (held back there by a long kernel) give the state behind it; moments() are copies"""
    g = gen(21)
    ps = [randn(g, 700, 501).requires_grad_(), randn(g, 70).requires_grad_()]
    qs = [p.detach().clone().requires_grad_() for p in ps]
    one, two = optim.HipAdam(ps, lr=1e-2, state_bits=bits), optim.HipAdam(qs, lr=1e-2, state_bits=bits)
    two.defer(qs)
    for t in range(4):
        for p, q in zip(ps, qs):
            p.grad = randn(g, *p.shape)
            q.grad = p.grad.clone()
        one.step()
        want = one.moments()
        torch.cuda.synchronize()
        with torch.cuda.stream(two._side):
            torch.cuda._sleep(20_000_000)                       # (some 10 ms)
        two.step()
        if t % 2:
            got = two.moments()
        else:
            sd = two.state_dict()["state"]
            names = ("exp_avg_q", "exp_avg_sq_q") if bits == 8 else ("exp_avg", "exp_avg_sq")
            got = {q: tuple(sd[i][k].clone() for k in names) for i, q in enumerate(qs)}
            want = {p: tuple(one.state[p][k] for k in names) for p in ps}
        assert two._late_done is not None                       # (still there for the stream that reads the parameters)
        assert all(torch.equal(a, b) for p, q in zip(ps, qs) for a, b in zip(want[p], got[q])), t
        two.wait_deferred()
    m = two.moments()[qs[0]][0]
    before = m.clone()
    two.step()
    two.wait_deferred()
    assert torch.equal(m, before) and not torch.equal(two.moments()[qs[0]][0], before)


# ================================================================================================ views and versions of what is written
def test_overwriting_what_a_backward_pass_needs_is_noticed(ops):
    """queries that QkNormRopeFn saved, rotated in place afterwards, and a table gradient written over a saved tensor: the backward pass raises instead of using the new values"""
    g = gen(30)
    a = torch.arange(8, device="cuda", dtype=F32)[:, None] * torch.ones(16, device="cuda")
    w, cos, sin = torch.ones(16, device="cuda"), a.cos(), a.sin()
    q, k = randn(g, 2, 8, 64).requires_grad_(), randn(g, 2, 8, 32)
    x = q * 1.0
    y, _ = ops.QkNormRopeFn.apply(x, k, w, w, cos, sin, 4, 2, 16)
    with torch.no_grad():
        ops.qk_norm_rope_fwd(x, k, w, w, cos, sin, 4, 2, 16, out=(x, k))
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()
    table = randn(g, 20, 8).requires_grad_()
    t = table * 1.0
    z = (t * t).sum()
    ops.embedding_bwd(randn(g, 5, 8), torch.arange(5, device="cuda"), 20, out=t.detach())
    with pytest.raises(RuntimeError, match="inplace"):
        z.backward()


def test_qk_norm_rope_out_of_one_allocation(ops):
    """queries and a key cache in one arena, one part per sequence; outputs beside the inputs in their own buffer: the same values, nothing else touched"""
    g = gen(31)
    B, Hq, Hkv, D, L = 3, 4, 2, 64, 9
    a = torch.arange(L, device="cuda", dtype=F32)[:, None] * torch.logspace(0, -2, 64, device="cuda")
    cos, sin, w = a.cos(), a.sin(), 1 + randn(g, D, std=0.1)
    q, k = randn(g, B, 1, Hq * D, dtype=BF16), randn(g, B, 1, Hkv * D, dtype=BF16)
    yq, yk = ops.qk_norm_rope_fwd(q, k, w, w, cos, sin, Hq, Hkv, D, pos0=5)
    arena = torch.full((B, Hq * D + L * Hkv * D), 7.0, dtype=BF16, device="cuda")
    to = arena[:, None, :Hq * D], arena[:, Hq * D:].unflatten(1, (L, Hkv * D))[:, 5:6]
    ops.qk_norm_rope_fwd(q, k, w, w, cos, sin, Hq, Hkv, D, pos0=5, out=to)
    assert torch.equal(to[0], yq) and torch.equal(to[1], yk)
    to[0].fill_(7.0), to[1].fill_(7.0)
    assert bool((arena == 7.0).all())
    fused = randn(g, B, L, 2 * (Hq + Hkv) * D)
    kept = fused.clone()
    q, k = fused[..., :Hq * D], fused[..., Hq * D:(Hq + Hkv) * D]
    want = ops.qk_norm_rope_fwd(q, k, w, w, cos, sin, Hq, Hkv, D)
    to = fused[..., (Hq + Hkv) * D:(2 * Hq + Hkv) * D], fused[..., (2 * Hq + Hkv) * D:]
    ops.qk_norm_rope_fwd(q, k, w, w, cos, sin, Hq, Hkv, D, out=to)
    assert torch.equal(to[0], want[0]) and torch.equal(to[1], want[1]) and torch.equal(fused[..., :(Hq + Hkv) * D], kept[..., :(Hq + Hkv) * D])
    dq, dk = randn(g, B, L, Hq * D), randn(g, B, L, Hkv * D)
    want = ops.qk_norm_rope_bwd(dq, dk, q, k, w, w, cos, sin, Hq, Hkv, D)
    got = ops.qk_norm_rope_bwd(dq, dk, q, k, w, w, cos, sin, Hq, Hkv, D, out=to)
    assert all(torch.equal(x, y) for x, y in zip(got, want)) and torch.equal(fused[..., :(Hq + Hkv) * D], kept[..., :(Hq + Hkv) * D])
