"""GPU tests of the token table (lookup, gradient), the query / key norm with rotation, and the Adam step with 8-bit moments, against plain 64-bit forms.

Tolerances. A rounding to fp32 is off by at most U = 2^-24 of the value, to bf16 by 2^-8. A sum of n fp32 terms in any order is off by at most (n - 1) U times the sum of their
magnitudes, and what the terms themselves carry. The bounds below count the roundings of each formula on the magnitudes it adds up; they hold element by element."""
import math

import numpy as np
import pytest
import torch

import adam8_ref as A8

pytestmark = pytest.mark.gpu
F32, BF16, F64 = torch.float32, torch.bfloat16, torch.float64
U = 2.0 ** -24
HALF = {F32: U, BF16: 2.0 ** -8}


@pytest.fixture(scope="module")
def ops():
    from med_ts_llm_amd.hip import ops
    return ops


@pytest.fixture(scope="module")
def optim():
    from med_ts_llm_amd.hip import optim
    return optim


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=F32, std=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def within(y, ref, bound, what=""):
    off = (y.double() - ref).abs()
    assert bool((off <= bound).all()), (what, float((off - bound).max()), float((off / bound.clamp(min=1e-300)).max()))


# ================================================================================================ token table: lookup
@pytest.mark.parametrize("N,V,d,tt,ot", [((1,), 1, 1, F32, F32), ((3, 5), 17, 24, F32, BF16), ((133,), 50257, 768, F32, F32), ((2, 7), 100, 33, BF16, F32), ((31,), 9, 4096, BF16, BF16),
                                         ((4, 3), 50, 1000, F32, F32), ((1000,), 64, 16, BF16, BF16), ((70000,), 300, 8, F32, BF16)])
@pytest.mark.parametrize("idt", [torch.int32, torch.int64])
def test_embedding_lookup(ops, N, V, d, tt, ot, idt):
    g = gen(1)
    table = randn(g, V, d, dtype=tt)
    ids = torch.randint(-1, V + 1, N, generator=g, device="cuda").to(idt)
    out = ops.embedding_fwd(ids, table, scale=1.7, out_dtype=ot)
    assert out.shape == (*N, d) and out.dtype == ot
    ok = (ids >= 0) & (ids < V)
    s = float(np.float32(1.7))
    ref = torch.where(ok[..., None], table.double()[ids.long().clamp(0, V - 1)] * s, 0.0)
    within(out, ref, ref.abs() * (U + HALF[ot]) * 1.01)                   # one product, one store
    assert torch.equal(ops.embedding_fwd(ids, table), torch.where(ok[..., None], table[ids.long().clamp(0, V - 1)], 0.0).to(tt))


@pytest.mark.parametrize("N,V,d,tt,ot", [(16387, 500, 1024, BF16, BF16), (16389, 70, 1001, F32, F32), (131077, 300, 520, BF16, BF16), (131075, 40, 261, BF16, F32), (131073, 50, 301, F32, BF16), (9001, 60, 4100, F32, F32)])
def test_embedding_lookup_of_many_tokens(ops, N, V, d, tt, ot):
    test_embedding_lookup(ops, (N,), V, d, tt, ot, torch.int64)


@pytest.mark.parametrize("d,ot", [(8, F32), (264, BF16)])
def test_embedding_lookup_in_several_launches(ops, d, ot):
    """more tokens than one launch takes (8 388 608)"""
    N, V = (1 << 23) + 77, 100
    g = gen(5)
    table = randn(g, V, d, dtype=ot)
    ids = torch.randint(-1, V, (N,), generator=g, device="cuda", dtype=torch.int32)
    out = ops.embedding_fwd(ids, table)
    at, ok = ids.long().clamp(0), ids >= 0
    for i in range(0, N, 1 << 21):
        assert torch.equal(out[i:i + (1 << 21)], table[at[i:i + (1 << 21)]] * ok[i:i + (1 << 21), None])


def test_embedding_lookup_strides_and_empty(ops):
    g = gen(2)
    big = randn(g, 40, 70)
    for table in (big[:, :64], big[:, 1:65], big[::2, 3:20], big[:, 5:6]):
        ids = torch.randint(0, table.shape[0], (6, 4), generator=g, device="cuda").t()        # (not contiguous)
        assert torch.equal(ops.embedding_fwd(ids, table), table[ids])
    assert ops.embedding_fwd(torch.zeros(0, 3, dtype=torch.int64, device="cuda"), big).shape == (0, 3, 70)
    assert ops.embedding_fwd(torch.tensor(7, device="cuda"), big).shape == (70,)
    nan = big.clone()
    nan[3, 5], nan[4, 0] = math.nan, math.inf
    out = ops.embedding_fwd(torch.tensor([3, 4, -1, 40, 2], device="cuda"), nan)
    assert torch.equal(out[:2].isfinite(), nan[3:5].isfinite()) and not out[2:4].any() and torch.equal(out[4], nan[2])


# ================================================================================================ token table: gradient
def embed_ref(dout, ids, V, scale, pad):
    """(gradient, sum of magnitudes, terms per row) in 64 bits"""
    d = dout.shape[-1]
    ids, x = ids.reshape(-1).long(), dout.reshape(-1, d).double()
    ok = (ids >= 0) & (ids < V) & (ids != (-7 if pad is None else pad))
    ref = torch.zeros(V, d, dtype=F64, device="cuda").index_add_(0, ids[ok], x[ok])
    mag = torch.zeros(V, d, dtype=F64, device="cuda").index_add_(0, ids[ok], x[ok].abs())
    n = torch.bincount(ids[ok], minlength=V).double()[:, None]
    s = float(np.float32(scale))
    return ref * s, mag * abs(s), n


EMBED = [  # N, V, d, dout, grad, pad
    (0, 3, 8, F32, F32, None), (1, 1, 1, F32, F32, None), (7, 5, 3, BF16, F32, 2), (8, 100, 64, BF16, BF16, None), (9, 2, 65, F32, F32, 0), (64, 10, 66, F32, BF16, None),
    (1000, 7, 200, BF16, F32, 3), (1025, 513, 128, BF16, BF16, None), (4096, 262143, 20, F32, F32, None), (4097, 511, 96, F32, F32, 5), (5000, 50257, 768, BF16, F32, 11),
    (8192, 1, 512, BF16, F32, None), (8193, 262144, 24, F32, F32, None), (16384, 100, 2048, BF16, BF16, 4), (16385, 300001, 33, BF16, F32, None), (40000, 2, 130, F32, F32, None),
    (1100000, 5000, 4, F32, F32, 7), (50001, 32000, 256, BF16, BF16, 31999), (300000, 70000, 40, BF16, F32, 1), (200003, 3, 520, BF16, F32, None)]


@pytest.mark.parametrize("N,V,d,dt,gt,pad", EMBED)
def test_embedding_gradient(ops, N, V, d, dt, gt, pad):
    g = gen(N + V)
    ids = torch.randint(0, V + 1, (N,), generator=g, device="cuda") - (torch.rand(N, generator=g, device="cuda") < 0.02).long()      # some -1, some V
    ids = torch.where(torch.rand(N, generator=g, device="cuda") < 0.3, V // 2, ids)                                                  # one long run
    dout = randn(g, N, d, dtype=dt)
    grad = ops.embedding_bwd(dout, ids, V, scale=0.37, padding_idx=pad, out_dtype=gt)
    ref, mag, n = embed_ref(dout, ids, V, 0.37, pad)
    bound = (n + 2) * U * mag + HALF[gt] * (ref.abs() + (n + 2) * U * mag)
    within(grad, ref, bound)
    assert not grad[(n == 0)[:, 0]].any()
    # the same bits again, with int32 ids, and through a grid that runs in another order (a second stream)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        again = ops.embedding_bwd(dout, ids.int(), V, scale=0.37, padding_idx=pad, out_dtype=gt)
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(grad, again)
    # accumulate: only the rows that occur change
    base = randn(g, V, d, dtype=gt)
    acc = ops.embedding_bwd(dout, ids, V, scale=0.37, padding_idx=pad, out=base.clone(), accumulate=True)
    within(acc, ref + base.double(), (n + 3) * U * (mag + base.double().abs()) + HALF[gt] * ((ref + base.double()).abs() + (n + 3) * U * mag) * (n > 0))
    assert torch.equal(acc[(n == 0)[:, 0]], base[(n == 0)[:, 0]])


def test_embedding_gradient_layouts(ops):
    """row-strided and unaligned dout and out; what lies between out's rows and behind them stays; the expanded gradient of a sum"""
    g = gen(5)
    ids = torch.randint(0, 50, (3, 41), generator=g, device="cuda")
    wide = randn(g, 3, 41, 80)
    for lo, hi in ((0, 64), (1, 65), (2, 12), (7, 8)):
        dout = wide[..., lo:hi]
        ref, mag, n = embed_ref(dout, ids, 50, 1.0, None)
        buf = torch.full((52, 80), 9.0, device="cuda")
        ops.embedding_bwd(dout, ids, 50, out=buf[:50, lo:hi])
        within(buf[:50, lo:hi], ref, (n + 2) * U * mag + U * ref.abs())
        buf[:50, lo:hi] = 9.0
        assert bool((buf == 9.0).all())
    for lo, hi in ((0, 33), (1, 34), (3, 80)):                    # bf16 rows 162 bytes apart: 2-byte aligned
        x16 = randn(g, 3, 41, hi - lo, dtype=BF16)
        ref, mag, n = embed_ref(x16, ids, 50, 0.5, 3)
        buf = torch.full((51, 81), 9.0, dtype=BF16, device="cuda")
        ops.embedding_bwd(x16, ids, 50, scale=0.5, padding_idx=3, out=buf[:50, lo:hi])
        within(buf[:50, lo:hi], ref, (n + 2) * U * mag + HALF[BF16] * (ref.abs() + (n + 2) * U * mag))
        old = buf[:50, lo:hi].clone()
        ops.embedding_bwd(x16, ids, 50, scale=0.5, padding_idx=3, out=buf[:50, lo:hi], accumulate=True)
        twice = old.double() + ref
        within(buf[:50, lo:hi], twice, (n + 3) * U * (mag + old.double().abs()) + HALF[BF16] * (twice.abs() + (n + 3) * U * (mag + old.double().abs())))
        buf[:50, lo:hi] = 9.0
        assert bool((buf == 9.0).all())
    table = randn(g, 50, 16).requires_grad_()
    ops.EmbeddingFn.apply(ids, table, 2.0).sum().backward()
    assert torch.equal(table.grad, 2.0 * torch.bincount(ids.reshape(-1), minlength=50).float()[:, None].expand(50, 16))
    masked = randn(g, 3, 41, 16)
    masked[0, 5] = math.nan                                       # a NaN in a token without a gradient stays out; in one with a gradient it reaches its row only
    ids2 = ids.clone()
    ids2[0, 5] = -1
    assert bool(ops.embedding_bwd(masked, ids2, 50).isfinite().all())
    got = ops.embedding_bwd(masked, ids, 50).isfinite().all(1)
    assert not got[ids[0, 5]] and int((~got).sum()) == 1


@pytest.mark.parametrize("N", [1, 5000, 20000])
def test_embedding_without_a_token_that_counts(ops, N):
    """every token is padding or outside the table: zeros, or what was there with accumulate"""
    g = gen(N)
    ids = torch.where(torch.rand(N, generator=g, device="cuda") < 0.5, 7, -1)
    x = randn(g, N, 33)
    assert not ops.embedding_bwd(x, ids, 20, padding_idx=7).any()
    base = randn(g, 20, 33)
    assert torch.equal(ops.embedding_bwd(x, ids, 20, padding_idx=7, out=base.clone(), accumulate=True), base)


def test_calls_on_two_streams_at_once(ops):
    """gradients of two streams in flight together, each with its own workspace"""
    g = gen(21)
    cos, sin = turn_tables(512, 64)
    w = 1 + randn(g, 64, std=0.1)
    data = [(torch.randint(0, 400, (20000,), generator=g, device="cuda"), randn(g, 20000, 96), randn(g, 2, 512, 512), randn(g, 2, 512, 128), randn(g, 2, 512, 512), randn(g, 2, 512, 128)) for _ in range(2)]

    def work(ids, x, q, k, dq, dk):
        return [ops.embedding_bwd(x, ids, 400), ops.embedding_bwd(x[:3000], ids[:3000], 400), *ops.qk_norm_rope_bwd(dq, dk, q, k, w, w, cos, sin, 8, 2, 64)]

    want = [work(*d) for d in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in data]
    for _ in range(3):
        got = []
        for st, d in zip(streams, data):
            with torch.cuda.stream(st):
                got.append(work(*d))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for x, y in zip(got, want) for a, b in zip(x, y))


@pytest.mark.parametrize("N", [0, 1, 100, 9000])
@pytest.mark.parametrize("V,d,gt", [(137003, 1001, BF16), (66001, 1024, F32)])
def test_embedding_gradient_larger_than_the_cache(ops, N, V, d, gt):
    """256 MiB and more of rows, an odd end among them, written over other values: every row without a token is zero, the others hold the sum"""
    assert V * d * gt.itemsize >= 256 << 20
    g = gen(N + V)
    ids = torch.randint(0, V, (N,), generator=g, device="cuda")
    if N > 1:
        ids[0], ids[-1] = V - 1, 0
    dout = randn(g, N, d, dtype=gt)
    store = torch.ones(V * d + 64, dtype=gt, device="cuda")
    grad = ops.embedding_bwd(dout, ids, V, out=store[:V * d].view(V, d))
    n = torch.bincount(ids, minlength=V)
    at = n.nonzero()[:, 0]
    row = torch.zeros(V, dtype=torch.int64, device="cuda").index_put_((at,), torch.arange(len(at), device="cuda"))[ids]
    ref, mag = (torch.zeros(len(at), d, dtype=F64, device="cuda").index_add_(0, row, x) for x in (dout.double(), dout.double().abs()))
    bound = (n[at][:, None] + 1) * U * mag
    within(grad[at], ref, bound + HALF[gt] * (ref.abs() + bound))
    assert int(torch.count_nonzero(grad[n == 0])) == 0 and bool((store[V * d:] == 1).all())


def test_embedding_offsets_beyond_32_bits(ops):
    """table, output and gradient of more than 2^31 elements (4.6 GB each in bf16): rows at both ends, looked up, summed and zeroed"""
    V, d, N = 140000, 16384, 140001
    g = gen(13)
    table = torch.zeros(V, d, dtype=BF16, device="cuda")
    table[-3:] = randn(g, 3, d, dtype=BF16)
    ids = torch.randint(V // 2, V - 10, (N,), generator=g, device="cuda")
    ids[-1], ids[0], ids[N // 2] = V - 1, V - 2, V - 1
    out = ops.embedding_fwd(ids, table)
    assert torch.equal(out[-1], table[-1]) and torch.equal(out[0], table[-2]) and torch.equal(out[N // 2], table[-1]) and not out[1:1000].any()
    out.fill_(1.0)
    out[-1] = randn(g, d, dtype=BF16)
    want = (out[-1].double() + 1.0)
    grad = ops.embedding_bwd(out, ids, V, out_dtype=BF16, out=table)
    within(grad[-1], want, 3 * U * (want.abs() + 1) + HALF[BF16] * (want.abs() + 3 * U))
    assert bool((grad[-2] == 1).all()) and not grad[:V // 2].any() and not grad[-10:-2].any()
    n = torch.bincount(ids, minlength=V).double()
    assert torch.equal(grad[V // 2:V - 2, -1].double(), n[V // 2:V - 2].to(BF16).double())


def test_embedding_refuses_shared_memory(ops):
    x = torch.zeros(64, 8, device="cuda")
    with pytest.raises(ValueError):
        ops.embedding_bwd(x[:10], torch.zeros(10, dtype=torch.int64, device="cuda"), 20, out=x[5:25])
    assert ops.embedding_bwd(x[:10], torch.zeros(10, dtype=torch.int64, device="cuda"), 20, out=x[10:30]).shape == (20, 8)


def test_embedding_function_against_differences(ops):
    """the lookup is linear in the table: <dout, f(table + h v) - f(table)> / h = <grad, v> up to the roundings of f's outputs"""
    g = gen(6)
    ids = torch.randint(0, 30, (4, 9), generator=g, device="cuda")
    table = randn(g, 30, 12).requires_grad_()
    c, v, h = randn(g, 4, 9, 12), randn(g, 30, 12), 0.25
    out = ops.EmbeddingFn.apply(ids, table, 3.0, 7)
    (grad,) = torch.autograd.grad(out, table, c)
    assert not grad[7].any()
    keep = (ids != 7)[..., None]
    moved = ops.embedding_fwd(ids, (table.detach() + h * v), scale=3.0)
    num = (((moved.double() - out.detach().double()) * c.double() * keep).sum() / h).item()
    size = (moved.abs().double() * c.abs().double()).sum().item()
    assert abs(num - (grad.double() * v.double()).sum().item()) <= 8 * U * size / h


# ================================================================================================ query / key norm + rotation
def turn_tables(P, R):
    inv = 10000.0 ** (-torch.arange(0, R, 2, device="cuda", dtype=F64) / R)
    a = torch.arange(P, device="cuda", dtype=F64)[:, None] * inv
    a = torch.cat([a, a], 1)
    return a.cos().float(), a.sin().float()


def rot(x, c, s, R, inverse=False):
    a, b, rest = x[..., :R // 2], x[..., R // 2:R], x[..., R:]
    c, s = c[..., :R // 2], s[..., :R // 2]
    return torch.cat([a * c + b * s, b * c - a * s, rest], -1) if inverse else torch.cat([a * c - b * s, b * c + a * s, rest], -1)


def rot_abs(x, c, s, R):
    return rot(x.abs(), c.abs(), -s.abs(), R, False).abs().maximum(rot(x.abs(), c.abs(), s.abs(), R, False).abs())      # |a||c| + |b||s| in both halves


def qk_ref(x, w, c, s, R, eps, dy=None):
    """y and its bound's magnitudes; with dy: dx, dw and theirs. x [B, T, H, D] in 64 bits"""
    D = x.shape[-1]
    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    n = x * r
    if dy is None:
        return rot(n * w, c, s, R), rot_abs(n * w, c, s, R)
    u, ua = rot(dy, c, s, R, True), rot_abs(dy, c, s, R)
    dx = r * (u * w - n * (u * w * n).mean(-1, keepdim=True))
    dxa = r * (ua * w.abs() + n.abs() * (ua * w.abs() * n.abs()).mean(-1, keepdim=True))
    return dx, dxa, (u * n).sum((0, 1, 2)), (ua * n.abs()).sum((0, 1, 2))


QK = [  # B, T, Hq, Hkv, D, R, type, weights, positions
    (1, 1, 1, 1, 2, 2, F32, F32, None), (2, 3, 3, 1, 6, 4, F32, F32, "i64"), (1, 1, 32, 8, 128, 128, BF16, F32, "i32"), (4, 1, 12, 12, 64, 64, BF16, BF16, "i64"), (2, 17, 12, 4, 64, 32, BF16, F32, "pos0"),
    (3, 5, 5, 3, 80, 32, F32, F32, "row"), (2, 9, 7, 2, 96, 96, BF16, F32, None), (1, 33, 4, 4, 130, 64, F32, F32, "i64"), (1, 5, 3, 1, 256, 256, BF16, BF16, None), (2, 4, 2, 2, 512, 256, F32, F32, "i64"),
    (1, 3, 3, 2, 510, 2, BF16, F32, None), (3, 700, 32, 8, 128, 128, BF16, F32, None), (1, 2049, 9, 9, 32, 32, F32, F32, "i32"), (2, 3, 70, 1, 16, 16, F32, F32, None), (1, 4, 2, 2, 384, 384, BF16, F32, None),
    (2, 1030, 2, 1, 66, 20, BF16, F32, "i64"), (2, 5, 3, 3, 100, 100, BF16, F32, "i64"), (1, 7, 2, 1, 156, 34, F32, F32, None), (3, 40, 6, 2, 250, 250, BF16, BF16, None), (1, 9, 2, 2, 510, 254, F32, F32, "i32"),
    (2, 11, 5, 1, 18, 18, BF16, F32, None), (1, 130, 9, 3, 192, 64, BF16, F32, "pos0")]


@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("B,T,Hq,Hkv,D,R,dt,wt,pos", QK)
def test_qk_norm_rope(ops, B, T, Hq, Hkv, D, R, dt, wt, pos, fused):
    """forward, in place, backward (fused: strided views of one buffer, and gradients written into column ranges of one)"""
    g = gen(D + T)
    P, eps = T + 40, 1e-5
    cos, sin = turn_tables(P, R)
    W = (Hq + 2 * Hkv) * D
    if fused:
        qkv = randn(g, B, T, W, dtype=dt)
        q, k = qkv[..., :Hq * D], qkv[..., Hq * D:(Hq + Hkv) * D]
    else:
        q, k = randn(g, B, T, Hq * D, dtype=dt), randn(g, T, B, Hkv * D, dtype=dt).transpose(0, 1)
    q[0, 0] *= 1e-3                                                          # (a row whose mean square is near eps)
    k[-1, -1] = 0                                                            # and an empty one
    wq, wk = (1 + randn(g, D, std=0.3)).to(wt), (1 + randn(g, D, std=0.3)).to(wt)
    kw, at = {}, torch.arange(T, device="cuda").expand(B, T)
    if pos == "pos0":
        kw, at = {"pos0": 40}, at + 40
    elif pos == "row":
        at = torch.randint(0, P, (T,), generator=g, device="cuda")
        kw, at = {"positions": at}, at.expand(B, T)
    elif pos:
        at = torch.randint(0, P, (B, T), generator=g, device="cuda")
        kw = {"positions": at.to(torch.int32 if pos == "i32" else torch.int64)}
    c, s = cos.double()[at][:, :, None], sin.double()[at][:, :, None]
    args = (wq, wk, cos, sin, Hq, Hkv, D, eps)
    yq, yk = ops.qk_norm_rope_fwd(q, k, *args, **kw)
    dyq, dyk = randn(g, B, T, Hq * D, dtype=dt), randn(g, B, T, Hkv * D, dtype=dt)
    out = None
    if fused:
        dqkv = torch.full((B, T, W), 5.0, dtype=dt, device="cuda")
        out = (dqkv[..., :Hq * D], dqkv[..., Hq * D:(Hq + Hkv) * D])
    dq, dk, dwq, dwk = ops.qk_norm_rope_bwd(dyq, dyk, q, k, *args, **kw, out=out)
    # forward: D squares and their sum, mean, eps, root, quotient (D / 2 + 5 on r, which sees half of the sum's error), n, n w, two products and their sum
    Cf, Cb = D / 2 + 10, D + 24
    for y, x, w, dy, dx, dw, H in ((yq, q, wq, dyq, dq, dwq, Hq), (yk, k, wk, dyk, dk, dwk, Hkv)):
        x4, d4 = x.double().unflatten(-1, (H, D)), dy.double().unflatten(-1, (H, D))
        ref, mag = qk_ref(x4, w.double(), c, s, R, eps)
        within(y.unflatten(-1, (H, D)), ref, Cf * U * mag * 1.01 + HALF[dt] * (ref.abs() + Cf * U * mag), "y")
        rdx, mdx, rdw, mdw = qk_ref(x4, w.double(), c, s, R, eps, d4)
        within(dx.unflatten(-1, (H, D)), rdx, Cb * U * mdx * 1.01 + HALF[dt] * (rdx.abs() + Cb * U * mdx), "dx")
        within(dw, rdw, (B * T * H + D + 24) * U * mdw, "dw")
    again = ops.qk_norm_rope_bwd(dyq, dyk, q, k, *args, **kw)
    assert all(torch.equal(a, b) for a, b in zip(again, (dq, dk, dwq, dwk)))
    only = ops.qk_norm_rope_bwd(dyq, dyk, q, k, *args, **kw, want_dw=False)
    assert torch.equal(only[0], dq) and torch.equal(only[1], dk) and only[2] is None
    if fused:
        assert bool((dqkv[..., (Hq + Hkv) * D:] == 5.0).all())
        v = qkv[..., (Hq + Hkv) * D:].clone()
        a, b = ops.qk_norm_rope_fwd(q, k, *args, **kw, out=(q, k))           # in place: same bits, values untouched
        assert a.data_ptr() == q.data_ptr() and torch.equal(q, yq) and torch.equal(k, yk) and torch.equal(qkv[..., (Hq + Hkv) * D:], v)
        assert b.data_ptr() == k.data_ptr()


@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("B,T,Hq,Hkv,D,R,pos", [(3, 2785, 32, 8, 128, 128, "i64"), (1, 3001, 24, 24, 256, 256, None), (1, 9001, 3, 5, 512, 256, "pos0")])
def test_qk_norm_rope_larger_than_the_cache(ops, B, T, Hq, Hkv, D, R, pos, fused):
    """64 MiB and more of queries and keys, whose loads pass the cache by: heads in 8, 16 and 32 lanes, in place among them"""
    assert B * T * (Hq + Hkv) * D * 2 >= 64 << 20
    test_qk_norm_rope(ops, B, T, Hq, Hkv, D, R, BF16, F32, pos, fused)


def test_qk_norm_rope_positions_outside_the_table_and_masked_values(ops):
    """a row whose position is not in the table is NaN, and only that row; a NaN or an infinity in a head stays in that head; empty batches"""
    g = gen(9)
    cos, sin = turn_tables(8, 32)
    q, k, w = randn(g, 2, 3, 4 * 32), randn(g, 2, 3, 2 * 32), torch.ones(32, device="cuda")
    at = torch.tensor([[0, -1, 7], [8, 3, 1 << 40]], device="cuda")
    yq, yk = ops.qk_norm_rope_fwd(q, k, w, w, cos, sin, 4, 2, 32, positions=at)
    bad = (at < 0) | (at >= 8)
    assert torch.equal(yq.isnan().all(-1), bad) and torch.equal(yq.isnan().any(-1), bad) and torch.equal(yk.isnan().any(-1), bad)
    dq, dk, _, _ = ops.qk_norm_rope_bwd(q, k, q, k, w, w, cos, sin, 4, 2, 32, positions=at, want_dw=False)
    assert torch.equal(dq.isnan().all(-1), bad) and torch.equal(dk.isnan().any(-1), bad)
    q[0, 0, 40], q[1, 1, 5] = math.nan, math.inf
    yq, _ = ops.qk_norm_rope_fwd(q, k, w, w, cos, sin, 4, 2, 32)
    broken = (~yq.unflatten(-1, (4, 32)).isfinite()).any(-1).nonzero().tolist()
    assert broken == [[0, 0, 1], [1, 1, 0]]
    e = ops.qk_norm_rope_bwd(q[:0], k[:0], q[:0], k[:0], w, w, cos, sin, 4, 2, 32)
    assert e[0].shape == (0, 3, 128) and not e[2].any() and not e[3].any()
    assert ops.qk_norm_rope_fwd(q[:, :0], k[:, :0], w, w, cos, sin, 4, 2, 32)[0].shape == (2, 0, 128)


def test_qk_norm_rope_into_a_cache(ops):
    """one token of every sequence at its own position: the keys go straight to their places in a cache, the rest of which stays as it is"""
    g = gen(41)
    B, Hq, Hkv, D, L = 5, 8, 2, 64, 37
    cos, sin = turn_tables(L, D)
    wq, wk = 1 + randn(g, D, std=0.1), 1 + randn(g, D, std=0.1)
    q, k = randn(g, B, 1, Hq * D, dtype=BF16), randn(g, B, 1, Hkv * D, dtype=BF16)
    cache = torch.full((B, L, 2, Hkv * D), 3.0, dtype=BF16, device="cuda")
    yq, yk = ops.qk_norm_rope_fwd(q, k, wq, wk, cos, sin, Hq, Hkv, D, pos0=11)
    oq = torch.empty_like(q)
    ops.qk_norm_rope_fwd(q, k, wq, wk, cos, sin, Hq, Hkv, D, pos0=11, out=(oq, cache[:, 11:12, 0]))
    assert torch.equal(oq, yq) and torch.equal(cache[:, 11:12, 0], yk)
    cache[:, 11:12, 0] = 3.0
    assert bool((cache == 3.0).all())


def test_qk_norm_rope_function_against_differences(ops):
    """directional derivative by central differences: f is smooth with derivatives of order 1 at these inputs; h = 2^-6 leaves a cubic term below h^2 times the magnitudes (2.5e-4) and
    roundings of 2 U / h (8e-6)"""
    g = gen(10)
    cos, sin = turn_tables(20, 16)
    x = [randn(g, 2, 5, 3 * 24), randn(g, 2, 5, 1 * 24), 1 + randn(g, 24, std=0.2), 1 + randn(g, 24, std=0.2)]
    c = [randn(g, 2, 5, 72), randn(g, 2, 5, 24)]
    v = [randn(g, *t.shape, std=0.5) for t in x]
    leaves = [t.clone().requires_grad_() for t in x]
    y = ops.QkNormRopeFn.apply(*leaves, cos, sin, 3, 1, 24, 1e-6)
    grads = torch.autograd.grad(y, leaves, c)
    f = lambda t: sum((a.double() * b.double()).sum().item() for a, b in zip(ops.qk_norm_rope_fwd(*t, cos, sin, 3, 1, 24), c))      # noqa: E731
    h = 2.0 ** -6
    num = (f([a + h * b for a, b in zip(x, v)]) - f([a - h * b for a, b in zip(x, v)])) / (2 * h)
    ana = sum((a.double() * b.double()).sum().item() for a, b in zip(grads, v))
    size = sum((a.double() * b.double()).abs().sum().item() for a, b in zip(grads, v))
    assert abs(num - ana) <= 2 * h * h * size, (num, ana, size)
    partial = torch.autograd.grad(ops.QkNormRopeFn.apply(*leaves, cos, sin, 3, 1, 24)[0], leaves[2], c[0])       # one output only, one input only
    assert torch.equal(partial[0], grads[2])


def test_second_derivatives_are_refused(ops):
    """the gradients are not differentiable again: under create_graph the first ones come out, a second pass through them raises"""
    g = gen(22)
    cos, sin = turn_tables(4, 8)
    table, w = randn(g, 6, 8).requires_grad_(), torch.ones(8, device="cuda", requires_grad=True)
    q = randn(g, 1, 4, 8).requires_grad_()
    for y, leaf in ((ops.EmbeddingFn.apply(torch.arange(4, device="cuda"), table), table), (ops.QkNormRopeFn.apply(q, q, w, w, cos, sin, 1, 1, 8)[0], q)):
        (first,) = torch.autograd.grad((y * y).sum(), leaf, create_graph=True)
        assert first.shape == leaf.shape
        with pytest.raises(RuntimeError):
            torch.autograd.grad(first.sum(), leaf)


def test_saved_tensor_hooks(ops):
    """activations that a hook moves between forward and backward (here: cloned) give the same gradients"""
    g = gen(23)
    cos, sin = turn_tables(5, 16)
    leaves = [randn(g, 2, 5, 64).requires_grad_(), randn(g, 2, 5, 32).requires_grad_(), (1 + randn(g, 16)).requires_grad_(), (1 + randn(g, 16)).requires_grad_()]
    c = (randn(g, 2, 5, 64), randn(g, 2, 5, 32))
    want = torch.autograd.grad(ops.QkNormRopeFn.apply(*leaves, cos, sin, 4, 2, 16), leaves, c)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), lambda t: t.clone()):
        y = ops.QkNormRopeFn.apply(*leaves, cos, sin, 4, 2, 16)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves, c), want))


# ================================================================================================ 8-bit Adam
def np_of(t):
    return t.detach().float().cpu().numpy().reshape(-1)


def codes_of(st):
    return st.exp_avg.cpu().numpy().reshape(-1), st.exp_avg_sq.cpu().numpy().reshape(-1), st.exponents.cpu().numpy().view(np.int8)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("wd,decoupled", [(0.0, False), (0.01, False), (0.01, True)])
def test_adam8_step_bit_for_bit(optim, dt, wd, decoupled):
    """parameters, codes and exponents equal the numpy restatement's bits over six steps: odd sizes, unaligned views, gradients of every magnitude, zeros, NaN and infinities"""
    g = gen(3)
    sizes = [1, 3, 63, 64, 65, 1000, 4096, 4097, 70001]
    base = [randn(g, n + 1, dtype=dt, std=0.1) for n in sizes]
    ps = [b[1:] if i % 2 else b[:-1] for i, b in enumerate(base)]                  # every other one starts off a 16-byte border
    edge = [(b[:1] if i % 2 else b[-1:]).clone() for i, b in enumerate(base)]       # the element beside each parameter
    sts = [optim.adam8_state(p) for p in ps]
    want = [(np_of(p), codes_of(st)) for p, st in zip(ps, sts)]
    for t in range(1, 7):
        gs = [(randn(g, p.numel()) * torch.exp(3 * randn(g, p.numel()))).to(dt) * 10.0 ** (t - 4) for p in ps]
        if t == 1:
            gs[5][100:300] = 0
        if t == 4:
            gs[5][10], gs[5][11], gs[6][64] = math.nan, math.inf, -math.inf
        optim.adam8_step(ps, gs, sts, t, lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=wd, decoupled_weight_decay=decoupled)
        for i, (p, gr, st) in enumerate(zip(ps, gs, sts)):
            wp, wc = A8.step(want[i][0], np_of(gr), want[i][1], t, 1e-2, 0.9, 0.999, 1e-8, wd, decoupled)
            if dt == BF16:
                wp = torch.from_numpy(wp).to(BF16).float().numpy()
            want[i] = (wp, wc)
            got = codes_of(st)
            assert np.array_equal(np_of(p), wp, equal_nan=True), (t, sizes[i])
            for a, b, what in zip(got, wc, "mre"):
                assert np.array_equal(a, b), (t, sizes[i], what, np.flatnonzero(a != b)[:5])
    assert all(torch.equal(b[:1] if i % 2 else b[-1:], e) for i, (b, e) in enumerate(zip(base, edge)))


def test_adam8_moments_and_quantize(optim):
    g = gen(4)
    shapes = [(5, 77), (3,), (64, 64), (0,), (70001,)]
    ms = [randn(g, *s) * 1e-3 for s in shapes]
    vs = [(randn(g, *s) * 1e-3) ** 2 for s in shapes]
    sts = [optim.adam8_quantize(m, v, 9) for m, v in zip(ms, vs)]
    for m, v, st, (a, b), (a16, b16) in zip(ms, vs, sts, optim.adam8_moments(sts), optim.adam8_moments(sts, BF16)):
        if not m.numel():
            continue
        want = A8.encode(np_of(m), np.sqrt(np_of(v)), 9)
        assert all(np.array_equal(x, y) for x, y in zip(codes_of(st), want))
        dm, dr = A8.decode(*want)
        assert np.array_equal(np_of(a), dm) and np.array_equal(np_of(b), dr * dr) and a.shape == m.shape
        assert torch.equal(a16.float(), a) and torch.equal(b16, b.to(BF16))


def test_adam8_moments_larger_than_the_cache(optim):
    """192 MiB and more written by one call, ends that fill no vector: the values that the codes stand for, from packed moments that start on and off a 16-byte boundary"""
    g = gen(8)
    ns = (50_000_003, 1, 700_002)
    sts = []
    for n, off in zip(ns, (1, 0, 0)):
        m, v = randn(g, n + off) * 1e-3, randn(g, n + off).square() * 1e-6
        sts.append(optim.adam8_quantize(m[off:], v[off:], 7))
        if off:
            again = optim.adam8_quantize(m[off:].clone(), v[off:].clone(), 7)
            assert all(torch.equal(getattr(again, k), getattr(sts[0], k)) for k in ("exp_avg", "exp_avg_sq", "exponents"))
            del again
        del m, v
    e4m3, root = (torch.from_numpy(x).cuda() for x in (A8.E4M3, A8.ROOT))
    for dt in (F32, BF16):
        for n, st, (a, b) in zip(ns, sts, optim.adam8_moments(sts, dt)):
            ex = torch.exp2(st.exponents.view(torch.int8).view(-1, 2).float()).repeat_interleave(64, 0)[:n]
            r = root[st.exp_avg_sq.view(-1).int()] * ex[:, 1]
            assert torch.equal(a.float(), e4m3[st.exp_avg.view(-1).int()] * ex[:, 0]) and torch.equal(b, (r * r).to(dt))


def _run(opt_args, steps, seed, ps, opt=None):
    from med_ts_llm_amd.hip.optim import HipAdam
    opt = HipAdam(ps, **opt_args) if opt is None else opt
    for t in range(steps):
        g = gen(seed + t)
        for p in ps:
            p.grad = randn(g, *p.shape, dtype=p.dtype, std=1e-2)
        opt.step()
    return opt


def test_hip_adam_with_8_bit_state(optim):
    """HipAdam(state_bits=8): equals adam8_step; more tensors than one launch holds, empty ones among them; shadows; a state dict taken and continued gives the same bits"""
    g = gen(7)
    shapes = [(37, 101), (0,), (5,)] + [(9, 3)] * 60
    ps = [randn(g, *s).requires_grad_() for s in shapes]
    ref, sts = [p.detach().clone() for p in ps], [optim.adam8_state(p) for p in ps]
    from med_ts_llm_amd.hip.optim import Bf16Shadow, HipAdam
    opt = HipAdam(ps, lr=1e-2, weight_decay=0.01, decoupled_weight_decay=True, state_bits=8)
    sh = Bf16Shadow(ps[0], torch.zeros(37, 128, dtype=BF16, device="cuda"))
    opt.register_shadow(sh)
    v0 = ps[0]._version
    _run(None, 3, 50, ps, opt)
    for t in range(3):
        gg = gen(50 + t)
        optim.adam8_step(ref, [randn(gg, *p.shape, std=1e-2) for p in ref], sts, t + 1, lr=1e-2, weight_decay=0.01, decoupled_weight_decay=True, first_moment="threshold")
    assert all(torch.equal(a, b) for a, b in zip(ps, ref)) and ps[0]._version > v0 and sh.fresh()
    assert torch.equal(sh.tensor[:, :101], ps[0].detach().to(BF16)) and not sh.tensor[:, 101:].any()
    sd = opt.state_dict()
    assert set(sd["state"][0]) == {"step", "exp_avg_q", "exp_avg_sq_q", "q_exp"} and sd["state"][0]["exp_avg_q"].shape == (37, 101)
    qs = [p.detach().clone().requires_grad_() for p in ps]
    two = HipAdam(qs, lr=1e-2, weight_decay=0.01, decoupled_weight_decay=True, state_bits=8)
    two.load_state_dict(sd)
    _run(None, 2, 90, ps, opt), _run(None, 2, 90, qs, two)
    assert all(torch.equal(a, b) for a, b in zip(ps, qs))


def test_hip_adam_changes_width_on_load(optim):
    """a 32-bit checkpoint continues in 8 bits and back; moments() reads either"""
    from med_ts_llm_amd.hip.optim import HipAdam
    g = gen(8)
    a = [randn(g, 33, 70).requires_grad_(), randn(g, 7).to(BF16).requires_grad_()]
    wide = _run({"lr": 1e-2}, 3, 10, a)
    b = [p.detach().clone().requires_grad_() for p in a]
    narrow = HipAdam(b, lr=1e-2, state_bits=8)
    narrow.load_state_dict(wide.state_dict())
    want = [optim.adam8_quantize(wide.state[p]["exp_avg"], wide.state[p]["exp_avg_sq"], 3) for p in a]
    _run(None, 1, 20, b, narrow)
    ref = [p.detach().clone() for p in a]
    gg = gen(20)
    optim.adam8_step(ref, [randn(gg, *p.shape, dtype=p.dtype, std=1e-2) for p in ref], want, 4, lr=1e-2)
    assert all(torch.equal(x, y) for x, y in zip(b, ref))
    held = narrow.moments()
    c = [p.detach().clone().requires_grad_() for p in b]
    back = HipAdam(c, lr=1e-2)
    back.load_state_dict(narrow.state_dict())
    _run(None, 1, 30, c, back)
    assert set(back.state[c[0]]) == {"step", "exp_avg", "exp_avg_sq"} and back.state[c[0]]["step"] == 5 and back.state[c[1]]["exp_avg"].dtype == F32
    # (first moment after one more step: 0.9 of what was held plus 0.1 of the gradient; one product, one difference, one sum)
    gg = gen(30)
    for p, q in zip(b, c):
        gr = randn(gg, *p.shape, dtype=p.dtype, std=1e-2).double()
        m = held[p][0].double()
        within(back.moments()[q][0], m + (gr - m) * 0.1, 1e-6 * (m.abs() + gr.abs()))


def test_hip_adam_with_8_bit_state_on_a_side_stream(optim):
    """HipAdam.defer with 8-bit state: the deferred parameters' updates run on the side stream and are the same bits"""
    from med_ts_llm_amd.hip.optim import HipAdam
    g = gen(31)
    a = [randn(g, 300, 500).requires_grad_(), randn(g, 70, 11).requires_grad_()]
    b = [p.detach().clone().requires_grad_() for p in a]
    late = HipAdam(b, lr=1e-2, state_bits=8)
    late.defer(b[:1])
    _run({"lr": 1e-2, "state_bits": 8}, 4, 60, a)
    for t in range(4):
        _run(None, 1, 60 + t, b, late)
        late.wait_deferred()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_adam8_refuses_capture_and_large_tensor_indexing(optim):
    """a captured HipAdam step is refused; in a tensor of more than 2^31 elements the ones behind 2^31 get their own thresholds and codes (checked on the last blocks)"""
    from med_ts_llm_amd.hip import _native as N
    from med_ts_llm_amd.hip.optim import HipAdam
    p = torch.zeros(64, device="cuda", requires_grad=True)
    opt = HipAdam([p], state_bits=8)
    p.grad = torch.ones_like(p)
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(N.MtlError):
            opt.step()
        q = p.detach() * 2                                     # (a graph with something in it)
    graph.replay()
    n = (1 << 31) + 4097
    big = torch.zeros(n, dtype=BF16, device="cuda")
    gr = torch.full((n,), 1e-3, dtype=BF16, device="cuda")
    tail = randn(gen(1), 4097 + 64, dtype=BF16, std=1e-3)
    gr[-tail.numel():] = tail
    st = optim.adam8_state(big)
    optim.adam8_step([big], [gr], [st], 1, lr=1e-2)
    k = tail.numel() // 64 * 64                                # whole blocks at the end (n - 1 is a multiple of 64)
    lo = (n - 1) // 64 * 64 - k
    u0 = A8.thresholds
    try:
        A8.thresholds = lambda cnt, step: ((np.arange(lo, lo + cnt, dtype=np.uint64) * np.uint64(0xC13FA9A9) + np.uint64((step * 0x91E10DA5) & 0xFFFFFFFF)) & np.uint64(0xFFFFFFFF)).astype(np.uint32)
        zero = (np.zeros(k + 1, np.uint8), np.zeros(k + 1, np.uint8), np.zeros(((k + 64) // 64, 2), np.int8))
        wp, wc = A8.step(np.zeros(k + 1, np.float32), np_of(gr[lo:]), zero, 1, 1e-2, 0.9, 0.999, 1e-8)
    finally:
        A8.thresholds = u0
    assert gr[lo:].numel() == k + 1
    assert np.array_equal(np_of(big[lo:]), torch.from_numpy(wp).to(BF16).float().numpy())
    assert np.array_equal(st.exp_avg[lo:].cpu().numpy(), wc[0]) and np.array_equal(st.exp_avg_sq[lo:].cpu().numpy(), wc[1])
    assert np.array_equal(st.exponents[lo // 64:].cpu().numpy().view(np.int8), wc[2])


def test_adam8_step_captured(optim):
    """the raw step in a graph repeats the step number it was captured with, on what the tensors hold at the replay"""
    g = gen(51)
    p, gr = randn(g, 5000), randn(g, 5000, std=1e-2)
    st = optim.adam8_state(p)
    ref, rst = p.clone(), optim.adam8_state(p)
    optim.adam8_step([p.clone()], [gr], [optim.adam8_state(p)], 7, lr=1e-2)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        optim.adam8_step([p], [gr], [st], 7, lr=1e-2)
    for i in range(4):
        gr.copy_(randn(g, 5000, std=1e-2))
        graph.replay()
        optim.adam8_step([ref], [gr], [rst], 7, lr=1e-2)
        torch.cuda.synchronize()
        assert torch.equal(p, ref) and all(torch.equal(a, b) for a, b in zip(st, rst)), i


# ================================================================================================ together
def test_graph_replays_equal_eager(ops):
    """lookup, gradient, norm + rotation and its backward captured once and replayed on changing inputs, with eager work in between"""
    g = gen(11)
    V, d, H, D = 300, 128, 4, 32
    ids = torch.randint(0, V, (2, 40), generator=g, device="cuda")
    table, w = randn(g, V, d), 1 + randn(g, D, std=0.1)
    cos, sin = turn_tables(64, D)
    many = torch.randint(0, V, (20000,), generator=g, device="cuda")
    dmany = randn(g, 20000, 16)

    def work():
        x = ops.embedding_fwd(ids, table, 2.0)
        q, k = ops.qk_norm_rope_fwd(x, x[..., :64], w, w, cos, sin, H, 2, D)
        dq, dk, dwq, dwk = ops.qk_norm_rope_bwd(q, k, x, x[..., :64], w, w, cos, sin, H, 2, D)
        return [x, q, k, dq, dk, dwq, dwk, ops.embedding_bwd(dq, ids, V, 2.0), ops.embedding_bwd(dmany, many, V)]

    work()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work()
    for i in range(4):
        ids.copy_(torch.randint(0, V, (2, 40), generator=g, device="cuda"))
        many.copy_(torch.randint(0, V if i % 2 else 2, (20000,), generator=g, device="cuda"))
        table.copy_(randn(g, V, d))
        want = work()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for j, (a, b) in enumerate(zip(got, want)):
            assert torch.equal(a, b), (i, j)


def test_training_run_of_them_together(ops):
    """token table -> fused projection -> norm + rotation -> attention -> loss, every gradient against a 64-bit model, and one 8-bit Adam step on all of them. At most 12 tensors on the
    way to a gradient are rounded to bf16, 2^-8 each at most: 12 * 2^-8 = 4.7e-2 in the norm"""
    from med_ts_llm_amd.hip.optim import HipAdam
    g = gen(12)
    B, T, V, d, H, Hkv, D = 2, 24, 50, 128, 4, 2, 64
    table = randn(g, V, d, std=0.5).requires_grad_()
    W = randn(g, (H + 2 * Hkv) * D, d, std=d ** -0.5).requires_grad_()
    wq, wk = (1 + randn(g, D, std=0.1)).requires_grad_(), (1 + randn(g, D, std=0.1)).requires_grad_()
    ids = torch.randint(0, V, (B, T), generator=g, device="cuda")
    ids[0, :5] = 0
    cos, sin = turn_tables(T, D)
    c = randn(g, B, T, H * D)

    class Attention(torch.autograd.Function):
        @staticmethod
        def forward(ctx, q, k, v):
            o, lse = ops.attention_fwd(q, k, v, H, Hkv, D, D ** -0.5, causal=True)
            ctx.save_for_backward(q, k, v, o, lse)
            return o

        @staticmethod
        def backward(ctx, do):
            return ops.attention_bwd(*ctx.saved_tensors, do, H, Hkv, D, D ** -0.5, causal=True)

    def forward():
        x = ops.EmbeddingFn.apply(ids, table, 2.0, 0, BF16)
        qkv = ops.LinearFn.apply(x, W, None)
        q, k = ops.QkNormRopeFn.apply(qkv[..., :H * D], qkv[..., H * D:(H + Hkv) * D], wq, wk, cos, sin, H, Hkv, D)
        return Attention.apply(q, k, qkv[..., (H + Hkv) * D:].contiguous())

    leaves = [table, W, wq, wk]
    (forward().float() * c).sum().backward()
    p = [t.detach().double().cpu().requires_grad_() for t in leaves]
    x = p[0][ids.cpu()] * 2.0
    x = torch.where((ids.cpu() == 0)[..., None], x.detach(), x)
    qkv = x @ p[1].t()
    cs, sn = cos.double().cpu()[:T][None, :, None], sin.double().cpu()[:T][None, :, None]

    def heads(t, w):
        t = t.unflatten(-1, (-1, D))
        return rot(t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-6) * w, cs, sn, D)

    q, k, v = heads(qkv[..., :H * D], p[2]), heads(qkv[..., H * D:(H + Hkv) * D], p[3]), qkv[..., (H + Hkv) * D:].unflatten(-1, (-1, D))
    k, v = (t.repeat_interleave(H // Hkv, 2) for t in (k, v))
    a = torch.einsum("bthd,bshd->bhts", q, k) * D ** -0.5
    a = a.masked_fill(torch.ones(T, T).triu(1).bool(), -math.inf).softmax(-1)
    (torch.einsum("bhts,bshd->bthd", a, v).flatten(-2) * c.double().cpu()).sum().backward()
    for n, t, r in zip("table W wq wk".split(), leaves, p):
        off = float((t.grad.double().cpu() - r.grad).norm() / r.grad.norm())
        assert off < 12 * 2.0 ** -8, (n, off)
    assert not table.grad[0].any()
    before = [t.detach().clone() for t in leaves]
    opt = HipAdam(leaves, lr=1e-3, state_bits=8)
    opt.step()
    for t, b in zip(leaves, before):
        # first step: m / (sqrt(v) + eps) is the gradient's sign wherever |g| is far above eps: lr within the roundings of seven operations and of the parameter
        big = t.grad.abs() > 1e-4
        moved = (b - t.detach())[big] * t.grad[big].sign()
        assert bool(((moved - 1e-3).abs() <= 1e-3 * 2e-4 + b[big].abs() * 2 * U).all())
    assert bool(torch.isfinite(forward()).all())


def test_trainer_with_8_bit_optimiser_state(tmp_path):
    """setup.optimizer_state_bits = 8 through the product trainer: it runs, its checkpoint record holds the codes, and another trainer takes them over"""
    from test_gpu_model import _trainer_config, _write_hf_dir
    from med_ts_llm_amd.tasks import get_trainer
    from med_ts_llm_amd.utils import dict_to_object
    _write_hf_dir(tmp_path, "gpt2")

    def cfg(epochs):
        c = _trainer_config("forecasting", str(tmp_path), epochs=epochs)
        c["setup"]["optimizer_state_bits"] = 8
        return dict_to_object(c)

    trainer = get_trainer("DEBUG-8bit", cfg(1))
    assert trainer.optimizer.state_bits == 8
    trainer.train()
    st = trainer.optimizer.state[next(p for p in trainer.model.parameters() if p.requires_grad)]
    assert st["exp_avg_q"].dtype == torch.uint8 and "exp_avg" not in st
    twin = get_trainer("DEBUG-8bit-2", cfg(1))
    assert twin.load_optimizer_state(trainer.optimizer_state())
    for p, q in zip(trainer.model.parameters(), twin.model.parameters()):
        if p in trainer.optimizer.state:
            assert all(torch.equal(trainer.optimizer.state[p][k], twin.optimizer.state[q][k]) for k in ("exp_avg_q", "exp_avg_sq_q", "q_exp"))
    twin.train()
