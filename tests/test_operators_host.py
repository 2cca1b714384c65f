"""CPU tests of the token-table, query / key norm and 8-bit Adam entry points: what they refuse, the 8-bit formats, the trainer's option."""
import numpy as np
import pytest
import torch

import adam8_ref as A8

F32, BF16 = torch.float32, torch.bfloat16


# ---------------------------------------------------------------- formats
def test_eight_bit_formats_round_trip_and_order():
    """every code decodes to a value that encodes to itself, the values are ordered, a block's largest value lands below both formats' ends"""
    finite = np.array([c for c in range(256) if (c & 0x7F) != 0x7F and c != 0x80])
    assert np.array_equal(A8.encode_e4m3(A8.E4M3[finite]), finite)
    assert np.all(np.diff(A8.ROOT[:255]) > 0) and A8.ROOT[240] == 2.0 ** 18 and np.isnan(A8.ROOT[255])
    assert np.array_equal(A8.E4M3[finite], torch.arange(256).to(torch.uint8).view(torch.float8_e4m3fn).float().numpy()[finite])
    g = np.random.RandomState(0)
    m = (g.randn(64 * 50) * np.exp(g.randn(64 * 50) * 3)).astype(np.float32)
    r = np.abs(g.randn(64 * 50) * np.exp(g.randn(64 * 50) * 3)).astype(np.float32)
    cm, cr, ex = A8.encode(m, r, 7)
    assert (cr <= 240).all() and ((cm & 0x7F) <= 0x78).all()             # 0x78 = 256
    dm, dr = A8.decode(cm, cr, ex)
    # half a step of a 3-bit mantissa, or half of the smallest step 2^-9 of the block's scale; a whole step of a 4-bit mantissa, or of 1, for the threshold rounding
    sm, sr = (np.exp2(ex[:, i].astype(np.float64))[np.arange(m.size) // 64] for i in (0, 1))
    assert np.all(np.abs(dm - m) <= np.maximum(np.abs(m) * 2.0 ** -4, sm * 2.0 ** -10))
    assert np.all(np.abs(dr - r) <= np.maximum(r * 2.0 ** -4, sr))
    assert np.all(dr[r > 0] > 0)
    again = A8.encode(dm, dr, 8)                                         # values on their grid stay there, whatever the threshold
    same_scale = np.repeat((again[2] == ex).all(1), 64)
    assert np.array_equal(again[0][same_scale], cm[same_scale]) and np.array_equal(again[1][same_scale], cr[same_scale])


def test_second_moment_follows_its_gradients_in_eight_bits():
    """After 800 steps at one gradient scale and 3000 at half of it, the mean second moment is what the exact average says, within 5 %: the threshold rounding adds a variance of
    (relative step of r) x (its movement per step, about 1 / 2000) = 0.0625 x 0.0005 per step in r, i.e. 2 x that as a bias of the mean of v = r^2 per step against a decay of 1e-3:
    at most 2 * 0.0625 * 0.0005 / 2 / 1e-3 = 3.2 %, and a standard deviation of the mean over 4096 elements below 1 %. Rounding to nearest does not follow at all."""
    g = np.random.RandomState(1)
    n, b2 = 4096, 0.999
    out = {}
    for nearest in (False, True):
        gr = np.random.RandomState(2)
        p, codes, v = np.zeros(n, np.float32), A8.encode(np.zeros(n, np.float32), np.zeros(n, np.float32), 0), np.zeros(n)
        for t in range(1, 3801):
            x = (gr.randn(n) * (1e-2 if t <= 800 else 5e-3)).astype(np.float32)
            v = b2 * v + (1 - b2) * x.astype(np.float64) ** 2
            p, codes = A8.step(p, x, codes, t, 1e-3, 0.9, b2, 1e-8, nearest=nearest)
        r = A8.decode(*codes)[1].astype(np.float64)
        out[nearest] = (r ** 2).mean() / v.mean()
    assert abs(out[False] - 1) < 0.05, out
    assert abs(out[True] - 1) > 0.2, out


# ---------------------------------------------------------------- refusals (each before anything touches a GPU)
def test_embedding_refusals():
    from med_ts_llm_amd.hip import ops
    t = torch.zeros(5, 8)
    ids = torch.zeros(3, dtype=torch.int64)
    for bad in (lambda: ops.embedding_fwd(ids.float(), t), lambda: ops.embedding_fwd(ids.to(torch.int16), t), lambda: ops.embedding_fwd(ids, t.half()),
                lambda: ops.embedding_fwd(ids, t[0]), lambda: ops.embedding_fwd(ids, t, out_dtype=torch.float16), lambda: ops.embedding_fwd(ids, t.t()),
                lambda: ops.embedding_fwd(ids, torch.zeros(1, 8).expand(5, 8)), lambda: ops.embedding_fwd(ids, torch.zeros(0, 8)), lambda: ops.embedding_fwd(ids, t),
                lambda: ops.embedding_bwd(torch.zeros(4, 8), ids, 5), lambda: ops.embedding_bwd(torch.zeros(3, 8).half(), ids, 5), lambda: ops.embedding_bwd(torch.zeros(3, 8), ids, 5, padding_idx=5),
                lambda: ops.embedding_bwd(torch.zeros(3, 8), ids, 5, padding_idx=-1), lambda: ops.embedding_bwd(torch.zeros(3, 8), ids, 5, accumulate=True),
                lambda: ops.embedding_bwd(torch.zeros(3, 8), ids, 5, out=torch.zeros(5, 7)), lambda: ops.embedding_bwd(torch.zeros(3, 8), ids, 5, out=torch.zeros(1, 8).expand(5, 8)),
                lambda: ops.embedding_bwd(torch.zeros(3, 8), ids, 5, out_dtype=torch.float64), lambda: ops.embedding_bwd(torch.zeros(3, 8), ids, 5),
                lambda: ops.EmbeddingFn.apply(ids, t, 1.0, 5, None)):
        with pytest.raises(ValueError):
            bad()


def test_qk_norm_rope_refusals():
    from med_ts_llm_amd.hip import ops

    def call(q=None, k=None, w=None, wk=None, cos=None, sin=None, Hq=2, Hkv=1, D=8, bwd=False, **kw):
        q = torch.zeros(2, 3, 16) if q is None else q
        k = torch.zeros(2, 3, 8) if k is None else k
        w = torch.ones(8) if w is None else w
        cos = torch.ones(10, 8) if cos is None else cos
        return ops.qk_norm_rope_fwd(q, k, w, w if wk is None else wk, cos, cos if sin is None else sin, Hq, Hkv, D, **kw)

    fused = torch.zeros(2, 3, 32)
    q, k = fused[..., :16], fused[..., 16:24]
    bad = [dict(q=torch.zeros(2, 3, 15)), dict(q=torch.zeros(6, 16)), dict(k=torch.zeros(2, 4, 8)), dict(k=torch.zeros(2, 3, 8, dtype=BF16)), dict(q=torch.zeros(2, 3, 16).half(), k=torch.zeros(2, 3, 8).half()),
           dict(q=torch.zeros(2, 3, 32)[..., ::2]), dict(w=torch.ones(7)), dict(wk=torch.ones(8, dtype=BF16)), dict(w=torch.ones(8).double()), dict(cos=torch.ones(10, 10)), dict(cos=torch.ones(10, 5)),
           dict(cos=torch.ones(10, 8).double()), dict(sin=torch.ones(9, 8)), dict(cos=torch.ones(10, 16)[:, ::2]), dict(pos0=8), dict(pos0=-1), dict(positions=torch.zeros(2, 4, dtype=torch.int64)),
           dict(positions=torch.zeros(2, 3)), dict(positions=torch.zeros(2, 3, dtype=torch.int64), pos0=1), dict(Hq=0), dict(q=torch.zeros(2, 3, 14), k=torch.zeros(2, 3, 7), D=7, w=torch.ones(7), cos=torch.ones(10, 6)),
           dict(q=torch.zeros(1, 1, 1028), k=torch.zeros(1, 1, 514), D=514, w=torch.ones(514), cos=torch.ones(10, 8)),
           dict(out=(torch.zeros(2, 3, 16), torch.zeros(2, 3, 16))), dict(out=(torch.zeros(1, 1, 16).expand(2, 3, 16), torch.zeros(2, 3, 8))),
           dict(q=q, k=k, out=(k.expand(2, 3, 8).repeat(1, 1, 2), fused[..., 24:32])),          # an output in the inputs' buffer that is not its own input
           dict(q=q, k=fused[..., 8:16], out=(q, fused[..., 8:16])),                              # in place with overlapping inputs
           dict()]                                                                                 # (sound, but on the CPU)
    for kw in bad:
        with pytest.raises(ValueError):
            call(**kw)
    with pytest.raises(ValueError):
        ops.qk_norm_rope_bwd(torch.zeros(2, 3, 16), torch.zeros(2, 3, 8, dtype=BF16), torch.zeros(2, 3, 16), torch.zeros(2, 3, 8), torch.ones(8), torch.ones(8), torch.ones(10, 8), torch.ones(10, 8), 2, 1, 8)


def test_adam8_refusals():
    from med_ts_llm_amd.hip import _native as N
    from med_ts_llm_amd.hip import optim
    p, g = torch.zeros(10, 7), torch.zeros(10, 7)
    st = optim.adam8_state(p)
    assert st.exponents.shape == (2, 2)
    for bad in (lambda: optim.adam8_step([p], [g], [], 1), lambda: optim.adam8_step([p], [g], [st], 0), lambda: optim.adam8_step([p], [g], [st], 1, betas=(1.0, 0.9)),
                lambda: optim.adam8_step([p], [g], [st], 1, eps=-1.0), lambda: optim.adam8_step([p.half()], [g.half()], [st], 1), lambda: optim.adam8_step([p], [g.to(BF16)], [st], 1),
                lambda: optim.adam8_step([p.t()], [g.t()], [st], 1), lambda: optim.adam8_step([p], [g[:5]], [st], 1), lambda: optim.adam8_step([p], [g], [optim.adam8_state(p[:5])], 1),
                lambda: optim.adam8_step([p], [g], [optim.Adam8State(st.exp_avg, st.exp_avg_sq, st.exponents[:1])], 1), lambda: optim.adam8_step([p, p], [g, g], [st, optim.adam8_state(p)], 1),
                lambda: optim.adam8_step([p, torch.zeros(10, 7)], [g, g], [st, st], 1), lambda: optim.adam8_moments([st], torch.float16), lambda: optim.adam8_quantize(p, g[:5]),
                lambda: optim.adam8_quantize(p.double(), g.double()), lambda: optim.HipAdam([torch.nn.Parameter(p)], state_bits=4)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(N.MtlError):
        optim.adam8_step([p], [g], [st], 1)
    assert optim.adam8_step([], [], [], 1) is None and optim.adam8_moments([]) == []


def test_c_entry_points_refuse_bad_arguments_without_a_gpu():
    """null pointers, sizes, alignments and too small workspaces come back as error codes"""
    import ctypes as C
    from med_ts_llm_amd.hip import _native as N
    lib = N.lib()
    buf = (C.c_char * 4096)()
    at = (C.addressof(buf) + 255) // 256 * 256
    ARG, ALIGN, UNSUPPORTED, WORKSPACE = -1, -2, -3, -5
    assert lib.mtl_embedding_fwd(None, 1, 4, at, 0, 5, 8, 8, 1.0, at, 0, 8, None) == ARG
    assert lib.mtl_embedding_fwd(at, 1, 4, at, 0, 5, 8, 7, 1.0, at, 0, 8, None) == ARG
    assert lib.mtl_embedding_fwd(at, 1, 4, at, 2, 5, 8, 8, 1.0, at, 0, 8, None) == ARG
    assert lib.mtl_embedding_fwd(at + 4, 1, 4, at, 0, 5, 8, 8, 1.0, at, 0, 8, None) == ALIGN
    assert lib.mtl_embedding_fwd(None, 1, 0, None, 0, 5, 8, 8, 1.0, None, 0, 8, None) == 0
    assert lib.mtl_embedding_bwd(at, 1, 4, at, 0, 8, 5, 8, -1, 1.0, at, 0, 8, 0, at, 16, None) == WORKSPACE
    assert lib.mtl_embedding_bwd(at, 1, 1 << 31, at, 0, 8, 5, 8, -1, 1.0, at, 0, 8, 0, at, 1 << 40, None) == UNSUPPORTED
    assert lib.mtl_embedding_bwd(at, 1, 4, at, 0, 8, 5, 8, -1, 1.0, None, 0, 8, 0, at, 4096, None) == ARG
    assert lib.mtl_embedding_bwd(None, 1, 0, None, 0, 8, 5, 8, -1, 1.0, at, 0, 8, 1, None, 0, None) == 0
    a = N.QkNormRopeArgs()
    assert lib.mtl_qk_norm_rope_fwd(C.byref(a), None) == ARG
    a.B, a.T, a.Hq, a.Hkv, a.D, a.R, a.n_pos = 1, 1, 1, 1, 8, 8, 4
    assert lib.mtl_qk_norm_rope_fwd(C.byref(a), None) == ARG
    for n in ("q", "k", "q_out", "k_out", "wq", "wk", "cos_t", "sin_t", "dq_out", "dk_out", "dwq", "dwk"):
        setattr(a, n, at)
    assert lib.mtl_qk_norm_rope_bwd(C.byref(a), None) == WORKSPACE
    a.q = at + 2
    assert lib.mtl_qk_norm_rope_fwd(C.byref(a), None) == ALIGN
    a.q, a.D, a.R = at, 514, 8
    assert lib.mtl_qk_norm_rope_fwd(C.byref(a), None) == UNSUPPORTED
    a.D, a.T = 8, 0
    assert lib.mtl_qk_norm_rope_fwd(C.byref(a), None) == 0
    t = (N.Adam8Tensor * 1)()
    t[0].n, t[0].p = 4, at
    assert lib.mtl_adam8_step(t, 1, 1e-3, 0.9, 0.999, 1e-8, 0.0, 0, 1, None) == ARG
    t[0].g = t[0].m8 = t[0].r8 = at
    t[0].ex = at + 1
    assert lib.mtl_adam8_step(t, 1, 1e-3, 0.9, 0.999, 1e-8, 0.0, 0, 1, None) == ALIGN
    assert lib.mtl_adam8_step(t, 1, 1e-3, 1.0, 0.999, 1e-8, 0.0, 0, 1, None) == ARG
    t[0].n = 0
    assert lib.mtl_adam8_step(t, 1, 1e-3, 0.9, 0.999, 1e-8, 0.0, 0, 1, None) == 0


def test_c_entry_points_refuse_more_threads_than_a_launch_holds():
    """2^32 threads and more: an error before the first launch, also where a smaller tensor stands in front"""
    import ctypes as C
    from med_ts_llm_amd.hip import _native as N
    lib = N.lib()
    buf = (C.c_char * 4096)()
    at = (C.addressof(buf) + 255) // 256 * 256
    assert lib.mtl_embedding_bwd(at, 1, 1 << 30, at, 0, 4096, 5, 4096, -1, 1.0, at, 0, 4096, 0, at, 1 << 62, None) == -3
    t = (N.Adam8Tensor * 200)()
    s = (N.Adam8State * 200)()
    for i in range(200):
        t[i].p = t[i].g = t[i].m8 = t[i].r8 = t[i].ex = s[i].m8 = s[i].r8 = s[i].ex = s[i].m = s[i].v = at
        t[i].n = s[i].n = 4 if i < 199 else 1 << 34
    assert lib.mtl_adam8_step(t, 200, 1e-3, 0.9, 0.999, 1e-8, 0.0, 0, 1, None) == -3
    assert lib.mtl_adam8_moments(s, 200, None) == -3 and lib.mtl_adam8_quantize(s, 200, 1, None) == -3


def test_embedding_workspace_holds_every_part():
    from med_ts_llm_amd.hip import _native as N
    f = N.lib().mtl_embedding_bwd_workspace_bytes
    for n, v, d in ((1, 1, 1), (16384, 50257, 768), (16385, 50257, 768), (200003, 32000, 1024)):
        assert f(n, v, d) >= 8 * n + 8 * ((n + 63) // 64) * d
    assert f(0, 5, 8) > 0
