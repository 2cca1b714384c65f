"""CPU tests of what the token table's and the query / key norm's entry points say about the tensors they write: versions for autograd, shared memory. The library's calls are replaced by
nothing (each would return success), the checks in front of them and what follows them run as they are."""
import contextlib

import pytest
import torch

F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture
def ops(monkeypatch):
    from med_ts_llm_amd.hip import ops

    class Library:
        def __getattr__(self, name):
            return lambda *a: 256 if name.endswith("_bytes") else 0

    monkeypatch.setattr(ops, "lib", Library)
    monkeypatch.setattr(ops, "_req_gpu", lambda *t: None)
    monkeypatch.setattr(ops, "stream", lambda: None)
    monkeypatch.setattr(ops.N, "on_device", lambda t: contextlib.nullcontext())
    return ops


def qk(B=2, T=3, Hq=2, Hkv=1, D=8):
    cos = torch.ones(10, D)
    return torch.zeros(B, T, Hq * D), torch.zeros(B, T, Hkv * D), torch.ones(D), torch.ones(D), cos, cos, Hq, Hkv, D


# ---------------------------------------------------------------- versions
def test_given_outputs_change_their_version(ops):
    """what a call writes through a pointer counts as an in-place operation: autograd then notices that a tensor saved for a backward pass has changed"""
    a = qk()
    base = torch.zeros(2, 3, 40)
    new = (base[..., :16], base[..., 16:24])
    for call in (lambda: ops.qk_norm_rope_fwd(*a, out=a[:2]), lambda: ops.qk_norm_rope_fwd(*a, out=new), lambda: ops.qk_norm_rope_bwd(torch.ones(2, 3, 16), torch.ones(2, 3, 8), *a, out=new)):
        before = [t._version for t in (a[0], a[1], base)]
        call()
        after = [t._version for t in (a[0], a[1], base)]
        assert (after[2] > before[2]) if after[:2] == before[:2] else (after[0] > before[0] and after[1] > before[1])
    grad = torch.zeros(5, 16)
    for kw in ({}, {"accumulate": True}):
        before = grad._version
        ops.embedding_bwd(torch.ones(3, 8), torch.zeros(3, dtype=torch.int64), 5, out=grad[:, :8], **kw)
        assert grad._version > before


def test_rotation_in_place_of_a_saved_tensor_is_noticed(ops):
    q, k, *rest = qk()
    q.requires_grad_()
    x = q * 1.0
    y = (x * x).sum()                                            # (saves x)
    with torch.no_grad():
        ops.qk_norm_rope_fwd(x, k, *rest, out=(x, k))
    with pytest.raises(RuntimeError, match="inplace"):
        y.backward()


# ---------------------------------------------------------------- shared memory
def elements(t):
    return set(torch.arange(t.untyped_storage().nbytes() // t.element_size()).as_strided(t.shape, t.stride(), t.storage_offset()).reshape(-1).tolist())


def test_apart_is_what_the_elements_say(ops):
    """random views of one buffer: rows, columns, batches, orders, broadcast dimensions; the answer is exact"""
    import random
    rng = random.Random(1)
    buf = torch.zeros(6000)
    seen = [0, 0]
    for _ in range(4000):
        views = []
        for _ in range(2):
            B, T, W = rng.randint(1, 4), rng.randint(1, 5), rng.randint(1, 9)
            strides = [rng.choice([0, W, W + 3, 16, 40, 48, 60, 100, 240]) for _ in range(2)]
            views.append(buf.as_strided((B, T, W), (*strides, 1), rng.randint(0, 300)))
        a, b = views
        want = not (elements(a) & elements(b))
        assert ops._apart(a, b) == want == ops._apart(b, a), [(v.shape, v.stride(), v.storage_offset()) for v in views]
        seen[want] += 1
    assert min(seen) > 500
    assert ops._apart(buf[:0], buf) and ops._apart(buf[:10], buf[10:]) and not ops._apart(buf[:10], buf[9:])


def test_outputs_and_inputs_out_of_one_allocation(ops):
    """a query output and a key cache carved from one arena, an output beside the inputs in their own buffer: taken where no element is shared"""
    q, k, *rest = qk(B=2, T=1)
    arena = torch.zeros(2 * 16 + 2 * 10 * 8 * 2)
    new_q, cache = arena[:32].view(2, 1, 16), arena[32:].view(2, 10, 2, 8)
    ops.qk_norm_rope_fwd(q, k, *rest, out=(new_q, cache[:, 4:5, 0]))
    per_sequence = torch.zeros(2, 16 + 10 * 8)                     # [query | its cache] of every sequence
    ops.qk_norm_rope_fwd(q, k, *rest, out=(per_sequence[:, None, :16], per_sequence[:, 16:].view(2, 10, 8)[:, 4:5]))
    fused = torch.zeros(2, 3, 64)
    q, k, *rest = qk()
    q, k = fused[..., :16], fused[..., 16:24]
    ops.qk_norm_rope_fwd(q, k, *rest, out=(q, k))                  # in place
    ops.qk_norm_rope_fwd(q, k, *rest, out=(q, fused[..., 24:32]))   # the queries in place, the keys beside them
    ops.qk_norm_rope_fwd(q, k, *rest, out=(fused[..., 32:48], fused[..., 48:56]))
    one = fused[:1, :1]
    ops.qk_norm_rope_fwd(one[..., :16], one[..., 16:24], *rest, out=(one.as_strided((1, 1, 16), (16, 16, 1)), one[..., 16:24]))      # the same row under other strides
    dq, dk = torch.zeros(2, 3, 16), torch.zeros(2, 3, 8)
    ops.qk_norm_rope_bwd(dq, dk, q, k, *rest, out=(fused[..., 32:48], fused[..., 48:56]))
    both = torch.zeros(30, 16)
    ops.embedding_bwd(both[:3, 8:], torch.zeros(3, dtype=torch.int64), 30, out=both[:, :8])


def test_outputs_that_share_elements_are_refused(ops):
    q, k, *rest = qk()
    fused = torch.zeros(2, 3, 64)
    fq, fk = fused[..., :16], fused[..., 16:24]
    flat = torch.zeros(400)
    bad = [dict(q=fq, k=fk, out=(fq, fused[..., 8:16])), dict(q=fq, k=fk, out=(fk.expand(2, 3, 8).repeat(1, 1, 2), fq[..., :8])), dict(q=fq, k=fk, out=(fused[..., 8:24], fk)),
           dict(q=fq, k=fused[..., 8:16], out=(fq, fused[..., 8:16])), dict(out=(fused[..., :16], fused[..., 15:23])),
           dict(q=flat[:96].view(2, 3, 16), out=(flat[48:144].view(2, 3, 16), torch.zeros(2, 3, 8))),                         # the second sequence's queries where the first one's results go
           dict(q=fq[:, :, :], k=fk, out=(fused.as_strided((2, 3, 16), (16, 64, 1)), torch.zeros(2, 3, 8))),
           dict(out=(torch.zeros(2, 3), torch.zeros(2, 3, 8))), dict(out=(torch.zeros(()), torch.zeros(2, 3, 8)))]
    for kw in bad:
        out = kw.pop("out")
        with pytest.raises(ValueError):
            ops.qk_norm_rope_fwd(kw.get("q", q), kw.get("k", k), *rest, out=out)
        if "q" in kw:
            with pytest.raises(ValueError):
                ops.qk_norm_rope_bwd(torch.zeros(2, 3, 16), torch.zeros(2, 3, 8), kw["q"], kw.get("k", k), *rest, out=out)
    both = torch.zeros(30, 16)
    with pytest.raises(ValueError):
        ops.embedding_bwd(both[:3, 7:15], torch.zeros(3, dtype=torch.int64), 30, out=both[:, :8])


# ---------------------------------------------------------------- sizes
def test_token_gradient_sizes_and_their_workspace():
    """the limit that the header states, of the call and of its workspace query alike (no pointer is followed: all are null or the call is refused)"""
    from med_ts_llm_amd.hip import _native as N
    lib = N.lib()

    def call(n, v, d):
        return lib.mtl_embedding_bwd(None, 1, n, None, 0, d, v, d, -1, 1.0, None, 0, d, 0, None, 0, None)

    for n, v, d, fine in ((1, 5, 8, True), ((1 << 31) - 1, 5, 256, True), ((1 << 31) - 1, 5, 257, False), (1 << 31, 5, 8, False), (1, (1 << 31) - 1, 8, False), (1, (1 << 31) - 2, 8, True),
                          ((1 << 28) - 64, 1000, 4096, True), (1 << 28, 1000, 4096, False), (1 << 30, 5, 4096, False), (128, 5, 256 * ((1 << 25) - 2), True), (128, 5, 256 * ((1 << 25) - 1), False), (128, 5, 1 << 33, False)):
        assert call(n, v, d) == (-1 if fine else -3), (n, v, d)
        assert (lib.mtl_embedding_bwd_workspace_bytes(n, v, d) > 0) == fine, (n, v, d)
