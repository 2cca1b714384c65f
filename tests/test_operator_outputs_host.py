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
