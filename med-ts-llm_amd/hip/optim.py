"""Adam / AdamW on the HIP path: torch.optim.Adam semantics (R:tasks/base.py:97,99), one streaming launch for all
trainable tensors (`mtl_adam_step`), optionally emitting the bf16 autocast copy of a weight while it is being updated.

state_dict layout matches torch.optim.Adam ("step", "exp_avg", "exp_avg_sq"), so checkpoints interchange.

HipAdam(state_bits=8) holds both moments in 8 bits (`mtl_adam8_step`: 2.03 bytes of state per parameter instead of 8): state "step", "exp_avg_q", "exp_avg_sq_q" (codes of the
parameter's shape), "q_exp" (exponents [blocks of 64, 2]). Both are rounded against thresholds of (step, element), so that a run of steps is right in the mean. A state saved at the other width is converted at the first step after it is loaded."""
import collections
import ctypes as C
import warnings

import torch

from . import _native as N


class Bf16Shadow:
    """bf16 [rows, ld] copy of an fp32 [rows, cols] parameter, kept current by HipAdam. `version` is the parameter's
    `_version` the shadow corresponds to; owners compare it with `param._version` before trusting the copy."""

    def __init__(self, param, tensor):
        assert param.dim() == 2 and tensor.dim() == 2 and tensor.dtype == torch.bfloat16
        assert tensor.shape[0] == param.shape[0] and tensor.stride(1) == 1 and tensor.stride(0) >= param.shape[1]
        self.param, self.tensor, self.version = param, tensor, -1

    def fresh(self):
        return self.version == self.param._version


_STATE8 = ("exp_avg_q", "exp_avg_sq_q", "q_exp")
Adam8State = collections.namedtuple("Adam8State", ["exp_avg", "exp_avg_sq", "exponents"])
Adam8State.__doc__ = """moments in 8 bits: uint8 codes of the first moment and of the root of the second, in the parameter's shape, and one signed exponent byte of each per block of 64
consecutive elements, uint8 [ceil(n / 64), 2]"""


_PARAM_TYPES = {torch.float32: N.MTL_F32, torch.bfloat16: N.MTL_BF16}


def _state8_row(st, what):
    """(codes, codes, exponents, n) as pointers and the element count of a checked state"""
    m8, r8, ex = st
    n = m8.numel()
    u8 = torch.uint8
    if not (m8.dtype is u8 and r8.dtype is u8 and ex.dtype is u8 and r8.numel() == n and ex.numel() == (n + N.ADAM8_BLOCK - 1) // N.ADAM8_BLOCK * 2
            and m8.is_contiguous() and r8.is_contiguous() and ex.is_contiguous()):
        raise ValueError(f"{what}: an 8-bit state is contiguous uint8: two code tensors of one size and two exponents for every 64 of their elements")
    return m8.data_ptr(), r8.data_ptr(), ex.data_ptr(), n


def _one_gpu(tensors, what):
    dev = tensors[0].get_device()
    if dev < 0:
        raise N.MtlError(f"{what} needs tensors on the GPU (no CPU fallback)")
    for t in tensors:
        if t.get_device() != dev:
            raise ValueError(f"{what}: tensors on different devices")


def adam8_state(p):
    """the state of a parameter that has not been stepped: zero moments"""
    return Adam8State(torch.zeros(p.shape, dtype=torch.uint8, device=p.device), torch.zeros(p.shape, dtype=torch.uint8, device=p.device),
                      torch.zeros(((p.numel() + N.ADAM8_BLOCK - 1) // N.ADAM8_BLOCK, 2), dtype=torch.uint8, device=p.device))


_said_nearest = False


@torch.no_grad()
def adam8_step(params, grads, states, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, decoupled_weight_decay=False, shadows=None, first_moment=None):
    """one Adam / AdamW step, in place, of several tensors (contiguous, f32 or bf16, gradients likewise) whose moments are Adam8States; `step` counts from 1 and is the same for all.
    shadows: Bf16Shadow or None for each. One launch per 40 tensors. Same result for the same inputs and step, bit for bit. (In a captured graph the step number is a constant.)
    first_moment: how the new first moment is rounded to its code. "threshold": up or down, by a hash of (step, element), so that it is right in the mean over a run of steps, for every
    beta1 (what HipAdam takes). "nearest": the closest code, for a single step; over a run it stands still wherever (1 - beta1) |g - m| is below half a step of its grid: a constant
    gradient is held at 0.5 to 0.8 of its value, one that stops leaves a rest that moves its parameter for ever. Not given: "nearest", with a warning (once)."""
    global _said_nearest
    if first_moment is None:
        if not _said_nearest:
            _said_nearest = True
            warnings.warn('adam8_step rounds the first moment to the nearest code, which a run of steps cannot follow: give first_moment="threshold" (or "nearest", for a single step)', stacklevel=3)
    elif first_moment not in ("nearest", "threshold"):
        raise ValueError(f'adam8_step: first_moment is "nearest" or "threshold", got {first_moment!r}')
    flags = (N.ADAM8_DECOUPLED if decoupled_weight_decay else 0) | (N.ADAM8_M_THRESHOLD if first_moment == "threshold" else 0)
    params, grads, states = list(params), list(grads), list(states)
    shadows = [None] * len(params) if shadows is None else list(shadows)
    if not len(params) == len(grads) == len(states) == len(shadows):
        raise ValueError("adam8_step: as many gradients, states and shadows as parameters")
    step, (b1, b2), lr, eps, weight_decay = int(step), map(float, betas), float(lr), float(eps), float(weight_decay)
    if step < 1 or not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0 and eps >= 0.0 and weight_decay >= 0.0):
        raise ValueError("adam8_step: step >= 1, betas in [0, 1), eps and weight_decay not negative")
    if not params:
        return
    rows, touched, read = [], [], []
    for p, g, st, sh in zip(params, grads, states, shadows):
        dt = p.dtype
        if dt not in _PARAM_TYPES or g.dtype is not dt or g.shape != p.shape or not p.is_contiguous() or not g.is_contiguous():
            raise ValueError("adam8_step: contiguous f32 or bf16 parameters with gradients of the same type and shape")
        m8, r8, ex, n = _state8_row(st, "adam8_step")
        if n != p.numel():
            raise ValueError("adam8_step: a state of another size than its parameter")
        rows += (p.data_ptr(), g.data_ptr(), m8, r8, ex, n)
        if sh is not None and (p.dim() != 2 or sh.tensor.shape[0] < p.shape[0] or sh.tensor.shape[1] < p.shape[1]):
            raise ValueError("adam8_step: a bf16 copy of another parameter")
        rows += (0, 0, 0) if sh is None else (sh.tensor.data_ptr(), p.shape[1], sh.tensor.stride(0))
        rows.append(_PARAM_TYPES[dt])
        touched += (p, *st)
        read.append(g)
        if sh is not None:
            read.append(sh.tensor)
    held = rows[5::10]
    for name, columns in (("parameter", (0,)), ("state", (2, 3, 4))):
        ptrs = [x for at in columns for x, n in zip(rows[at::10], held) if n]
        if len(set(ptrs)) < len(ptrs):
            raise ValueError(f"adam8_step: the same {name} twice in one step")
    _one_gpu(touched + read, "adam8_step")
    with N.on_device(params[0]):
        N.check(N.lib().mtl_adam8_step((N.i64 * len(rows))(*rows), len(params), lr, b1, b2, eps, weight_decay, flags, step, N.stream()), "mtl_adam8_step")
    torch.autograd.graph.increment_version(touched)   # the kernel wrote through raw pointers: bump the autograd versions like an in-place op
    for p, sh in zip(params, shadows):
        if sh is not None:
            sh.version = p._version


def _state8_rows(rows, ms, vs):
    """mtl_adam8_state structures (7 64-bit words each)"""
    flat = []
    for (m8, r8, ex, n), m, v in zip(rows, ms, vs):
        flat += (m8, r8, ex, n, m.data_ptr(), v.data_ptr(), _PARAM_TYPES[m.dtype])
    return (N.i64 * len(flat))(*flat)


@torch.no_grad()
def adam8_moments(states, dtype=torch.float32):
    """[(exp_avg, exp_avg_sq)] that the states' codes stand for: exact in f32; in bf16 the first moment is exact, the second rounded once"""
    states = list(states)
    if dtype not in _PARAM_TYPES:
        raise ValueError("adam8_moments: f32 or bf16")
    rows = [_state8_row(st, "adam8_moments") for st in states]
    if not states:
        return []
    _one_gpu([t for st in states for t in st], "adam8_moments")
    with N.on_device(states[0].exp_avg):
        ms, vs = ([torch.empty_like(st.exp_avg, dtype=dtype) for st in states] for _ in range(2))
        N.check(N.lib().mtl_adam8_moments(_state8_rows(rows, ms, vs), len(rows), N.stream()), "mtl_adam8_moments")
    return list(zip(ms, vs))


@torch.no_grad()
def adam8_quantize(exp_avg, exp_avg_sq, step=0):
    """Adam8State of fp32 moments (`step`: how many steps they have seen; it selects the rounding thresholds)"""
    if exp_avg.dtype != torch.float32 or exp_avg_sq.dtype != torch.float32 or exp_avg.shape != exp_avg_sq.shape or int(step) < 0:
        raise ValueError("adam8_quantize: two fp32 moments of one shape, step not negative")
    m, v = exp_avg.contiguous(), exp_avg_sq.contiguous()
    _one_gpu([m, v], "adam8_quantize")
    with N.on_device(m):
        st = adam8_state(m)
        N.check(N.lib().mtl_adam8_quantize(_state8_rows([_state8_row(st, "adam8_quantize")], [m], [v]), 1, int(step), N.stream()), "mtl_adam8_quantize")
    return st


class HipAdam(torch.optim.Optimizer):
    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, decoupled_weight_decay=False, state_bits=32):
        """state_bits = 8: both moments of every parameter in 8 bits (see the module's docstring)"""
        if state_bits not in (8, 32):
            raise ValueError(f"HipAdam: state_bits is 8 or 32, got {state_bits!r}")
        self.state_bits = state_bits
        defaults = dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, decoupled_weight_decay=decoupled_weight_decay)
        super().__init__(params, defaults)
        self._shadows = {}
        self._late, self._side, self._late_done = set(), None, None

    def register_shadow(self, shadow):
        self._shadows[id(shadow.param)] = shadow

    def defer(self, params):
        """Parameters that the NEXT forward reads only after the frozen backbone (down-sample layer, flatten head): their update runs on a side
        stream, ordered after everything the step has enqueued so far, and overlaps the next step's front end and backbone — HBM-bound Adam traffic
        under MFMA-bound GEMMs (the PSM head: 8 ms of a 226 ms step). Whoever reads such a parameter next must call wait_deferred() first
        (MedTsLLM.predict does, in front of the down-sample GEMM; the trainer before validation / checkpoints). Same arithmetic, same results."""
        self._late = {id(p) for p in params}
        if self._late and self._side is None:
            self._side = torch.cuda.Stream()

    def wait_deferred(self):
        """make the current stream wait for the deferred updates launched by the last step() (no-op when there are none)"""
        if self._late_done is not None:
            torch.cuda.current_stream().wait_event(self._late_done)
            self._late_done = None

    def _after_deferred(self):
        """the current stream waits for the deferred updates, whose event stays for the stream that reads the parameters: whoever reads or replaces the optimiser's state comes here first"""
        if self._late_done is not None:
            torch.cuda.current_stream().wait_event(self._late_done)

    def state_dict(self):
        self._after_deferred()
        return super().state_dict()

    def load_state_dict(self, state_dict):
        """torch's Optimizer.load_state_dict casts every floating-point state tensor to its parameter's dtype; the moments of bf16 parameters
        (setup.dtype = "bf16") must stay fp32 — the kernel reads and writes them as float*."""
        self._after_deferred()
        super().load_state_dict(state_dict)
        # (re-widening the narrowed copies would keep their bf16 rounding: take the moments from the saved tensors themselves)
        mine = [p for g in self.param_groups for p in g["params"]]
        saved = [i for g in state_dict["param_groups"] for i in g["params"]]
        for idx, p in zip(saved, mine):
            rec = state_dict["state"].get(idx)
            if not rec:
                continue
            for k in ("exp_avg", "exp_avg_sq"):
                if torch.is_tensor(rec.get(k)):
                    self.state[p][k] = rec[k].detach().to(device=p.device, dtype=torch.float32).contiguous().clone()
            for k in _STATE8:
                if torch.is_tensor(rec.get(k)):
                    self.state[p][k] = rec[k].detach().to(device=p.device).contiguous().clone()

    def moments(self, dtype=torch.float32):
        """{parameter: (exp_avg, exp_avg_sq)} of every parameter that has been stepped, whatever width they are held in: copies, as of the last step, its deferred updates among it"""
        self._after_deferred()
        held = {p: st for p, st in self.state.items() if st}
        coded = [p for p, st in held.items() if _STATE8[0] in st]
        out = dict(zip(coded, adam8_moments([Adam8State(*(held[p][k] for k in _STATE8)) for p in coded], dtype)))
        return {p: out[p] if p in out else (st["exp_avg"].to(dtype, copy=True), st["exp_avg_sq"].to(dtype, copy=True)) for p, st in held.items()}

    def _to_width(self, st, p):
        """a state at the optimiser's own width: new, or converted from what a checkpoint of the other width held (which goes only once the conversion is done)"""
        wide = ("exp_avg", "exp_avg_sq")
        if self.state_bits == 8 and _STATE8[0] not in st:
            st.update(zip(_STATE8, adam8_quantize(*(st[k] for k in wide), st["step"]) if wide[0] in st else adam8_state(p)))
            old = wide
        elif self.state_bits == 32 and wide[0] not in st:
            # moments are fp32 also for bf16 parameters (setup.dtype = "bf16"): the update is formed in fp32 and the parameter rounded once
            st.update(zip(wide, adam8_moments([Adam8State(*(st[k] for k in _STATE8))])[0] if _STATE8[0] in st else
                          [torch.zeros_like(p, dtype=torch.float32, memory_format=torch.contiguous_format) for _ in range(2)]))
            old = _STATE8
        else:
            return
        for k in old:
            st.pop(k, None)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if self.state_bits == 8 and torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            raise N.MtlError("HipAdam(state_bits=8).step() inside a graph capture: a replay would repeat one step number (its bias corrections and rounding thresholds)")
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            by_step = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                if not (p.is_cuda and p.dtype in (torch.float32, torch.bfloat16) and p.is_contiguous()):
                    raise N.MtlError("HipAdam needs contiguous fp32 (or, with setup.dtype = \"bf16\", bf16) parameters on the GPU (no CPU fallback)")
                st = self.state[p]
                if not st:
                    st["step"] = 0
                self._to_width(st, p)
                st["step"] = int(st["step"]) + 1
                by_step.setdefault(st["step"], []).append(p)
            batches = []
            for step, ps in by_step.items():
                late = [p for p in ps if id(p) in self._late]
                batches.append((step, [p for p in ps if id(p) not in self._late], False))
                if late:
                    batches.append((step, late, True))
            for step, ps, deferred in batches:
                if not ps:
                    continue
                if deferred:
                    self._side.wait_stream(torch.cuda.current_stream())       # after the backward / all-reduce that produced the gradients
                    with torch.cuda.stream(self._side):
                        self._launch(group, step, ps)
                        self._late_done = torch.cuda.Event()
                        self._late_done.record(self._side)
                    for p in ps:
                        if p.grad is not None:
                            p.grad.record_stream(self._side)                      # zero_grad() may release it while the side stream still reads it
                else:
                    self._launch(group, step, ps)
        return loss

    def _launch(self, group, step, ps):
        """one mtl_adam_step / mtl_adam8_step launch (all tensors of `ps`, which share `step`) on the current stream"""
        if self.state_bits == 8:
            grads = [p.grad if p.grad.dtype == p.dtype and p.grad.is_contiguous() else p.grad.to(p.dtype).contiguous() for p in ps]
            adam8_step(ps, grads, [Adam8State(*(self.state[p][k] for k in _STATE8)) for p in ps], step, group["lr"], group["betas"], group["eps"], group["weight_decay"],
                       group["decoupled_weight_decay"], [self._shadows.get(id(p)) for p in ps], "threshold")
            return
        arr = (N.AdamTensor * len(ps))()
        keep = []
        for i, p in enumerate(ps):
            st = self.state[p]
            for k in ("exp_avg", "exp_avg_sq"):
                m = st[k]
                if not (m.is_cuda and m.dtype == torch.float32 and m.is_contiguous() and m.numel() == p.numel()):
                    raise N.MtlError(f"HipAdam: state['{k}'] must be a contiguous fp32 GPU tensor of the parameter's size (got {m.dtype}, {tuple(m.shape)})")
            g = p.grad
            if g.dtype != p.dtype or not g.is_contiguous():
                g = g.to(p.dtype).contiguous()
            keep.append(g)
            sh = self._shadows.get(id(p))
            arr[i].p, arr[i].g, arr[i].m, arr[i].v = p.data_ptr(), g.data_ptr(), st["exp_avg"].data_ptr(), st["exp_avg_sq"].data_ptr()
            arr[i].n = p.numel()
            arr[i].param_dtype = N.MTL_BF16 if p.dtype == torch.bfloat16 else N.MTL_F32
            if sh is not None:
                arr[i].shadow, arr[i].cols, arr[i].ld_shadow = sh.tensor.data_ptr(), p.shape[1], sh.tensor.stride(0)
            else:
                arr[i].shadow, arr[i].cols, arr[i].ld_shadow = None, 0, 0
        b1, b2 = group["betas"]
        N.check(N.lib().mtl_adam_step(arr, len(ps), float(group["lr"]), float(b1), float(b2), float(group["eps"]),
                                      float(group["weight_decay"]), 1 if group["decoupled_weight_decay"] else 0,
                                      int(step), N.stream()), "mtl_adam_step")
        for p in ps:   # the kernel wrote through raw pointers: bump the autograd version like an in-place op
            torch.autograd.graph.increment_version(p)
            sh = self._shadows.get(id(p))
            if sh is not None:
                sh.version = p._version
