"""Operators of a training step around a language model, as cases that can be timed and compared.

Three operators:

  embed_fwd / embed_train   rows of a (trainable) token table, scaled, and the table's gradient summed token by token
  qk_fwd / qk_train         RMS norm of every query and key head with the rotary position embedding in the same pass, and its backward pass
  adam8                     one Adam / AdamW step of several tensors whose moments are held in 8 bits

`run` computes them in elementary torch operations, or with this repository's kernels where `own` is true. `exact` computes them in 64 bits.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}

# ---------------------------------------------------------------------------------------------------------------- the cases


def listed():
    return [
        # the text prompt of one sample, looked up in a GPT-2-sized table: latency
        {"name": "embed_prompt", "op": "embed_fwd", "B": 1, "T": 133, "V": 50257, "d": 768, "table": "f32", "out": "f32", "scaled": False, "pad": 0.0},
        # a training step over B x T = 8192 tokens with a GPT-2-sized table, a quarter of them left padding
        {"name": "embed_train_50257x768", "op": "embed_train", "B": 32, "T": 256, "V": 50257, "d": 768, "table": "f32", "out": "bf16", "scaled": True, "pad": 0.25},
        # the same with a Llama-3-sized vocabulary: the dense gradient is 2.1 GB
        {"name": "embed_train_128256x4096", "op": "embed_train", "B": 8, "T": 1024, "V": 128256, "d": 4096, "table": "f32", "out": "f32", "scaled": False, "pad": 0.1},
        # many tokens on a small vocabulary (Llama-2's 32000), bf16 model: long runs of equal tokens, ragged count
        {"name": "embed_train_200003_tokens", "op": "embed_train", "B": 1, "T": 200003, "V": 32000, "d": 1024, "table": "bf16", "out": "bf16", "scaled": True, "pad": 0.0},
        # one new token of 32 sequences, each at its own position (grouped heads as in Llama-3-8B)
        {"name": "qk_one_token", "op": "qk_fwd", "B": 32, "T": 1, "Hq": 32, "Hkv": 8, "D": 128, "R": 128, "type": "bf16", "positions": True},
        # forward of B = 32 windows of 257 rows at Llama-2-7B's heads
        {"name": "qk_fwd_32x257", "op": "qk_fwd", "B": 32, "T": 257, "Hq": 32, "Hkv": 32, "D": 128, "R": 128, "type": "bf16", "positions": False},
        # a training step of the long interleaved sequences (T = 1664), grouped heads
        {"name": "qk_train_4x1664", "op": "qk_train", "B": 4, "T": 1664, "Hq": 32, "Hkv": 8, "D": 128, "R": 128, "type": "bf16", "positions": False},
        # a small fp32 model with an odd head width of which only a part is rotated, packed sequences
        {"name": "qk_train_f32_odd", "op": "qk_train", "B": 3, "T": 517, "Hq": 12, "Hkv": 12, "D": 80, "R": 32, "type": "f32", "positions": True},
        # the few small tensors of a fine-tuned tail: latency
        {"name": "adam8_small", "op": "adam8", "shapes": "32x16x3,1024x32,1024,128x768,128", "type": "f32", "wd": 0.0, "decoupled": False},
        # every trainable tensor of the B = 32, L = 1024, C = 12 forecasting workload on a GPT-2-sized backbone
        {"name": "adam8_forecasting", "op": "adam8", "shapes": "1024x50257,1024,32x16x3,1024x384,1024,1024x768,1024,1024x768,1024,768x1024,768,128x768,128,1152x16384,1152",
         "type": "f32", "wd": 0.01, "decoupled": True},
        # a model held in bf16
        {"name": "adam8_bf16", "op": "adam8", "shapes": "1024x50257,1024,128x4096,128,4096x1024,4096", "type": "bf16", "wd": 0.0, "decoupled": False},
        # a trainable vocabulary of 100 000 rows at Llama width
        {"name": "adam8_100000x4096", "op": "adam8", "shapes": "100000x4096,1024x100000,1024", "type": "f32", "wd": 0.0, "decoupled": False},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["embed_fwd", "embed_train", "embed_train", "qk_fwd", "qk_train", "adam8", "adam8"])
    if op.startswith("embed"):
        V, d = _log(rng, 64, 128256), _log(rng, 16, 4096)
        n = min(_log(rng, 1, 200003), 200003 * 1024 // d)
        B = rng.choice([1, 2, 3, 8, 32])
        return {"op": op, "B": B, "T": max(1, n // B), "V": V, "d": d, "table": rng.choice(["f32", "bf16"]), "out": rng.choice(["f32", "bf16"]),
                "scaled": rng.random() < 0.5, "pad": rng.choice([0.0, 0.0, 0.1, 0.5])}
    if op.startswith("qk"):
        Hkv = rng.choice([1, 2, 4, 8, 12, 32])
        Hq = Hkv * rng.choice([1, 1, 4]) if Hkv < 12 else Hkv
        D = rng.choice([64, 128, 128, 256, 2 * rng.randint(8, 128)])
        R = D if rng.random() < 0.7 else 2 * rng.randint(1, D // 2)
        rows = min(_log(rng, 1, 8224), 8224 * 96 * 128 // ((Hq + 2 * Hkv) * D))
        B = rng.choice([1, 2, 3, 8, 32])
        return {"op": op, "B": B, "T": max(1, rows // B), "Hq": Hq, "Hkv": Hkv, "D": D, "R": R, "type": rng.choice(["f32", "bf16", "bf16"]), "positions": rng.random() < 0.5}
    left, shapes = 400_000_000, []
    for _ in range(rng.randint(1, 12)):
        rows, cols = _log(rng, 1, 8192), _log(rng, 1, 20000)
        if rows * cols <= left:
            left -= rows * cols
            shapes.append("%dx%d" % (rows, cols))
    return {"op": op, "shapes": ",".join(shapes or ["%dx%d" % (rng.randint(1, 99), rng.randint(1, 99))]), "type": rng.choice(["f32", "f32", "bf16"]), "wd": rng.choice([0.0, 0.01]),
            "decoupled": rng.random() < 0.5}


def _shapes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split(",")]


# ---------------------------------------------------------------------------------------------------------------- inputs


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 13)

    def normal(*shape, dtype=torch.float32, std=1.0):
        return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)

    s = {"case": case}
    if case["op"].startswith("embed"):
        B, T, V, d = case["B"], case["T"], case["V"], case["d"]
        # text: the k-th most frequent of V tokens is drawn with a probability that falls like 1 / k; frequent ones are spread over the table
        u = torch.rand(B, T, generator=g, device=DEV, dtype=torch.float64)
        rank = (torch.exp(u * math.log(V + 1.0)) - 1.0).long().clamp_(0, V - 1)
        ids = (rank * 1000003 + 11) % V
        s["pad_id"] = None
        if case["pad"]:
            s["pad_id"] = V // 3
            length = (torch.rand(B, 1, generator=g, device=DEV) * 2 * case["pad"] * T).long()
            ids = torch.where(torch.arange(T, device=DEV)[None, :] < length, s["pad_id"], ids)
        s["ids"] = ids
        s["scale"] = math.sqrt(d) if case["scaled"] else 1.0
        s["table"] = normal(V, d, dtype=TYPES[case["table"]], std=0.02)
        if case["op"] == "embed_train":
            s["table"].requires_grad_(True)
            s["dout"] = normal(B, T, d, dtype=TYPES[case["out"]])
    elif case["op"].startswith("qk"):
        B, T, Hq, Hkv, D, R, dt = (case[k] for k in ("B", "T", "Hq", "Hkv", "D", "R", "type"))
        dt = TYPES[dt]
        P = max(2048, T)
        inv = 10000.0 ** (-torch.arange(0, R, 2, device=DEV, dtype=torch.float64) / R)
        a = torch.arange(P, device=DEV, dtype=torch.float64)[:, None] * inv[None, :]
        a = torch.cat([a, a], dim=1)
        s["cos"], s["sin"] = a.cos().float(), a.sin().float()
        qkv = normal(B, T, (Hq + 2 * Hkv) * D, dtype=dt)                 # the fused projection's output: queries and keys are read in place
        s["q"], s["k"] = qkv[..., :Hq * D], qkv[..., Hq * D:(Hq + Hkv) * D]
        s["wq"], s["wk"] = 1 + normal(D, std=0.1), 1 + normal(D, std=0.1)
        s["positions"] = torch.randint(0, P, (B, T), generator=g, device=DEV) if case["positions"] else None
        s["eps"] = 1e-6
        if case["op"] == "qk_train":
            s["dq"], s["dk"] = normal(B, T, Hq * D, dtype=dt), normal(B, T, Hkv * D, dtype=dt)
            for n in ("q", "k", "wq", "wk"):
                s[n].requires_grad_(True)
    else:
        dt = TYPES[case["type"]]
        s["p"] = [normal(*sh, dtype=dt, std=0.02) for sh in _shapes(case)]
        s["g"] = [normal(*sh, dtype=dt, std=1e-3) for sh in _shapes(case)]
        s["step"] = 100
        s["state"] = []                                                   # (codes of the first moment, codes of the second's root, exponents)
        for p in s["p"]:
            m, r = normal(p.numel(), std=3e-4), normal(p.numel(), std=1e-3).abs_()
            s["state"].append(tuple(t.view(sh) for t, sh in zip(_encode(m, r, 100), (p.shape, p.shape, (-1, 2)))))
            del m, r
        s["hyper"] = {"lr": 1e-3, "beta1": 0.9, "beta2": 0.999, "eps": 1e-8, "wd": case["wd"], "decoupled": case["decoupled"]}
    return s


# ---------------------------------------------------------------------------------------------------------------- the plain forms


def _embed(s):
    c = s["case"]
    return (s["table"].detach()[s["ids"]].float() * s["scale"]).to(TYPES[c["out"]])


def _embed_grad(s):
    ids, dout, table = s["ids"].reshape(-1), s["dout"].reshape(-1, s["dout"].shape[-1]).float(), s["table"].detach()
    if s["pad_id"] is not None:
        dout = torch.where((ids == s["pad_id"])[:, None], 0.0, dout)
    grad = torch.zeros(table.shape, device=table.device).index_add_(0, ids, dout)
    return (grad * s["scale"]).to(table.dtype)


def _norm_rotate(x, w, cos, sin, D, R, eps):
    """[B, T, H D] -> rotate(w x / rms(x)) of every head"""
    h = x.float().unflatten(-1, (-1, D))
    n = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + eps) * w
    a, b, rest = n[..., :R // 2], n[..., R // 2:R], n[..., R:]
    c, z = cos[:, :, None, :R // 2], sin[:, :, None, :R // 2]
    return torch.cat([a * c - b * z, b * c + a * z, rest], dim=-1).flatten(-2).to(x.dtype)


def _norm_rotate_grad(dy, x, w, cos, sin, D, R, eps):
    h, g = x.float().unflatten(-1, (-1, D)), dy.float().unflatten(-1, (-1, D))
    c, z = cos[:, :, None, :R // 2], sin[:, :, None, :R // 2]
    a, b, rest = g[..., :R // 2], g[..., R // 2:R], g[..., R:]
    u = torch.cat([a * c + b * z, b * c - a * z, rest], dim=-1)
    r = torch.rsqrt((h * h).mean(-1, keepdim=True) + eps)
    n = h * r
    dn = u * w
    dx = r * (dn - n * (dn * n).mean(-1, keepdim=True))
    return dx.flatten(-2).to(x.dtype), (u * n).sum(dim=(0, 1, 2))


# Moments in 8 bits, in blocks of 64 consecutive elements with two power-of-two scales: the first moment as e4m3 numbers, rounded to nearest, the ROOT of the second as unsigned
# numbers of 4 exponent and 4 mantissa bits (0, 1 .. 15, then (16 + f) 2^(e-1)), rounded up or down by a threshold that runs through the unit interval with the step.
BLOCK = 64


def _root_values(device):
    c = torch.arange(256, device=device)
    e, f = c >> 4, c & 15
    v = torch.where(e == 0, f, (16 + f) << (e - 1).clamp(min=0)).float()
    v[255] = math.nan
    return v


def _pow2(e):
    return ((e.int() + 127) << 23).view(torch.float32)


def _exponents(x, below):
    """floor(log2 of each block's largest finite value) - below, in [-126, 126]"""
    top = torch.where(x.isfinite(), x, 0.0).view(-1, BLOCK).amax(1)
    return ((top.view(torch.int32) >> 23) - 127 - below).clamp(-126, 126)


def _threshold(n, step, device):
    return (torch.arange(n, device=device, dtype=torch.int64) * 0xC13FA9A9 + step * 0x91E10DA5) & 0xFFFFFFFF


def _encode(m, r, step):
    n = m.numel()
    pad = -n % BLOCK
    if pad:
        m, r = (torch.cat([t, t.new_zeros(pad)]) for t in (m, r))
    em, er = _exponents(m.abs(), 7), _exponents(r, 17)
    cm = (m.view(-1, BLOCK) * _pow2(-em)[:, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    cm = torch.where(m.isfinite().view(-1, BLOCK), cm, 0x7F).view(-1)[:n]
    y = (r.view(-1, BLOCK) * _pow2(-er)[:, None]).view(-1)
    u = _threshold(m.numel(), step, m.device)
    large = (((y.view(torch.int32) + (u >> 13).int()) >> 19) - 130 * 16)
    small = torch.floor(y + (u >> 8).float() * 2.0 ** -24).nan_to_num(0.0).int()
    cr = torch.where(y >= 16, large, small)
    cr = torch.where((r > 0) & (cr < 1), 1, cr)
    cr = torch.where(r.isfinite(), cr, 255)[:n].to(torch.uint8)
    return cm, cr, torch.stack([em, er], dim=1).to(torch.int8).view(torch.uint8).view(-1)


def _decode(state, n):
    cm, cr, ex = (t.reshape(-1) for t in state)
    ex = ex.view(torch.int8).view(-1, 2)
    at = torch.arange(n, device=cm.device) // BLOCK
    m = cm.view(torch.float8_e4m3fn).float() * _pow2(ex[:, 0])[at]
    r = _root_values(cm.device)[cr.int()] * _pow2(ex[:, 1])[at]
    return m, r


def _adam8_one(p, g, state, step, h):
    n = p.numel()
    m, r = _decode(state, n)
    v = r * r
    w, g = p.detach().reshape(-1).float(), g.reshape(-1).float()
    if h["wd"] and h["decoupled"]:
        w = w * (1.0 - h["lr"] * h["wd"])
    elif h["wd"]:
        g = g + w * h["wd"]
    m = m + (g - m) * (1.0 - h["beta1"])
    v = v * h["beta2"] + (g * g) * (1.0 - h["beta2"])
    r = torch.sqrt(v)
    denom = r * (1.0 / math.sqrt(1.0 - h["beta2"] ** step)) + h["eps"]
    w = w - (m / denom) * (h["lr"] / (1.0 - h["beta1"] ** step))
    new = _encode(m, r, step)
    p.copy_(w.view(p.shape))
    for t, x in zip(state, new):
        t.copy_(x.view(t.shape))
    m, r = _decode(state, n)
    return p, m.view(p.shape).to(torch.bfloat16), (r * r).view(p.shape).to(torch.bfloat16)


def run(s):
    c = s["case"]
    if own:
        return _run_own(s)
    if c["op"] == "embed_fwd":
        return _embed(s)
    if c["op"] == "embed_train":
        return {"out": _embed(s), "grad": _embed_grad(s)}
    if c["op"].startswith("qk"):
        with torch.no_grad():
            at = torch.arange(c["T"], device=s["q"].device).expand(c["B"], -1) if s["positions"] is None else s["positions"]
            cos, sin = s["cos"][at], s["sin"][at]
            q = _norm_rotate(s["q"], s["wq"], cos, sin, c["D"], c["R"], s["eps"])
            k = _norm_rotate(s["k"], s["wk"], cos, sin, c["D"], c["R"], s["eps"])
            if c["op"] == "qk_fwd":
                return {"q": q, "k": k}
            dq, dwq = _norm_rotate_grad(s["dq"], s["q"], s["wq"], cos, sin, c["D"], c["R"], s["eps"])
            dk, dwk = _norm_rotate_grad(s["dk"], s["k"], s["wk"], cos, sin, c["D"], c["R"], s["eps"])
            return {"q": q, "k": k, "dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}
    s["step"] += 1
    got = [_adam8_one(p, g, st, s["step"], s["hyper"]) for p, g, st in zip(s["p"], s["g"], s["state"])]
    return {"p": [x[0] for x in got], "m": [x[1] for x in got], "v": [x[2] for x in got]}


def _run_own(s):
    from med_ts_llm_amd.hip import ops, optim
    c = s["case"]
    if c["op"] == "embed_fwd":
        return ops.embedding_fwd(s["ids"], s["table"], scale=s["scale"], out_dtype=TYPES[c["out"]])
    if c["op"] == "embed_train":
        out = ops.EmbeddingFn.apply(s["ids"], s["table"], s["scale"], s["pad_id"], TYPES[c["out"]])
        (grad,) = torch.autograd.grad(out, s["table"], s["dout"])
        return {"out": out.detach(), "grad": grad}
    if c["op"] == "qk_fwd":
        q, k = ops.qk_norm_rope_fwd(s["q"], s["k"], s["wq"], s["wk"], s["cos"], s["sin"], c["Hq"], c["Hkv"], c["D"], eps=s["eps"], positions=s["positions"])
        return {"q": q, "k": k}
    if c["op"] == "qk_train":
        q, k = ops.QkNormRopeFn.apply(s["q"], s["k"], s["wq"], s["wk"], s["cos"], s["sin"], c["Hq"], c["Hkv"], c["D"], s["eps"], s["positions"])
        dq, dk, dwq, dwk = torch.autograd.grad((q, k), (s["q"], s["k"], s["wq"], s["wk"]), (s["dq"], s["dk"]))
        return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}
    s["step"] += 1
    h = s["hyper"]
    states = [optim.Adam8State(*st) for st in s["state"]]
    optim.adam8_step(s["p"], s["g"], states, s["step"], lr=h["lr"], betas=(h["beta1"], h["beta2"]), eps=h["eps"], weight_decay=h["wd"], decoupled_weight_decay=h["decoupled"])
    mv = optim.adam8_moments(states, dtype=torch.bfloat16)
    return {"p": s["p"], "m": [x[0] for x in mv], "v": [x[1] for x in mv]}


# ---------------------------------------------------------------------------------------------------------------- what a pass cannot do without


def work(case):
    size = {"f32": 4, "bf16": 2}
    if case["op"].startswith("embed"):
        n, V, d = case["B"] * case["T"], case["V"], case["d"]
        k = np.arange(1, V + 1, dtype=np.float64)
        seen = float(np.sum(-np.expm1(n * np.log1p(-np.minimum(np.log1p(1 / k) / math.log(V + 1.0), 1 - 1e-12)))))      # distinct tokens among n
        moved = n * 8 + seen * d * size[case["table"]] + n * d * size[case["out"]]
        if case["op"] == "embed_train":
            moved += n * 8 + n * d * size[case["out"]] * (1 - case["pad"]) + V * d * size[case["table"]]
        return {"bytes": moved, "flops": n * d * (2 if case["op"] == "embed_train" else 1)}
    if case["op"].startswith("qk"):
        rows, e = case["B"] * case["T"], size[case["type"]]
        n = rows * (case["Hq"] + case["Hkv"]) * case["D"]
        tables = (rows if case["positions"] else case["T"]) * case["R"] * 4 + case["D"] * 8 + (rows * 8 if case["positions"] else 0)
        if case["op"] == "qk_fwd":
            return {"bytes": 2 * n * e + tables, "flops": 8 * n}
        return {"bytes": 5 * n * e + 2 * tables, "flops": 8 * n + 16 * n}        # x, y; then x again, dy, dx
    n, e = sum(math.prod(sh) for sh in _shapes(case)), size[case["type"]]
    return {"bytes": n * (3 * e + 4 + 4 + 4 / BLOCK), "flops": 30 * n}             # p and the codes read and written, g read; the moments' values written


# ---------------------------------------------------------------------------------------------------------------- the definitions in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    f8 = torch.float64
    with torch.no_grad():
        if case["op"].startswith("embed"):
            table = s["table"].to(f8)
            out = table.index_select(0, s["ids"].reshape(-1)).view(*s["ids"].shape, -1).mul_(s["scale"])
            if case["op"] == "embed_fwd":
                return out
            del table
            ids = s["ids"].reshape(-1)
            keep = torch.ones_like(ids, dtype=torch.bool) if s["pad_id"] is None else ids != s["pad_id"]
            grad = torch.zeros(case["V"], case["d"], dtype=f8, device=ids.device)
            grad.index_add_(0, ids[keep], s["dout"].reshape(-1, case["d"])[keep].to(f8), alpha=s["scale"])
            return {"out": out, "grad": grad}
    if case["op"].startswith("qk"):
        return _exact_qk(s)
    return _exact_adam8(s)


def _exact_qk(s):
    c = s["case"]
    f8, R, D = torch.float64, c["R"], c["D"]
    train = c["op"] == "qk_train"
    x = {n: s[n].detach().to(torch.float64).requires_grad_(train) for n in ("q", "k", "wq", "wk")}
    rows = torch.arange(c["T"], device=s["cos"].device).repeat(c["B"], 1) if s["positions"] is None else s["positions"]
    turn = torch.complex(s["cos"][:, :R // 2].to(f8), s["sin"][:, :R // 2].to(f8))[rows][:, :, None, :]       # e^(i angle) of every pair

    def one(t, w):
        t = t.reshape(c["B"], c["T"], -1, D)
        t = t / t.pow(2).mean(-1, keepdim=True).add(s["eps"]).sqrt() * w
        z = torch.complex(t[..., :R // 2], t[..., R // 2:R]) * turn
        return torch.cat((z.real, z.imag, t[..., R:]), -1).reshape(c["B"], c["T"], -1)

    q, k = one(x["q"], x["wq"]), one(x["k"], x["wk"])
    if not train:
        return {"q": q, "k": k}
    dq, dk, dwq, dwk = torch.autograd.grad((q, k), (x["q"], x["k"], x["wq"], x["wk"]), (s["dq"].to(f8), s["dk"].to(f8)))
    return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}


def _exact_adam8(s):
    f8, h, t = torch.float64, s["hyper"], s["step"] + 1
    out = {"p": [], "m": [], "v": []}
    for p, g, (cm, cr, ex) in zip(s["p"], s["g"], s["state"]):
        n = p.numel()
        ex = ex.view(torch.int8).view(-1, 2).to(f8).repeat_interleave(BLOCK, 0)[:n]
        code = cr.reshape(-1).to(f8)
        e = torch.floor(code / 16)
        root = torch.where(e < 1, code, (16 + code - 16 * e) * torch.exp2(e - 1)) * torch.exp2(ex[:, 1])
        del e, code
        m = cm.reshape(-1).view(torch.float8_e4m3fn).to(f8) * torch.exp2(ex[:, 0])
        w, d = p.reshape(-1).to(f8), g.reshape(-1).to(f8)
        if h["wd"]:
            w, d = (w * (1 - h["lr"] * h["wd"]), d) if h["decoupled"] else (w, d + h["wd"] * w)
        m = h["beta1"] * m + (1 - h["beta1"]) * d
        root = torch.sqrt(h["beta2"] * root ** 2 + (1 - h["beta2"]) * d ** 2)
        w = w - h["lr"] / (1 - h["beta1"] ** t) * m / (root / math.sqrt(1 - h["beta2"] ** t) + h["eps"])
        out["p"].append(w.view(p.shape))
        del d, ex

        def scale(x, below):
            top = torch.nn.functional.pad(x.abs(), (0, -n % BLOCK)).view(-1, BLOCK).amax(1).clamp(min=2.0 ** -200)
            return torch.exp2((torch.floor(torch.log2(top)) - below).clamp(-126, 126)).repeat_interleave(BLOCK)[:n]

        a = scale(m, 7)
        x = m / a
        step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
        out["m"].append((torch.round(x / step) * step * a).view(p.shape))
        del x, step, m
        a = scale(root, 17)
        x = root / a
        u = ((torch.arange(n, device=x.device) * 0xC13FA9A9 + t * 0x91E10DA5) % 2 ** 32).to(f8)
        u = torch.where(x >= 16, torch.floor(u / 2 ** 13) / 2 ** 19, torch.floor(u / 2 ** 8) / 2 ** 24)
        step = torch.exp2(torch.floor(torch.log2(x.clamp(min=16.0))) - 4)
        x = torch.floor(x / step + u) * step
        x = torch.where(root > 0, x.clamp(min=1.0), x) * a
        out["v"].append((x * x).view(p.shape))
    return out
