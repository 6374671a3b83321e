"""The 8-bit floating point operators, as cases that can be timed and compared.

Four operators of a prompt's or a decode step's projections in e4m3 with one f32
scale for each 128 columns (activations, per row) or 128 x 128 block (weights):

  norm    residual += x, RMS norm, quantise          fp8.add_rms_norm_fp8
  act     silu(gate) * up, quantise                  fp8.swiglu_fp8
  matmul  y = dequant(a) . dequant(W)^T              fp8.Fp8Weight.matmul
  ffn     norm, gate / up product, act, down product fp8.Fp8SwigluBlock

With G = 128, F = 448 (the largest e4m3 number) and TINY = 2^-100:

  quantise(z):  g = max(max |z| over the group, TINY), scale = g / F, q = e4m3(z * F / g)
  norm:         h = x + residual rounded to the residual's type, r = 1 / sqrt(mean h^2 + eps),
                z = h * w, scale = g * r / F, q = e4m3(z * F / g)
"""
import math

import torch

own = False

G, F, TINY, EPS = 128, 448.0, 2.0**-100, 1e-5
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one token of an 8B-wide decoder: only latency counts
        {"name": "norm one token", "op": "norm", "m": 1, "k": 4096, "dtype": "f32", "residual": True},
        # a small batch at a width that ends inside a group and inside a 16-byte piece
        {"name": "norm ragged", "op": "norm", "m": 77, "k": 1003, "dtype": "f16", "residual": False},
        # 8 prompts of 2048 tokens at a 70B width: only bandwidth counts
        {"name": "norm prompts", "op": "norm", "m": 16384, "k": 8192, "dtype": "bf16", "residual": True},
        # 16 sequences decoded together, 8B feed-forward width
        {"name": "act decode batch", "op": "act", "m": 16, "k": 14336, "dtype": "f32"},
        # a 2048-token prompt, 70B feed-forward width
        {"name": "act prompt", "op": "act", "m": 2048, "k": 28672, "dtype": "bf16"},
        # one token through an attention projection of the 8B width
        {"name": "matmul one token", "op": "matmul", "m": 1, "n": 4096, "k": 4096, "dtype": "f32"},
        # the vocabulary's logits of 16 sequences
        {"name": "matmul logits", "op": "matmul", "m": 16, "n": 128256, "k": 4096, "dtype": "f32"},
        # every size odd, a few dozen tokens
        {"name": "matmul ragged", "op": "matmul", "m": 77, "n": 1003, "k": 1001, "dtype": "f16"},
        # a 512-token chunk through the 8B up projection
        {"name": "matmul chunk", "op": "matmul", "m": 512, "n": 14336, "k": 4096, "dtype": "bf16"},
        # a 2048-token prompt through the 70B up projection
        {"name": "matmul prompt", "op": "matmul", "m": 2048, "n": 28672, "k": 8192, "dtype": "bf16"},
        # one token through the whole 8B feed-forward block
        {"name": "ffn one token", "op": "ffn", "m": 1, "k": 4096, "n_ff": 14336, "dtype": "bf16"},
        # a 2048-token prompt through it
        {"name": "ffn prompt", "op": "ffn", "m": 2048, "k": 4096, "n_ff": 14336, "dtype": "bf16"},
    ]


def draw(rng):
    def size(lo, hi):
        return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))

    op = rng.choice(["norm", "act", "matmul", "matmul", "matmul", "ffn"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "norm":
        return {"op": op, "m": size(1, 16384), "k": size(32, 8192), "dtype": dtype,
                "residual": rng.random() < 0.7} if dtype != "f32" else {
            "op": op, "m": size(1, 8192), "k": size(32, 8192), "dtype": dtype, "residual": rng.random() < 0.7}
    if op == "act":
        return {"op": op, "m": size(1, 1024 if dtype == "f32" else 2048), "k": size(32, 28672), "dtype": dtype}
    if op == "matmul":
        return {"op": op, "m": size(1, 2048), "n": size(64, 28672), "k": size(32, 8192), "dtype": dtype}
    return {"op": op, "m": size(1, 2048), "k": size(128, 4096), "n_ff": size(128, 14336),
            "dtype": rng.choice(["f16", "bf16"])}


# ---- inputs ------------------------------------------------------------------------


def _groups(k):
    return (k + G - 1) // G


def _activations(m, k, gen, dtype):
    """Normal rows with a few channels an order of magnitude larger, as hidden states have."""
    x = torch.randn(m, k, generator=gen, device="cuda")
    x *= 1.0 + 15.0 * (torch.rand(k, generator=gen, device="cuda") < 0.01)
    return x.to(dtype)


def _weight(n, k, gen):
    """e4m3 blocks [n][k] and their scales [n / 128][k / 128] of a matrix whose blocks differ in size."""
    nb, kb = _groups(n), _groups(k)
    w = torch.empty(nb * G, kb * G, dtype=torch.bfloat16, device="cuda").normal_(generator=gen)
    w = w.view(nb, G, kb, G)
    s = w.abs().amax(dim=(1, 3)).float() / F
    q = (w / s.to(w.dtype)[:, None, :, None]).clamp_(-F, F).to(torch.float8_e4m3fn)
    s *= 0.02 * (0.5 + torch.rand(nb, kb, generator=gen, device="cuda"))
    return q.view(nb * G, kb * G)[:n, :k].contiguous(), s


def _rows16(m, k):
    """[m][k] e4m3 whose rows start at multiples of 16 bytes."""
    return torch.zeros(m, (k + 15) // 16 * 16, dtype=torch.float8_e4m3fn, device="cuda")[:, :k]


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    op, m, k, dtype = case["op"], case["m"], case["k"], DTYPES[case["dtype"]]
    s = {"op": op, "m": m, "k": k, "dtype": dtype}
    if op in ("norm", "ffn"):
        s["x"] = _activations(m, k, gen, dtype)
        s["residual"] = _activations(m, k, gen, dtype) if case.get("residual", True) else None
        s["w"] = (1.0 + 0.1 * torch.randn(k, generator=gen, device="cuda")).half()
    if op == "act":
        gate_up = torch.randn(m, 2 * k, generator=gen, device="cuda").to(dtype)
        s["gate"], s["up"] = gate_up[:, :k], gate_up[:, k:]
    if op == "matmul":
        z = torch.nn.functional.pad(_activations(m, k, gen, torch.float32), (0, -k % G)).view(m, -1, G)
        g = z.abs().amax(2).clamp_(min=TINY)
        s["a"], s["a_scale"] = _rows16(m, k), g / F
        s["a"].copy_((z * (F / g)[:, :, None]).view(m, -1)[:, :k].to(torch.float8_e4m3fn))
        w = _weight(case["n"], k, gen)
    if op == "ffn":
        n = case["n_ff"]
        w = (*_weight(n, k, gen), *_weight(n, k, gen), *_weight(k, n, gen))
    if own:
        from agent_harness_b200 import fp8

        if op in ("norm", "act"):
            s["q"], s["scale"] = fp8.alloc(m, k, "cuda")
        if op == "matmul":
            s["weight"] = fp8.Fp8Weight.from_blocks(*w)
            s["y"] = torch.empty(m, case["n"], dtype=dtype, device="cuda")
        if op == "ffn":
            s["block"] = fp8.Fp8SwigluBlock.from_blocks(*w)
            s["y"] = torch.empty(m, k, dtype=dtype, device="cuda")
    elif op in ("matmul", "ffn"):
        s["weight"] = w
    return s


# ---- the plain forms ---------------------------------------------------------------


def _quantise(z):
    """(q, g): z [m][k] in e4m3 and the largest |z| of each group (at least TINY)."""
    m, k = z.shape
    z = torch.nn.functional.pad(z, (0, -k % G)).view(m, -1, G)
    g = z.abs().amax(2).clamp_(min=TINY)
    q = (z / (g / F)[:, :, None]).clamp_(-F, F).to(torch.float8_e4m3fn)
    return q.view(m, -1)[:, :k], g


def _norm(x, residual, w):
    h = x
    if residual is not None:
        residual.copy_(x.float() + residual.float())
        h = residual
    h = h.float()
    q, g = _quantise(h * w.float())
    return q, g * torch.rsqrt(h.square().mean(1, keepdim=True) + EPS) / F


def _act(gate, up):
    gate = gate.float()
    q, g = _quantise(gate / (1.0 + torch.exp(-gate)) * up.float())
    return q, g / F


def _spread(scale, rows, cols):
    """Each scale over its 128 columns (and 128 rows, where rows is given)."""
    scale = scale.repeat_interleave(G, 1)[:, :cols]
    return scale if rows is None else scale.repeat_interleave(G, 0)[:rows]


def _matmul(q, scale, wq, wscale):
    a = q.float() * _spread(scale, None, q.shape[1])
    return a @ (wq.float() * _spread(wscale, *wq.shape)).t()


def run(s):
    op = s["op"]
    if own:
        from agent_harness_b200 import fp8

        if op == "norm":
            fp8.add_rms_norm_fp8(s["x"], s["w"], residual=s["residual"], eps=EPS, out=s["q"], scales=s["scale"])
            return {"q": s["q"], "scale": s["scale"], **({} if s["residual"] is None else {"residual": s["residual"]})}
        if op == "act":
            fp8.swiglu_fp8(s["gate"], s["up"], out=s["q"], scales=s["scale"])
            return {"q": s["q"], "scale": s["scale"]}
        if op == "matmul":
            return s["weight"].matmul(s["a"], s["a_scale"], out=s["y"])
        y = s["block"](s["x"], s["w"], residual=s["residual"], eps=EPS, out=s["y"])
        return {"y": y, "residual": s["residual"]}
    if op == "norm":
        q, scale = _norm(s["x"], s["residual"], s["w"])
        return {"q": q, "scale": scale, **({} if s["residual"] is None else {"residual": s["residual"]})}
    if op == "act":
        q, scale = _act(s["gate"], s["up"])
        return {"q": q, "scale": scale}
    if op == "matmul":
        return _matmul(s["a"], s["a_scale"], *s["weight"]).to(s["dtype"])
    gq, gs, uq, us, dq, ds = s["weight"]
    a, a_scale = _norm(s["x"], s["residual"], s["w"])
    a, a_scale = _act(_matmul(a, a_scale, gq, gs), _matmul(a, a_scale, uq, us))
    return {"y": _matmul(a, a_scale, dq, ds).to(s["dtype"]), "residual": s["residual"]}


# ---- what a pass cannot do without ---------------------------------------------------


def work(case):
    op, m, k, e = case["op"], case["m"], case["k"], 4 if case["dtype"] == "f32" else 2
    quantised = m * k + 4 * m * _groups(k)
    if op == "norm":
        return {"bytes": m * k * e * (3 if case["residual"] else 1) + 2 * k + quantised, "flops": 7 * m * k}
    if op == "act":
        return {"bytes": 2 * m * k * e + quantised, "flops": 8 * m * k}
    if op == "matmul":
        n = case["n"]
        return {"bytes": quantised + n * k + 4 * _groups(n) * _groups(k) + m * n * e, "flops": 2 * m * n * k}
    n = case["n_ff"]
    return {"bytes": 4 * m * k * e + 2 * k + 3 * (n * k + 4 * _groups(n) * _groups(k)), "flops": 6 * m * n * k}


# ---- the definition in 64 bits -------------------------------------------------------


def _e4m3_exact(v):
    """v (64 bits) on the e4m3 grid: 3 mantissa bits down to 2^-6, steps of 2^-9 below, half to even."""
    e = torch.floor(torch.log2(v.abs().clamp(min=2.0**-20))).clamp(min=-6.0)
    step = torch.exp2(e - 3.0)
    return (torch.round(v / step) * step).clamp(-F, F)


def _groups_exact(z):
    m, k = z.shape
    padded = torch.zeros(m, _groups(k) * G, dtype=torch.float64, device=z.device)
    padded[:, :k] = z.abs()
    g = padded.view(m, _groups(k), G).max(dim=2).values.clamp(min=TINY)
    column = torch.arange(k, device=z.device) // G
    return _e4m3_exact(z * F / g[:, column]), g


def _norm_exact(x, residual, w):
    h = x.double() if residual is None else (x.double() + residual.double()).to(residual.dtype).double()
    q, g = _groups_exact(h * w.double()[None, :])
    return q, g / F / (h.pow(2).sum(1, keepdim=True) / h.shape[1] + EPS).sqrt(), h


def _act_exact(gate, up):
    q, g = _groups_exact(gate.double() * torch.sigmoid(gate.double()) * up.double())
    return q, g / F


def _matmul_exact(q, scale, wq, wscale):
    row, col = (torch.arange(n, device=wq.device) // G for n in wq.shape)
    w = wq.double()
    w *= wscale.double()[row][:, col]
    return (q.double() * scale.double()[:, col]) @ w.t()


def exact(case, seed):
    global own
    mine, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = mine
    op = s["op"]
    if op == "norm":
        q, scale, h = _norm_exact(s["x"], s["residual"], s["w"])
        return {"q": q, "scale": scale, **({} if s["residual"] is None else {"residual": h})}
    if op == "act":
        q, scale = _act_exact(s["gate"], s["up"])
        return {"q": q, "scale": scale}
    if op == "matmul":
        return _matmul_exact(s["a"], s["a_scale"], *s["weight"])
    gq, gs, uq, us, dq, ds = s["weight"]
    a, a_scale, h = _norm_exact(s["x"], s["residual"], s["w"])
    a, a_scale = _act_exact(_matmul_exact(a, a_scale, gq, gs), _matmul_exact(a, a_scale, uq, us))
    return {"y": _matmul_exact(a, a_scale, dq, ds), "residual": h}
