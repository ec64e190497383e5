"""Measured cases of the feed-forward operators: the gated block in 16 bits (forward and backward) and
the 8-bit integer products (rows quantised on the way in, a plain and a gated product).

    ffn_forward    y = (act(x Wg^T) * (x Wu^T)) Wd^T
    ffn_backward   dx, dWg, dWu, dWd of that block, from dy and the saved projections x Wg^T and x Wu^T
    int8_linear    q, s = rows of x in 8 bits;  y = act(s * sw * (q Wq^T) + bias)
    int8_gated     q, s = rows of x in 8 bits;  h = act(s * sg * (q Gq^T)) * (s * su * (q Uq^T))

``own`` chooses between the plain form of each (elementary torch operations in 32 bits) and the calls a
user makes of the package.  A case is a dict of plain values; see ``listed``.
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
#: Rows whose largest magnitude is below this count as zero when they are quantised.
_TINY = 2.0 ** -100


# ---- cases -------------------------------------------------------------------------------------

def listed():
    return [
        # one token of a decoding loop through a wide block: every weight is read once
        dict(name="ffn_fwd_decode_1", op="ffn_forward", tokens=1, d=4096, f=16384, dtype="bf16", act="silu"),
        # a small batch of decoding streams through a block of a few MB, where latency counts
        dict(name="ffn_fwd_decode_24", op="ffn_forward", tokens=24, d=1024, f=4096, dtype="fp16", act="gelu"),
        # the character model's training batch: 64 sequences of 128, width 256, four times that inside
        dict(name="ffn_fwd_char_lm", op="ffn_forward", tokens=8192, d=256, f=1024, dtype="bf16", act="silu"),
        # a long prompt, or a training batch, through the wide block
        dict(name="ffn_fwd_large", op="ffn_forward", tokens=8192, d=4096, f=16384, dtype="bf16", act="silu"),
        # the character model's training step
        dict(name="ffn_bwd_char_lm", op="ffn_backward", tokens=8192, d=256, f=1024, dtype="bf16", act="gelu"),
        # a short last batch of odd sizes
        dict(name="ffn_bwd_ragged", op="ffn_backward", tokens=333, d=520, f=1405, dtype="fp16", act="silu"),
        # the training step of the wide block
        dict(name="ffn_bwd_large", op="ffn_backward", tokens=8192, d=4096, f=16384, dtype="bf16", act="silu"),
        # one token of a decoding loop through the scaled linear layer, in 8 bits
        dict(name="int8_linear_decode_1", op="int8_linear", tokens=1, d=4096, n=16384, dtype="bf16", out="bf16",
             bias=False, act="none"),
        # the character model's query-key-value projection, 32-bit activations in and out
        dict(name="int8_linear_char_lm", op="int8_linear", tokens=8192, d=256, n=768, dtype="fp32", out="fp32",
             bias=True, act="none"),
        # the scaled linear layer with its bias and GELU over a long prompt
        dict(name="int8_linear_large", op="int8_linear", tokens=8192, d=4096, n=16384, dtype="bf16", out="bf16",
             bias=True, act="gelu"),
        # the first half of the quantised block for a ragged batch of decoding streams
        dict(name="int8_gated_ragged", op="int8_gated", tokens=57, d=4096, n=11009, dtype="fp16", out="fp16",
             bias=False, act="silu"),
        # the same half for a long prompt with one token over a whole tile
        dict(name="int8_gated_prompt", op="int8_gated", tokens=4097, d=4096, n=11008, dtype="bf16", out="bf16",
             bias=False, act="silu"),
    ]


def _size(rng, lo, hi):
    """Log-uniform in [lo, hi]; half of the draws are multiples of 64, the others as they come."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))
    v = min(max(v, lo), hi)
    if rng.random() < 0.5:
        v = min(hi, max(64, v // 64 * 64))
    return v


def draw(rng):
    op = rng.choice(["ffn_forward", "ffn_backward", "int8_linear", "int8_gated"])
    tokens = min(8192, max(1, int(round(math.exp(rng.uniform(0.0, math.log(8192.4)))))))
    c = dict(op=op, tokens=tokens, d=_size(rng, 64, 4096))
    if op.startswith("ffn"):
        c.update(f=_size(rng, 64, 16384), dtype=rng.choice(["bf16", "fp16"]),
                 act=rng.choice(["silu", "gelu", "relu", "none"]))
    else:
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        c.update(n=_size(rng, 64, 16384), dtype=dtype, out=dtype, bias=op == "int8_linear" and rng.random() < 0.5,
                 act=rng.choice(["silu", "gelu", "relu", "none"]))
    return c


# ---- inputs ------------------------------------------------------------------------------------

def _quantize_weight(w):
    """Weights are quantised once, when a model is loaded: rows of [out, in] by their largest magnitude."""
    top = w.abs().amax(dim=1)
    return torch.round(w * (127.0 / top)[:, None]).to(torch.int8), top / 127.0


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = _DTYPES[case["dtype"]]
    t, d = case["tokens"], case["d"]

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * std

    s = dict(case=dict(case))
    x = normal(t, d)
    if case["op"].startswith("ffn"):
        f = case["f"]
        s["x"] = x.to(dt)
        s["w_gate"] = normal(f, d, std=d ** -0.5).to(dt)
        s["w_up"] = normal(f, d, std=d ** -0.5).to(dt)
        s["w_down"] = normal(d, f, std=f ** -0.5).to(dt)
        if case["op"] == "ffn_backward":
            s["dy"] = normal(t, d, std=0.05).to(dt)
            # what the forward pass of the step saved, in the type it saves it in
            s["gate"] = (s["x"].float() @ s["w_gate"].float().t()).to(dt)
            s["up"] = (s["x"].float() @ s["w_up"].float().t()).to(dt)
        return s
    n = case["n"]
    # some channels of a model's activations are far larger than the rest
    x[:, torch.randint(0, d, (max(1, d // 128),), generator=g, device="cuda")] *= 8.0
    if t >= 32:
        x[-(t // 32):] = 0.0                 # the padding at the end of a batch
    s["x"] = x.to(dt)
    if case["op"] == "int8_linear":
        s["wq"], s["ws"] = _quantize_weight(normal(n, d, std=d ** -0.5))
        s["bias"] = normal(n, std=0.1) if case["bias"] else None
    else:
        s["gq"], s["gs"] = _quantize_weight(normal(n, d, std=d ** -0.5))
        s["uq"], s["us"] = _quantize_weight(normal(n, d, std=d ** -0.5))
    return s


# ---- the operators -----------------------------------------------------------------------------

def _act(x, act):
    if act == "silu":
        return x / (1.0 + torch.exp(-x))
    if act == "gelu":
        return 0.5 * x * (1.0 + torch.erf(x * math.sqrt(0.5)))
    if act == "relu":
        return torch.clamp(x, min=0.0)
    return x


def _act_grad(x, act):
    if act == "silu":
        p = 1.0 / (1.0 + torch.exp(-x))
        return p * (1.0 + x * (1.0 - p))
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(x * math.sqrt(0.5))) + x * torch.exp(-0.5 * x * x) * (1.0 / math.sqrt(2.0 * math.pi))
    if act == "relu":
        return (x > 0).to(x.dtype)
    return torch.ones_like(x)


def _quantize_rows(x):
    """Rows in 8 bits: scale = largest magnitude / 127, q = round to even of x * (127 / largest magnitude)."""
    x = x.float()
    top = x.abs().amax(dim=1)
    live = top >= _TINY
    full = torch.full_like(top, 127.0)            # tensor by tensor: torch turns a scalar divisor into a product
    q = torch.round(x * torch.where(live, full / top, 0.0)[:, None]).to(torch.int8)
    return q, torch.where(live, top / full, 0.0)


def _product(q, s, wq, ws):
    return (q.float() @ wq.float().t()) * (s[:, None] * ws[None, :])


def _plain(s):
    c = s["case"]
    act = c["act"]
    dt = _DTYPES[c["dtype"]]
    if c["op"].startswith("ffn"):
        wg, wu, wd = s["w_gate"].float(), s["w_up"].float(), s["w_down"].float()
        x = s["x"].float()
        if c["op"] == "ffn_forward":
            return ((_act(x @ wg.t(), act) * (x @ wu.t())) @ wd.t()).to(dt)
        gate, up, dy = s["gate"].float(), s["up"].float(), s["dy"].float()
        a = _act(gate, act)
        dh = dy @ wd
        dgate = dh * up * _act_grad(gate, act)
        dup = dh * a
        dx = dgate @ wg + dup @ wu
        return dx.to(dt), (dgate.t() @ x).to(dt), (dup.t() @ x).to(dt), (dy.t() @ (a * up)).to(dt)
    out = _DTYPES[c["out"]]
    q, scale = _quantize_rows(s["x"])
    if c["op"] == "int8_linear":
        y = _product(q, scale, s["wq"], s["ws"])
        if s["bias"] is not None:
            y = y + s["bias"]
        return q, scale, _act(y, act).to(out)
    gate = _product(q, scale, s["gq"], s["gs"])
    return q, scale, (_act(gate, act) * _product(q, scale, s["uq"], s["us"])).to(out)


def _framework(s):
    import fastnn_b200 as f
    c = s["case"]
    act = {"silu": f.ACT_SILU, "gelu": f.ACT_GELU, "relu": f.ACT_RELU, "none": f.ACT_NONE}[c["act"]]
    if c["op"] == "ffn_forward":
        return f.gated_ffn_forward(s["x"], s["w_gate"], s["w_up"], s["w_down"], act=act)
    if c["op"] == "ffn_backward":
        return f.gated_ffn_backward(s["dy"], s["x"], s["gate"], s["up"], s["w_gate"], s["w_up"], s["w_down"], act=act)
    out = _DTYPES[c["out"]]
    q, scale = f.quantize_rows(s["x"])
    if c["op"] == "int8_linear":
        return q, scale, f.int8_linear_forward(q, scale, s["wq"], s["ws"], bias=s["bias"], act=act, out_dtype=out)
    return q, scale, f.int8_gated_forward(q, scale, s["gq"], s["gs"], s["uq"], s["us"], act=act, out_dtype=out)


def run(state):
    return _framework(state) if own else _plain(state)


# ---- what a pass cannot do without ---------------------------------------------------------------

def work(case):
    t, d = case["tokens"], case["d"]
    e = _BYTES[case["dtype"]]
    if case["op"].startswith("ffn"):
        f = case["f"]
        if case["op"] == "ffn_forward":
            return {"bytes": e * (2 * t * d + 3 * d * f), "flops": 6.0 * t * d * f}
        return {"bytes": e * (3 * t * d + 2 * t * f + 6 * d * f), "flops": 12.0 * t * d * f}
    n = case["n"]
    k = 2 if case["op"] == "int8_gated" else 1
    read = e * t * d + k * (n * d + 4 * n) + (4 * n if case["bias"] else 0)
    return {"bytes": read + t * d + 4 * t + _BYTES[case["out"]] * t * n, "flops": 2.0 * k * t * d * n}


# ---- the same in 64 bits -------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    kind = case["act"]

    def phi(v):                                   # the activation and its derivative
        if kind == "silu":
            p = torch.special.expit(v)
            return v * p, p + v * p * (1 - p)
        if kind == "gelu":
            p = torch.special.ndtr(v)
            return v * p, p + v * torch.exp(-v.square() / 2) / math.sqrt(2 * math.pi)
        if kind == "relu":
            return v.clamp_min(0), torch.heaviside(v, torch.zeros((), dtype=v.dtype, device=v.device))
        return v, torch.ones((), dtype=v.dtype, device=v.device)

    if case["op"].startswith("ffn"):
        w1, w2, w3, x = (s[k].double() for k in ("w_gate", "w_up", "w_down", "x"))
        if case["op"] == "ffn_forward":
            inner = phi(torch.einsum("td,fd->tf", x, w1))[0].mul_(torch.einsum("td,fd->tf", x, w2))
            return torch.einsum("tf,df->td", inner, w3)
        a, slope = phi(s["gate"].double())
        u, dy = s["up"].double(), s["dy"].double()
        back = torch.einsum("td,df->tf", dy, w3)
        d1 = back * u * slope
        d2 = back * a
        return (torch.einsum("tf,fd->td", d1, w1) + torch.einsum("tf,fd->td", d2, w2),
                torch.einsum("tf,td->fd", d1, x), torch.einsum("tf,td->fd", d2, x),
                torch.einsum("td,tf->df", dy, a * u))
    # The 8-bit values are defined by 32-bit arithmetic (largest magnitude, one quotient, one product, round to
    # even), so they are formed in it here too; everything after them is in 64 bits.
    x = s["x"].float()
    top, _ = x.abs().max(dim=-1, keepdim=True)
    zero = top < 2.0 ** -100
    q = (x * (torch.full_like(top, 127.0) / top)).masked_fill(zero, 0.0).round_().double()
    scale = (top.double() / 127.0).masked_fill(zero, 0.0)
    if case["op"] == "int8_linear":
        y = torch.einsum("tk,nk->tn", q, s["wq"].double()) * scale * s["ws"].double()
        return None, scale[:, 0], phi(y if s["bias"] is None else y + s["bias"].double())[0]
    one = torch.einsum("tk,nk->tn", q, s["gq"].double()) * scale * s["gs"].double()
    two = torch.einsum("tk,nk->tn", q, s["uq"].double()) * scale * s["us"].double()
    return None, scale[:, 0], phi(one)[0] * two
