"""The operators of a model served in 8 bits, with the inputs a user's program has in hand, the
calls in elementary torch operations and through the framework, and the same results in float64.

Rows and weights are held as e4m3 values in blocks of 32 along the axis that a product sums over,
each block with a power of two as its scale: the smallest one (from 2^-126 on) by which the block's
largest magnitude is at most 448. What is held in 8 bits is returned as the values it stands for.

* ``quant``  -- rows to 8 bits;
* ``norm``   -- the residual's addition and the root-mean-square norm, its rows in 8 bits;
* ``matmul`` -- rows times a weight in 8 bits, with bias, activation and residual;
* ``gate``   -- the gated MLP's first product, value times silu(gate), its rows in 8 bits;
* ``mlp``    -- an MLP block as a model calls it: norm, gate and the product back, with residual.
"""

from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
EPS = 1e-5
BLOCK = 32


def listed():
    return [
        # the scan's output on its way to the layer's last product, a prompt of eight sequences
        dict(name="quant_prompt", kind="quant", rows=16384, width=2048, dtype="bf16"),
        # one token's row of the byte LM's float32 stream: the smallest call
        dict(name="norm_token", kind="norm", rows=1, width=768, dtype="f32", add=True),
        # a prompt's rows between two blocks, a float32 stream
        dict(name="norm_prompt", kind="norm", rows=32768, width=1024, dtype="f32", add=True),
        # a short ragged batch of an odd width, a bf16 stream
        dict(name="norm_odd", kind="norm", rows=777, width=515, dtype="bf16", add=True),
        # one token through the layer's first product (d_model 1024)
        dict(name="matmul_token", kind="matmul", rows=1, inner=1024, outer=4480, dtype="bf16",
             bias=False, act="none", residual=False),
        # a decode step of 256 sequences through the same product
        dict(name="matmul_decode", kind="matmul", rows=256, inner=1024, outer=4480, dtype="bf16",
             bias=False, act="none", residual=False),
        # a prompt through the same product: its output is most of the traffic
        dict(name="matmul_prompt", kind="matmul", rows=16384, inner=1024, outer=4480, dtype="bf16",
             bias=False, act="none", residual=False),
        # the layer's last product, added to the stream
        dict(name="matmul_residual", kind="matmul", rows=32768, inner=2048, outer=1024, dtype="bf16",
             bias=False, act="none", residual=True),
        # odd sizes, a bias and an activation
        dict(name="matmul_odd", kind="matmul", rows=333, inner=515, outer=1027, dtype="f32",
             bias=True, act="gelu", residual=True),
        # a prompt through the gated MLP's first product
        dict(name="gate_prompt", kind="gate", rows=8192, width=1024, inner=2816, dtype="bf16",
             bias=False),
        # one token through the gate of a larger model
        dict(name="gate_token", kind="gate", rows=1, width=2048, inner=5632, dtype="bf16", bias=False),
        # a whole MLP block over a long prompt: the largest call
        dict(name="mlp_prompt", kind="mlp", rows=16384, width=2048, inner=5632, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A width: mostly multiples of 64, some odd."""
    n = _log_int(rng, lo, hi)
    return n if rng.random() < 0.3 else max(64, n // 64 * 64)


def draw(rng):
    kind = rng.choice(["quant", "norm", "norm", "matmul", "matmul", "matmul", "gate", "gate", "mlp"])
    rows = rng.choice([1, 2, 4]) if rng.random() < 0.25 else _log_int(rng, 1, 32768)
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if kind in ("quant", "norm"):
        case = dict(kind=kind, rows=rows, width=_size(rng, 64, 4096), dtype=dtype)
        return dict(case, add=rng.random() < 0.7) if kind == "norm" else case
    if kind == "matmul":
        inner, outer = _size(rng, 64, 4096), _size(rng, 64, 5632)
        # no more work than the largest listed case has
        rows = min(rows, 3 * 16384 * 2048 * 5632 // (inner * outer))
        return dict(kind=kind, rows=rows, inner=inner, outer=outer, dtype=dtype,
                    bias=rng.random() < 0.4,
                    act=rng.choice(["none", "none", "silu", "gelu", "relu"]),
                    residual=rng.random() < 0.5)
    width, inner = _size(rng, 64, 2048), _size(rng, 64, 5632)
    if kind == "gate":
        return dict(kind=kind, rows=min(rows, 16384), width=width, inner=inner, dtype=dtype,
                    bias=rng.random() < 0.3)
    return dict(kind=kind, rows=min(rows, 16384), width=width, inner=inner, dtype="bf16")


# ----------------------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------------------


def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def _acts(gen, rows, width, dt):
    """Rows as a model's blocks leave them: normal, with a few channels many times as large."""
    x = torch.randn(rows, width, generator=gen, device=DEVICE)
    loud = torch.rand(width, generator=gen, device=DEVICE) < 0.01
    return (x * torch.where(loud, 12.0, 1.0)).to(dt)


def _weight(gen, inner, outer):
    return (torch.randn(inner, outer, generator=gen, device=DEVICE) / math.sqrt(inner)).to(torch.bfloat16)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    kind, rows, dt = case["kind"], case["rows"], _dtype(case)
    state = dict(case=case)
    if own:
        import __graft_entry__

        state["m3"] = __graft_entry__.load_package()
    width = case["inner"] if kind == "matmul" else case["width"]
    state["x"] = _acts(gen, rows, width, dt)
    weights = {}
    if kind in ("norm", "mlp"):
        state["gain"] = 1.0 + 0.1 * torch.randn(width, generator=gen, device=DEVICE)
        if case.get("add", True):
            state["add"] = _acts(gen, rows, width, torch.bfloat16)
    if kind == "matmul":
        weights["w"] = _weight(gen, width, case["outer"])
        if case["residual"]:
            state["residual"] = _acts(gen, rows, case["outer"], torch.bfloat16)
    if kind in ("gate", "mlp"):
        weights["w1"] = _weight(gen, width, 2 * case["inner"])
    if kind == "mlp":
        weights["w2"] = _weight(gen, case["inner"], width)
    if case.get("bias"):
        n = case["outer"] if kind == "matmul" else 2 * case["inner"]
        state["bias"] = 0.1 * torch.randn(n, generator=gen, device=DEVICE)
    # weights are laid out once: packed in 8 bits, or as the values these stand for
    for name, w in weights.items():
        if own:
            state[name] = state["m3"].eightbit.pack8(w, gated=name == "w1")
        else:
            state[name] = _rows8(w.t().float()).t().contiguous()
    return state


# ----------------------------------------------------------------------------------------
# the calls, and their plain form
# ----------------------------------------------------------------------------------------


def run(state):
    with torch.no_grad():
        return _own(state) if own else _plain(state)


def _own(state):
    case, T = state["case"], state["m3"].eightbit
    kind, x = case["kind"], state["x"]
    if kind == "quant":
        return T.quantize8(x).dequantize()
    if kind == "norm":
        s, rows = T.rms_norm8(x, state["gain"], EPS, add=state.get("add"))
        return (s, rows.dequantize()) if "add" in state else rows.dequantize()
    if kind == "matmul":
        return T.matmul8(x, state["w"], bias=state.get("bias"),
                         activation=None if case["act"] == "none" else case["act"],
                         residual=state.get("residual"))
    if kind == "gate":
        return T.swiglu8(x, state["w1"], bias=state.get("bias")).dequantize()
    s, rows = T.rms_norm8(x, state["gain"], EPS, add=state["add"])
    return T.matmul8(T.swiglu8(rows, state["w1"]), state["w2"], residual=s)


def _rows8(x):
    """Float32 rows as the values that their 8 bits stand for."""
    k = x.shape[-1]
    b = torch.nn.functional.pad(x, (0, -k % BLOCK)).unflatten(-1, (-1, BLOCK))
    frac, e = torch.frexp(b.abs().amax(-1, keepdim=True))
    # amax = 2 frac 2^(e - 1), and 448 = 1.75 2^8
    e = (e.int() - 9 + (frac > 0.875)).clamp(min=-126)
    down = ((127 - e) << 23).view(torch.float32)
    up = ((127 + e) << 23).view(torch.float32)
    return ((b * down).to(torch.float8_e4m3fn).float() * up).flatten(-2)[..., :k]


def _norm_plain(state):
    s = state["x"].float()
    if "add" in state:
        s = (s + state["add"].float()).to(state["x"].dtype).float()
    rstd = 1.0 / torch.sqrt((s * s).sum(-1, keepdim=True) / s.shape[-1] + EPS)
    return s, _rows8(s * rstd * state["gain"])


def _gate_plain(rows, w, bias):
    h = rows @ w
    if bias is not None:
        h = h + bias
    n = h.shape[-1] // 2
    value, gate = h[..., :n], h[..., n:]
    return _rows8(value * (gate / (1.0 + torch.exp(-gate))))


def _plain(state):
    case, x, bf16 = state["case"], state["x"], torch.bfloat16
    kind = case["kind"]
    if kind == "quant":
        return _rows8(x.float()).to(bf16)
    if kind == "norm":
        s, rows = _norm_plain(state)
        return (s.to(x.dtype), rows.to(bf16)) if "add" in state else rows.to(bf16)
    if kind == "matmul":
        y = _rows8(x.float()) @ state["w"]
        if "bias" in state:
            y = y + state["bias"]
        if case["act"] == "silu":
            y = y / (1.0 + torch.exp(-y))
        elif case["act"] == "gelu":
            y = 0.5 * y * (1.0 + torch.erf(y * math.sqrt(0.5)))
        elif case["act"] == "relu":
            y = torch.clamp(y, min=0.0)
        if "residual" in state:
            y = y + state["residual"].float()
        return y.to(bf16)
    if kind == "gate":
        return _gate_plain(_rows8(x.float()), state["w1"], state.get("bias")).to(bf16)
    s, rows = _norm_plain(state)
    return (_gate_plain(rows, state["w1"], None) @ state["w2"] + s).to(bf16)


# ----------------------------------------------------------------------------------------
# what a pass cannot do without
# ----------------------------------------------------------------------------------------


def work(case):
    kind, rows = case["kind"], case["rows"]
    size = 2 if case["dtype"] == "bf16" else 4
    held = 1.0 + 1.0 / BLOCK   # an 8-bit value and its share of a scale
    if kind in ("quant", "norm"):
        d = case["width"]
        # the rows in 8 bits, and the values they stand for
        nbytes = rows * d * (size + held + 2)
        if kind == "norm":
            nbytes += 4 * d + (rows * d * (2 + size) if case["add"] else 0)
        return dict(bytes=int(nbytes), flops=(6 if kind == "norm" else 3) * rows * d)
    if kind == "matmul":
        k, n = case["inner"], case["outer"]
        nbytes = rows * k * size + k * n * held + rows * n * 2
        nbytes += (4 * n if case["bias"] else 0) + (rows * n * 2 if case["residual"] else 0)
        return dict(bytes=int(nbytes), flops=2 * rows * k * n)
    d, n = case["width"], case["inner"]
    nbytes = rows * d * size + 2 * d * n * held
    if kind == "gate":
        nbytes += rows * n * (held + 2) + (8 * n if case["bias"] else 0)
        return dict(bytes=int(nbytes), flops=4 * rows * d * n)
    nbytes += 4 * d + rows * d * 4 + d * n * held
    return dict(bytes=int(nbytes), flops=6 * rows * d * n)


# ----------------------------------------------------------------------------------------
# float64, from the definitions
# ----------------------------------------------------------------------------------------


def _exp2(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact8(x):
    """Float64 rows, each value the multiple of its e4m3 step that is nearest (ties to even)."""
    k = x.shape[-1]
    out = torch.zeros(*x.shape[:-1], -(-k // BLOCK) * BLOCK, dtype=torch.float64, device=x.device)
    out[..., :k] = x
    b = out.reshape(*x.shape[:-1], -1, BLOCK)
    top = b.abs().max(-1, keepdim=True).values
    frac, e = torch.frexp(top)
    e = e.long() - 9
    e = torch.where(frac * 2.0 > 1.75, e + 1, e).clamp(min=-126)
    v = b / _exp2(e)
    step = _exp2((torch.frexp(v)[1].long() - 1).clamp(min=-6) - 3)
    return (torch.round(v / step) * step * _exp2(e)).reshape(out.shape)[..., :k]


def _exact_norm(x, state, gain):
    s = x.double()
    if "add" in state:
        # the stream's next row, held in the stream's type
        s = (s + state["add"].double()).to(x.dtype).double()
    return s, _exact8(s * torch.rsqrt(s.square().mean(-1, keepdim=True) + EPS) * gain)


def exact(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    kind, rows, dt = case["kind"], case["rows"], _dtype(case)
    # the inputs of `prepare`, in its order, the weights before they are laid out
    state = {}
    width = case["inner"] if kind == "matmul" else case["width"]
    x = _acts(gen, rows, width, dt)
    gain = w = w1 = w2 = None
    if kind in ("norm", "mlp"):
        gain = (1.0 + 0.1 * torch.randn(width, generator=gen, device=DEVICE)).double()
        if case.get("add", True):
            state["add"] = _acts(gen, rows, width, torch.bfloat16)
    if kind == "matmul":
        w = _exact8(_weight(gen, width, case["outer"]).double().t()).t()
        residual = _acts(gen, rows, case["outer"], torch.bfloat16).double() if case["residual"] else 0.0
    if kind in ("gate", "mlp"):
        w1 = _exact8(_weight(gen, width, 2 * case["inner"]).double().t()).t()
    if kind == "mlp":
        w2 = _exact8(_weight(gen, case["inner"], width).double().t()).t()
    bias = 0.0
    if case.get("bias"):
        n = case["outer"] if kind == "matmul" else 2 * case["inner"]
        bias = (0.1 * torch.randn(n, generator=gen, device=DEVICE)).double()
    if kind == "quant":
        return _exact8(x.double())
    if kind == "norm":
        s, out = _exact_norm(x, state, gain)
        return (s, out) if "add" in state else out
    if kind == "matmul":
        y = _exact8(x.double()) @ w + bias
        acts = {"none": lambda t: t, "silu": lambda t: t * torch.sigmoid(t),
                "gelu": torch.nn.functional.gelu, "relu": torch.relu}
        return acts[case["act"]](y) + residual
    n = case["inner"]
    s, held = _exact_norm(x, state, gain) if kind == "mlp" else (None, _exact8(x.double()))
    h = held @ w1 + bias
    a = _exact8(h[:, :n] * h[:, n:] * torch.sigmoid(h[:, n:]))
    return a if kind == "gate" else a @ w2 + s
