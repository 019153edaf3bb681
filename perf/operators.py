"""The operators of a dense feed-forward block, as cases to be timed.

  norm  the norms around a block: ``rms_norm`` in front of it (form "pre"), or
        ``residual_norm`` behind it (form "post": norm of the block's output,
        gate, residual scale, residual add, and the next block's input norm in
        one), forward alone as in serving, or with all gradients
  mlp   ``gated_mlp``: gate and up projections, clamped SwiGLU, down
        projection in bf16 weights, forward alone or with all gradients
  int4  ``int4_linear``: a projection with 4-bit weights and group scales

``own`` False computes them from elementary torch operations in 32 bits,
rounded once; ``own`` True through the package's entry points.
"""

import importlib
import math

import torch

own = False

DEVICE = "cuda"
EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # one decode token between two blocks: the smallest call
        {"name": "norm post 1x4096", "kind": "norm", "form": "post", "rows": 1, "width": 4096, "residual": "bf16",
         "weights": "bf16", "gate": "channel", "train": False},
        # a prefill chunk entering a block from an fp32 residual stream
        {"name": "norm pre 2048x4096", "kind": "norm", "form": "pre", "rows": 2048, "width": 4096, "residual": "f32",
         "weights": "bf16", "gate": "none", "train": False},
        # a ragged batch in training, odd width, one gate value a token, fp32 stream and norm weights
        {"name": "norm post train 1501x1001", "kind": "norm", "form": "post", "rows": 1501, "width": 1001,
         "residual": "f32", "weights": "f32", "gate": "token", "train": True},
        # a training batch of 8,192 tokens at the model's width, all in bf16, a learned gate a channel
        {"name": "norm post train 8192x4096", "kind": "norm", "form": "post", "rows": 8192, "width": 4096,
         "residual": "bf16", "weights": "bf16", "gate": "channel", "train": True},
        # one decode token through a square projection
        {"name": "int4 1x4096x4096 g64", "kind": "int4", "rows": 1, "n": 4096, "k": 4096, "group": 64,
         "offsets": True, "scales": "bf16"},
        # 16 sequences decoding together through a stacked gate/up projection
        {"name": "int4 16x4096x7168 g128", "kind": "int4", "rows": 16, "n": 4096, "k": 7168, "group": 128,
         "offsets": False, "scales": "bf16"},
        # a short ragged prompt, the finest groups, fp32 scales
        {"name": "int4 300x1536x4096 g32", "kind": "int4", "rows": 300, "n": 1536, "k": 4096, "group": 32,
         "offsets": True, "scales": "f32"},
        # a prefill chunk through a square projection
        {"name": "int4 2048x4096x4096 g128", "kind": "int4", "rows": 2048, "n": 4096, "k": 4096, "group": 128,
         "offsets": True, "scales": "bf16"},
        # one decode token through the block
        {"name": "mlp 1x4096x2048", "kind": "mlp", "rows": 1, "hidden": 4096, "inter": 2048, "limit": 10.0,
         "train": False},
        # a short prompt, served
        {"name": "mlp 96x4096x1536", "kind": "mlp", "rows": 96, "hidden": 4096, "inter": 1536, "limit": 10.0,
         "train": False},
        # a small ragged training batch, no clamp
        {"name": "mlp train 777x2048x1000", "kind": "mlp", "rows": 777, "hidden": 2048, "inter": 1000, "limit": 0.0,
         "train": True},
        # a training batch of 8,192 tokens at the model's widths: the largest call
        {"name": "mlp train 8192x4096x2048", "kind": "mlp", "rows": 8192, "hidden": 4096, "inter": 2048,
         "limit": 10.0, "train": True},
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "int4", "int4", "mlp", "mlp"])
    if kind == "norm":
        form = rng.choice(["pre", "post", "post"])
        width = rng.choice([8 * _log_uniform(rng, 8, 1024), _log_uniform(rng, 33, 8192)])
        rows = _log_uniform(rng, 1, min(8192, 8192 * 4096 // width))
        return {"kind": kind, "form": form, "rows": rows, "width": width, "residual": rng.choice(["bf16", "f32"]),
                "weights": rng.choice(["bf16", "bf16", "f32"]),
                "gate": "none" if form == "pre" else rng.choice(["none", "channel", "token", "full"]),
                "train": rng.random() < 0.5}
    if kind == "int4":
        group = rng.choice([32, 64, 128])
        rows, n = _log_uniform(rng, 1, 4096), _log_uniform(rng, 64, 8192)
        k = group * _log_uniform(rng, max(2, 256 // group), 8192 // group)
        rows = max(1, min(rows, 2048 * 4096 * 4096 // (n * k)))
        return {"kind": kind, "rows": rows, "n": n, "k": k, "group": group, "offsets": rng.random() < 0.7,
                "scales": rng.choice(["bf16", "bf16", "f32"])}
    hidden, inter = 8 * _log_uniform(rng, 16, 896), 8 * _log_uniform(rng, 16, 512)
    rows = _log_uniform(rng, 1, 8192)
    rows = max(1, min(rows, 8192 * 4096 * 2048 // (hidden * inter)))
    return {"kind": kind, "rows": rows, "hidden": hidden, "inter": inter, "limit": rng.choice([0.0, 1.5, 10.0]),
            "train": rng.random() < 0.5}


# ------------------------------------------------------------------ inputs --


class _Inputs:
    def __init__(self, seed):
        self.g = torch.Generator(device=DEVICE)
        self.g.manual_seed(int(seed))

    def normal(self, *shape, std=1.0, mean=0.0, dtype=torch.bfloat16):
        return torch.randn(shape, generator=self.g, device=DEVICE, dtype=torch.float32).mul_(std).add_(mean).to(dtype)


def _quantise(w, group, offsets, dtype):
    """4-bit codes (two a byte, even columns in the low half), scales and
    offsets of w f32 [n, k], per row and `group` columns."""
    n, k = w.shape
    v = w.view(n, k // group, group)
    if offsets:
        lo, hi = v.amin(2), v.amax(2)
        scale = ((hi - lo) / 15).to(dtype)
        off = lo.to(dtype)
    else:
        scale = (v.abs().amax(2) / 7.5).to(dtype)
        off = None
    base = (off if offsets else -8 * scale).float()
    q = ((v - base[:, :, None]) / scale.float()[:, :, None]).round().clamp(0, 15).to(torch.uint8).view(n, k)
    return (q[:, 0::2] | (q[:, 1::2] << 4)).contiguous(), scale, off


def _residual_stream(rng, case):
    x = rng.normal(case["rows"], case["width"], std=1.5, dtype=torch.float32)
    x[:, :: max(1, case["width"] // 7)] *= 20  # the few wide channels that a residual stream has
    return x.to(TYPES[case["residual"]])


def prepare(case, seed):
    rng, s = _Inputs(seed), {"case": case}
    if case["kind"] == "norm":
        rows, width, wt = case["rows"], case["width"], TYPES[case["weights"]]
        s["x"] = _residual_stream(rng, case)
        s["next"] = rng.normal(width, std=0.1, mean=1.0, dtype=wt)
        if case["form"] == "post":
            s["out"] = rng.normal(rows, width, std=0.4)
            s["post"] = rng.normal(width, std=0.1, mean=1.0, dtype=wt)
            shape = {"none": None, "channel": (width,), "token": (rows, 1), "full": (rows, width)}[case["gate"]]
            s["gate"] = None if shape is None else rng.normal(*shape, std=0.3, mean=0.5, dtype=wt)
            s["scale"] = 0.25
        if case["train"]:
            s["dx"] = rng.normal(rows, width, std=0.01, dtype=TYPES[case["residual"]])
            s["dy"] = rng.normal(rows, width, std=0.01)
            for name in ("x", "out", "post", "gate", "next"):
                if s.get(name) is not None:
                    s[name].requires_grad_()
    elif case["kind"] == "int4":
        s["x"] = rng.normal(case["rows"], case["k"])
        w = rng.normal(case["n"], case["k"], std=0.02, dtype=torch.float32)
        s["codes"], s["scales"], s["offsets"] = _quantise(w, case["group"], case["offsets"], TYPES[case["scales"]])
    else:
        rows, hidden, inter = case["rows"], case["hidden"], case["inter"]
        s["x"] = rng.normal(rows, hidden)
        s["gate"], s["up"] = rng.normal(inter, hidden, std=0.02), rng.normal(inter, hidden, std=0.02)
        s["down"] = rng.normal(hidden, inter, std=0.02)
        if case["train"]:
            s["dy"] = rng.normal(rows, hidden, std=0.01)
            for name in ("x", "gate", "up", "down"):
                s[name].requires_grad_()
    return s


# --------------------------------------------------------------------- run --


def _package():
    return importlib.import_module("glm53-flash-mlx_amd")


def _grads(outputs, given, leaves):
    names = [n for n in leaves if leaves[n] is not None]
    got = torch.autograd.grad(outputs, [leaves[n] for n in names], given)
    return {"d_" + n: g for n, g in zip(names, got)}


def _plain_rms(x, weight):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()


def _plain_residual(s):
    out = _plain_rms(s["out"].float(), s["post"])
    if s["gate"] is not None:
        out = out * s["gate"].float()
    x = s["x"].float() + s["scale"] * out
    return x, _plain_rms(x, s["next"])


def _run_norm(s):
    case = s["case"]
    if case["form"] == "pre":
        if own:
            y = _package().rms_norm(s["x"], s["next"], EPS, dtype=torch.bfloat16)
        else:
            y = _plain_rms(s["x"].float(), s["next"]).to(torch.bfloat16)
        got = {"y": y}
        if case["train"]:
            got.update(_grads([y], [s["dy"]], {"x": s["x"], "next": s["next"]}))
        return got
    if own:
        x, y = _package().residual_norm(s["x"], s["out"], post_weight=s["post"], gate=s["gate"], scale=s["scale"],
                                        next_weight=s["next"], eps=EPS)
    else:
        x, y = _plain_residual(s)
        x, y = x.to(s["x"].dtype), y.to(torch.bfloat16)
    got = {"x": x, "y": y}
    if case["train"]:
        got.update(_grads([x, y], [s["dx"], s["dy"]], {n: s[n] for n in ("x", "out", "post", "gate", "next")}))
    return got


def _plain_mlp(s):
    x, limit = s["x"].float(), s["case"]["limit"]
    g, u = x @ s["gate"].float().T, x @ s["up"].float().T
    if limit:
        g, u = g.clamp(max=limit), u.clamp(-limit, limit)
    return ((g * torch.sigmoid(g) * u) @ s["down"].float().T).to(torch.bfloat16)


def _run_mlp(s):
    if own:
        y = _package().gated_mlp(s["x"], s["gate"], s["up"], s["down"], limit=s["case"]["limit"] or None)
    else:
        y = _plain_mlp(s)
    got = {"y": y}
    if s["case"]["train"]:
        got.update(_grads([y], [s["dy"]], {n: s[n] for n in ("x", "gate", "up", "down")}))
    return got


def _run_int4(s):
    if own:
        return _package().int4_linear(s["x"], s["codes"], s["scales"], s["offsets"])
    case, codes = s["case"], s["codes"]
    q = torch.stack([codes & 15, codes >> 4], 2).view(case["n"], -1, case["group"]).float()
    scale = s["scales"].float()[:, :, None]
    off = -8 * scale if s["offsets"] is None else s["offsets"].float()[:, :, None]
    w = (q * scale + off).view(case["n"], case["k"])
    return (s["x"].float() @ w.T).to(torch.bfloat16)


def run(state):
    return {"norm": _run_norm, "mlp": _run_mlp, "int4": _run_int4}[state["case"]["kind"]](state)


# -------------------------------------------------------------------- work --


def work(case):
    if case["kind"] == "norm":
        rows, width, r = case["rows"], case["width"], 4 if case["residual"] == "f32" else 2
        w = 4 if case["weights"] == "f32" else 2
        gates = {"none": 0, "channel": width, "token": rows, "full": rows * width}[case["gate"]]
        cells = rows * width
        if case["form"] == "pre":
            total = cells * (r + 2) + width * w  # x, y
            if case["train"]:
                total += cells * (2 + r) + width * w  # dy, d_x
        else:
            total = cells * (2 * r + 4) + (2 * width + gates) * w  # x, out, x', y
            if case["train"]:
                total += cells * (2 * r + 4) + (2 * width + gates) * w  # dx', dy, d_x, d_out
        return {"bytes": total, "flops": cells * (40 if case["train"] else 12)}
    if case["kind"] == "int4":
        rows, n, k = case["rows"], case["n"], case["k"]
        tables = (2 if case["offsets"] else 1) * n * (k // case["group"]) * (4 if case["scales"] == "f32" else 2)
        return {"bytes": n * k // 2 + tables + 2 * rows * (n + k), "flops": 2 * rows * n * k}
    rows, hidden, inter = case["rows"], case["hidden"], case["inter"]
    weights = 3 * hidden * inter * 2
    total, flops = weights + 2 * rows * hidden * 2, 6 * rows * hidden * inter
    if case["train"]:
        total, flops = total + weights + 2 * rows * hidden * 2, 3 * flops
    return {"bytes": total, "flops": flops}


# ------------------------------------------------------------------- exact --


def _norm64(v, w):
    """v / rms(v) * w in 64 bits, and 1 / rms."""
    r = (v.pow(2).sum(1, keepdim=True) / v.shape[1] + EPS).pow(-0.5)
    return v * r * w, r


def _norm64_back(v, r, t):
    """The gradient of v r by v, applied to t."""
    return r * t - v * r.pow(3) * (t * v).sum(1, keepdim=True) / v.shape[1]


def _exact_norm(s):
    case, d = s["case"], lambda n: s[n].detach().double()
    x, nw = d("x"), d("next")
    if case["form"] == "pre":
        y, r = _norm64(x, nw)
        got = {"y": y}
        if case["train"]:
            dy = d("dy")
            got.update(d_x=_norm64_back(x, r, dy * nw), d_next=(dy * x * r).sum(0))
        return got
    o, pw, a = d("out"), d("post"), s["scale"]
    gate = d("gate") if s["gate"] is not None else torch.ones((), dtype=torch.float64, device=DEVICE)
    normed, ro = _norm64(o, pw)
    x = x + a * gate * normed
    y, r = _norm64(x, nw)
    got = {"x": x, "y": y}
    if case["train"]:
        dy = d("dy")
        dx = d("dx") + _norm64_back(x, r, dy * nw)
        dn = a * gate * dx
        got.update(d_x=dx, d_out=_norm64_back(o, ro, dn * pw), d_post=(dn * o * ro).sum(0),
                   d_next=(dy * x * r).sum(0))
        if s["gate"] is not None:
            dg = a * normed * dx
            got["d_gate"] = {"channel": lambda: dg.sum(0), "token": lambda: dg.sum(1, keepdim=True),
                             "full": lambda: dg}[case["gate"]]()
    return got


def _exact_mlp(s):
    d = lambda n: s[n].detach().double()
    x, wg, wu, wd, limit = d("x"), d("gate"), d("up"), d("down"), s["case"]["limit"] or math.inf
    g, u = x.matmul(wg.t()), x.matmul(wu.t())
    gc, uc = torch.minimum(g, torch.full_like(g, limit)), u.clip(-limit, limit)
    sig = 1 / (1 + torch.exp(-gc))
    h = gc * sig * uc
    got = {"y": h.matmul(wd.t())}
    if s["case"]["train"]:
        dy = d("dy")
        dh = dy.matmul(wd)
        dg = dh * uc * sig * (1 + gc * (1 - sig)) * (g <= limit)
        du = dh * gc * sig * (u.abs() <= limit)
        got.update(d_x=dg.matmul(wg) + du.matmul(wu), d_gate=dg.t().matmul(x), d_up=du.t().matmul(x),
                   d_down=dy.t().matmul(h))
    return got


def _exact_int4(s):
    case = s["case"]
    q = torch.empty(case["n"], case["k"], dtype=torch.float64, device=DEVICE)
    q[:, 0::2], q[:, 1::2] = (s["codes"] % 16).double(), (s["codes"] // 16).double()
    scale = s["scales"].double().repeat_interleave(case["group"], 1)
    off = scale * -8 if s["offsets"] is None else s["offsets"].double().repeat_interleave(case["group"], 1)
    return s["x"].double().matmul((q * scale + off).t())


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "mlp": _exact_mlp, "int4": _exact_int4}[case["kind"]](s)
