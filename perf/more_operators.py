"""The operators of a transformer block on a frozen 8-bit base, as cases to measure: inputs, one pass through an operator,
what the pass cannot do without, and its value in 64 bits.

  quantize     torch_vulkan.quantize_int8_rows and dequant_int8_rows: 8-bit integers with one scale for each row
  linear       torch_vulkan.int8_linear: 16-bit rows, quantised on the way in, times frozen 8-bit weights, and the rows' and
               the bias's gradients
  norm         torch_vulkan.rms_norm: root-mean-square norm, with or without the residual's addition, and its gradients
  norm_linear  torch_vulkan.rms_norm_int8 and int8_linear on what it gives: residual, norm, 8-bit rows, product
  rotary       torch_vulkan.rotary_embedding: queries and keys turned by positions of several axes, and their gradients

`own` false: the operators written out in elementary torch operations in 32 bits on the GPU (64 for angles and for values next
to a rounding border); `own` true: the calls that a program makes of them on the "vk" device.  Sizes are those of this
repository's tests and benchmark (2048 and 8192 wide blocks, 77-token text, heads of 128, odd image token counts, positions
over frames, rows and columns) and generic ones around them."""

import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
EPS = 1e-6


def listed():
    return [
        # a frozen MLP weight is quantised when the model is loaded, and written out again where a merge needs it whole
        {"name": "quantize_weight", "kind": "quantize", "dtype": "bf16", "rows": 8192, "cols": 2048},
        # an fp32 checkpoint's weight of odd sizes
        {"name": "quantize_ragged", "kind": "quantize", "dtype": "f32", "rows": 517, "cols": 1001},
        # one conditioning vector through a frozen layer: latency and the weights' bytes
        {"name": "linear_token", "kind": "linear", "dtype": "bf16", "tokens": 1, "fin": 2048, "fout": 8192, "train": False},
        # the captions of four images (4 x 77 tokens) through a frozen projection, both directions
        {"name": "linear_text", "kind": "linear", "dtype": "f16", "tokens": 308, "fin": 2048, "fout": 2048, "train": True},
        # a frozen MLP layer under image tokens, both directions
        {"name": "linear_image", "kind": "linear", "dtype": "bf16", "tokens": 4096, "fin": 2048, "fout": 8192, "train": True},
        # four captions in full precision through a norm of odd width with its residual, both directions
        {"name": "norm_text", "kind": "norm", "dtype": "f32", "rows": 308, "cols": 1001, "residual": True, "train": True},
        # the queries' heads of image tokens, a slice of one projection of queries, keys and values
        {"name": "norm_heads", "kind": "norm", "dtype": "bf16", "rows": 4096, "heads": 16, "cols": 128, "residual": False, "train": True},
        # the residual stream of an odd aspect bucket (60 x 67 tokens)
        {"name": "norm_image", "kind": "norm", "dtype": "bf16", "rows": 4020, "cols": 2048, "residual": True, "train": True},
        # one token on its way into a frozen layer
        {"name": "norm_linear_token", "kind": "norm_linear", "dtype": "f16", "tokens": 1, "fin": 2048, "fout": 8192},
        # the image tokens of that bucket on their way into a frozen MLP layer while sampling
        {"name": "norm_linear_image", "kind": "norm_linear", "dtype": "bf16", "tokens": 4020, "fin": 2048, "fout": 8192},
        # one new token of each of eight sequences at far positions, shared keys, neighbouring values paired
        {"name": "rotary_token", "kind": "rotary", "dtype": "f16", "batch": 8, "heads": 16, "kv": 4, "frames": 1, "height": 1, "width": 1,
         "dim": 128, "sections": "64", "interleaved": True, "far": 1000000, "train": False},
        # queries and keys of two clips of 16 frames at 16 x 16 patches, heads split 44 / 42 / 42 over the axes
        {"name": "rotary_video", "kind": "rotary", "dtype": "bf16", "batch": 2, "heads": 16, "kv": 16, "frames": 16, "height": 16, "width": 16,
         "dim": 128, "sections": "22,21,21", "interleaved": False, "far": 0, "train": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return w["flops"] + w["bytes"] * 300


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(("quantize", "linear", "linear", "norm", "norm", "norm_linear", "rotary", "rotary"))
        half = rng.choice(("bf16", "f16"))
        any3 = rng.choice(("bf16", "f16", "f32"))
        width = rng.choice((64 * _log(rng, 2, 128), 16 * _log(rng, 8, 512), _log(rng, 100, 8192)))
        if kind == "quantize":
            c = {"dtype": any3, "rows": _log(rng, 64, 16384), "cols": width}
        elif kind in ("linear", "norm_linear"):
            step = rng.choice((64, 64, 64, 8, 1))  # output widths are mostly multiples of 64
            c = {"dtype": half, "tokens": _log(rng, 1, 8192), "fin": 16 * _log(rng, 16, 512), "fout": _log(rng, 256, 8192) // step * step}
            if kind == "linear":
                c["train"] = rng.random() < 0.5
        elif kind == "norm":
            c = {"dtype": any3, "rows": _log(rng, 1, 16384), "residual": rng.random() < 0.5, "train": rng.random() < 0.6}
            if rng.random() < 0.3:
                c.update(heads=rng.randint(1, 24), cols=rng.choice((64, 80, 128, 256)), residual=False)
            else:
                c["cols"] = width
        else:
            dim = rng.choice((64, 80, 96, 128, 128, 128, 256))
            axes = rng.choice((1, 2, 3, 3))
            pairs = dim // 2 if rng.random() < 0.7 else dim // 4
            sec = [pairs // axes] * axes
            sec[0] += pairs - sum(sec)
            train = rng.random() < 0.6
            c = {"dtype": any3, "batch": rng.randint(1, 4), "heads": rng.randint(1, 6) * 4, "kv": 4, "frames": 1, "height": 1, "width": 1, "dim": dim,
                 "sections": ",".join(map(str, sec)), "interleaved": rng.random() < 0.4, "far": 0 if train else _log(rng, 1000, 4000000), "train": train}
            if rng.random() < 0.5:
                c["kv"] = c["heads"]
            if train or rng.random() < 0.5:
                c.update(frames=rng.choice((1, 1, rng.randint(2, 16))), height=rng.randint(4, 64), width=rng.randint(4, 64))
        c = {"kind": kind, **c}
        if _cost(c) <= most:
            return c


# ---- inputs -------------------------------------------------------------------------------------------------------
_GRADS = {"linear": ("x", "b"), "norm": ("x", "w"), "rotary": ("q", "k")}


def _grads(case):
    if not case.get("train"):
        return ()
    return _GRADS[case["kind"]] + (("r",) if case.get("residual") else ())


def _sections(case):
    return tuple(int(s) for s in case["sections"].split(","))


def _inputs(case, seed):
    """Everything that a pass reads, from the seed alone: activations and output gradients ~ N(0, 1), a residual stream with a
    few large channels, weights ~ N(0, 0.02) with a size of its own in each row, norm weights around one, biases of a trained
    size."""
    dev = "cuda" if torch.cuda.is_available() else "cpu"
    g = torch.Generator(dev).manual_seed(seed)
    dt, kind = DTYPES[case["dtype"]], case["kind"]

    def r(*shape, scale=1.0, mean=0.0):
        return torch.randn(shape, generator=g, device=dev).mul_(scale).add_(mean).to(dt)

    def weight(o, i):
        return r(o, i, scale=0.02) * torch.exp(torch.randn((o, 1), generator=g, device=dev) * 0.5).to(dt)

    def stream(m, n):
        return r(m, n) * torch.exp(torch.randn((n,), generator=g, device=dev)).to(dt)

    if kind == "quantize":
        return {"x": weight(case["rows"], case["cols"])}
    if kind in ("linear", "norm_linear"):
        m, i, o = case["tokens"], case["fin"], case["fout"]
        codes, scale = _quantize(weight(o, i))
        t = {"x": r(m, i), "w8": codes.to(torch.int8), "s8": scale, "b": r(o, scale=0.02)}
        if kind == "norm_linear":
            t.update(r=stream(m, i), w=r(i, scale=0.2, mean=1.0))
        elif case["train"]:
            t["gy"] = r(m, o)
        return t
    if kind == "norm":
        m, n = case["rows"], case["cols"]
        if "heads" in case:  # queries, keys and values of one projection
            t = {"x": r(m, 3, case["heads"], n), "w": r(n, scale=0.2, mean=1.0)}
        else:
            t = {"x": r(m, n), "w": r(n, scale=0.2, mean=1.0)}
        if case["residual"]:
            t["r"] = stream(m, n)
        if case["train"]:
            t["gy"] = r(*_rows(case))
            if case["residual"]:
                t["gh"] = r(*_rows(case))
        return t
    n, d, sec = case["batch"], case["dim"], _sections(case)
    axes = [case["frames"], case["height"], case["width"]][3 - len(sec):]
    axes[0] *= case["frames"] * case["height"] * case["width"] // math.prod(axes)
    grid = torch.stack(torch.meshgrid(*(torch.arange(a, device=dev) for a in axes), indexing="ij"), -1).view(-1, len(sec))
    s = grid.shape[0]
    t = {"q": r(n, s, case["heads"], d), "k": r(n, s, case["kv"], d)}  # token-major, as a model's projections leave them
    t["pos"] = grid if not case["far"] else grid + torch.randint(0, case["far"], (n, 1, len(sec)), generator=g, device=dev)
    t["freqs"] = torch.cat([10000.0 ** (-torch.arange(a, device=dev, dtype=torch.float64) / a) for a in sec])
    if case["train"]:
        t.update(gq=r(n, s, case["heads"], d), gk=r(n, s, case["kv"], d))
    return t


def _rows(case):
    return (case["rows"], case["heads"], case["cols"]) if "heads" in case else (case["rows"], case["cols"])


def prepare(case, seed):
    t = _inputs(case, seed)
    if own:  # a program that uses the operators has its tensors on the framework's device
        path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "torch-vulkan_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        import torch_vulkan

        torch_vulkan.set_inline_backward()  # as a training loop on this device does once, on its own thread
        t = {k: v.cpu().to("vk") for k, v in t.items()}
        if "heads" in case and case["kind"] == "norm":
            t["x"] = t["x"][:, 0]
        for n in _grads(case):
            t[n] = t[n].detach().requires_grad_(True)
    elif "heads" in case and case["kind"] == "norm":
        t["x"] = t["x"][:, 0]
    return {"case": case, "t": t}


# ---- one pass -----------------------------------------------------------------------------------------------------
def run(state):
    case, t = state["case"], state["t"]
    return _own(case, t) if own else _plain(case, t)


def _own(case, t):
    import torch_vulkan as tv

    kind, dt = case["kind"], DTYPES[case["dtype"]]
    if kind == "quantize":
        codes, scale = tv.quantize_int8_rows(t["x"])
        return {"y": tv.dequant_int8_rows(codes, scale, dt)}
    if kind == "norm_linear":
        codes, scale, h = tv.rms_norm_int8(t["x"], t["w"], residual=t["r"], eps=EPS)
        return {"y": tv.int8_linear(codes, t["w8"], t["s8"], t["b"], x_scale=scale, out_dtype=dt), "h": h}
    if kind == "linear":
        out, of = {"y": tv.int8_linear(t["x"], t["w8"], t["s8"], t["b"])}, ("gy",)
    elif kind == "norm" and case["residual"]:
        y, h = tv.rms_norm(t["x"], t["w"], residual=t["r"], eps=EPS)
        out, of = {"y": y, "h": h}, ("gy", "gh")
    elif kind == "norm":
        out, of = {"y": tv.rms_norm(t["x"], t["w"], eps=EPS)}, ("gy",)
    else:
        q, k = tv.rotary_embedding(t["q"].transpose(1, 2), t["k"].transpose(1, 2), t["pos"], t["freqs"], _sections(case), interleaved=case["interleaved"])
        out, of = {"q": q.transpose(1, 2), "k": k.transpose(1, 2)}, ("gq", "gk")
    names = _grads(case)
    if not names:
        return out
    grads = torch.autograd.grad(list(out.values()), [t[n] for n in names], [t[n] for n in of])
    return {**{n: y.detach() for n, y in out.items()}, **{"d" + n: d for n, d in zip(names, grads)}}


def _quantize(x):
    """Codes (whole numbers in fp32) and fp32 scales of x [rows, cols]: nearest multiples of largest / 127, ties to even.  127 x
    is exact for 16-bit values, and its quotient in 32 bits is on the side of a border that the true one is on; for 32-bit
    values both need 64 bits."""
    v = x.double() if x.dtype == torch.float32 else x.float()
    top = v.abs().amax(-1, keepdim=True)
    codes = torch.where(top > 0, torch.round(v * 127.0 / top), 0.0).float()
    return codes, top.squeeze(-1).float() / 127.0


def _norm(h, w):
    inv = torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS)
    return h * inv * w, inv


def _plain(case, t):
    kind, dt = case["kind"], DTYPES[case["dtype"]]
    if kind == "quantize":
        codes, scale = _quantize(t["x"])
        return {"y": (codes * scale.unsqueeze(-1)).to(dt)}
    if kind == "linear":
        codes, scale = _quantize(t["x"])
        w = t["w8"].float()
        out = {"y": ((codes @ w.t()) * scale.unsqueeze(-1) * t["s8"] + t["b"].float()).to(dt)}
        if case["train"]:  # straight through, as if x had gone in unrounded
            g = t["gy"].float()
            out.update(dx=((g * t["s8"]) @ w).to(dt), db=g.sum(0).to(dt))
        return out
    if kind == "norm_linear":
        h = t["x"].float() + t["r"].float()
        y, _ = _norm(h, t["w"].float())
        top = y.abs().amax(-1, keepdim=True)
        codes, scale = torch.where(top > 0, torch.round(y * 127.0 / top), 0.0), top / 127.0
        return {"y": ((codes @ t["w8"].float().t()) * scale * t["s8"] + t["b"].float()).to(dt), "h": h.to(dt)}
    if kind == "norm":
        h, w = t["x"].detach().float(), t["w"].float()
        if case["residual"]:
            h = h + t["r"].float()
        y, inv = _norm(h, w)
        out = {"y": y.to(dt)}
        if case["residual"]:
            out["h"] = h.to(dt)
        if case["train"]:
            gy, n = t["gy"].float(), h * inv
            d = gy * w
            dx = (d - n * (d * n).mean(-1, keepdim=True)) * inv
            if case["residual"]:
                dx = dx + t["gh"].float()
            out.update(dx=dx.to(dt), dw=(gy * n).flatten(0, -2).sum(0).to(dt))
            if case["residual"]:
                out["dr"] = out["dx"]
        return out
    of = torch.repeat_interleave(torch.arange(len(_sections(case)), device=t["pos"].device), torch.tensor(_sections(case), device=t["pos"].device))
    angle = t["pos"].double()[..., of] * t["freqs"]
    cos, sin = (f(angle).float().unsqueeze(-2) for f in (torch.cos, torch.sin))  # one for all heads
    out = {n: _turn(t[n].float(), cos, sin, case["interleaved"]).to(dt) for n in "qk"}
    if case["train"]:
        out.update({"d" + n: _turn(t["g" + n].float(), cos, -sin, case["interleaved"]).to(dt) for n in "qk"})
    return out


def _turn(x, cos, sin, interleaved):
    p = cos.shape[-1]
    a, b = (x[..., : 2 * p : 2], x[..., 1 : 2 * p : 2]) if interleaved else (x[..., :p], x[..., p : 2 * p])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((turned, x[..., 2 * p :]), -1)


# ---- the same in 64 bits, from the definitions ----------------------------------------------------------------------
def _exact_int8(v):
    """The values that 8-bit rows of v keep: whole steps of a 127th of the largest magnitude."""
    step = v.abs().max(dim=-1, keepdim=True).values / 127
    n = torch.where(step > 0, torch.round(v / step.clamp(min=torch.finfo(torch.float64).tiny)), torch.zeros_like(v))
    # a quotient by the rounded step may sit on either side of a border: settled by the exact products around it
    twice = 254 * v - 2 * n * step * 127
    n = n + (twice > step * 127).double() - (twice < -step * 127).double()
    half = (twice.abs() == step * 127) & (n.remainder(2) == 1)
    n = torch.where(half, n + torch.sign(twice), n)
    return n, step


def exact(case, seed):
    t = {k: v.double() if v.is_floating_point() else v for k, v in _inputs(case, seed).items()}
    kind = case["kind"]
    if kind == "quantize":
        n, step = _exact_int8(t["x"])
        return {"y": n * step}
    if kind in ("linear", "norm_linear"):
        w = t["w8"].double() * t["s8"].view(-1, 1)
        if kind == "linear":
            x, out = t["x"], {}
        else:
            h = t["x"] + t["r"]
            out = {"h": h}
            x = t["w"] * h / torch.sqrt(h.pow(2).sum(-1, keepdim=True) / h.shape[-1] + EPS)
        n, step = _exact_int8(x)
        out = {"y": torch.addmm(t["b"], n * step, w.t()), **out}
        if case.get("train"):
            out.update(dx=torch.mm(t["gy"], w), db=t["gy"].sum(0))
        return out
    if kind == "norm":
        h = t["x"][:, 0] if "heads" in case else t["x"]
        h = h + t["r"] if case["residual"] else h
        size = torch.sqrt(h.pow(2).sum(-1, keepdim=True) / h.shape[-1] + EPS)
        out = {"y": t["w"] * h / size}
        if case["residual"]:
            out["h"] = h
        if case["train"]:
            gh = t["gy"] * t["w"]
            dx = gh / size - h * (gh * h).sum(-1, keepdim=True) / (h.shape[-1] * size.pow(3))
            dx = dx + t["gh"] if case["residual"] else dx
            out.update(dx=dx, dw=(t["gy"] * h / size).reshape(-1, h.shape[-1]).sum(0))
            if case["residual"]:
                out["dr"] = dx
        return out
    parts, at = [], 0
    for a, n in enumerate(_sections(case)):
        parts.append(t["pos"][..., a : a + 1].double() * t["freqs"][at : at + n])
        at += n
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=t["q"].device), torch.cat(parts, -1)).unsqueeze(-2)

    def turned(x, by):
        y = x.clone()
        one, two = (slice(0, 2 * at, 2), slice(1, 2 * at, 2)) if case["interleaved"] else (slice(0, at), slice(at, 2 * at))
        z = torch.complex(x[..., one].contiguous(), x[..., two].contiguous()) * by
        y[..., one], y[..., two] = z.real, z.imag
        return y

    out = {n: turned(t[n], turn) for n in "qk"}
    if case["train"]:
        out.update({"d" + n: turned(t["g" + n], turn.conj()) for n in "qk"})
    return out


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case):
    e, kind = SIZE[case["dtype"]], case["kind"]
    if kind == "quantize":  # read, kept in 8 bits, and written back
        n = case["rows"] * case["cols"]
        return {"bytes": 2 * e * n + n + 4 * case["rows"], "flops": 6 * n}
    if kind in ("linear", "norm_linear"):
        m, i, o, t = case["tokens"], case["fin"], case["fout"], 1 + case.get("train", False)
        more = e * (2 * m * i + i) if kind == "norm_linear" else 0  # the residual, the new one, the norm's weight
        return {"bytes": t * e * (m * i + m * o + o) + o * i + 4 * o + more, "flops": t * 2 * m * i * o}
    if kind == "norm":
        n = math.prod(_rows(case))
        side = 4 if case["residual"] else 2  # x and y; the residual and the sum
        back = side - (1 if case["residual"] else 0)  # their gradients: x and the residual share one
        return {"bytes": e * (n * (side + (back if case["train"] else 0)) + case["cols"] * (2 if case["train"] else 1)), "flops": n * (14 if case["train"] else 5)}
    s = case["frames"] * case["height"] * case["width"]
    n = case["batch"] * s * (case["heads"] + case["kv"]) * case["dim"]
    a = len(_sections(case))
    return {"bytes": e * n * (4 if case["train"] else 2) + 8 * a * s * (case["batch"] if case["far"] else 1), "flops": 3 * n * (2 if case["train"] else 1)}
