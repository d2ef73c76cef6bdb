"""The operators of a frozen 4-bit base and of attention with a learned relative position bias, as cases to measure:
inputs, one pass through an operator, what the pass cannot do without, and its value in 64 bits.

  quantize   torch_vulkan.quantize_mxfp4 and dequant_mxfp4: microscaled 4-bit floating point, blocks of 32
  linear     torch_vulkan.mxfp4_linear: 16-bit rows times frozen 4-bit weights, and the rows' and the bias's gradients
  product    the same with quantize_input=True: the rows are quantised too and the product runs on 4-bit operands
  attention  torch_vulkan.relative_bias_attention: softmax(scale q k^T + table[bucket(j - i)]) v, and its gradients

`own` false: the operators written out in elementary torch operations in 32 bits on the GPU; `own` true: the calls that
a program makes of them on the "vk" device.  Sizes are those of this repository's tests and benchmark (2048 and 8192
wide blocks, 77-token text, 512-wide models, odd image token counts) and generic ones around them."""

import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # a frozen MLP weight is packed when the model is loaded, and unpacked where a merge needs it whole
        {"name": "quantize_weight", "kind": "quantize", "dtype": "bf16", "rows": 8192, "cols": 2048},
        # an fp32 checkpoint's weight whose rows end inside a block
        {"name": "quantize_ragged", "kind": "quantize", "dtype": "f32", "rows": 517, "cols": 1000},
        # one conditioning vector through a frozen layer: latency and the weights' bytes
        {"name": "linear_token", "kind": "linear", "dtype": "bf16", "tokens": 1, "fin": 2048, "fout": 8192, "train": False},
        # the captions of four images (4 x 77 tokens) through a frozen projection, both directions
        {"name": "linear_text", "kind": "linear", "dtype": "f16", "tokens": 308, "fin": 2048, "fout": 2048, "train": True},
        # a frozen MLP layer under image tokens, both directions
        {"name": "linear_image", "kind": "linear", "dtype": "bf16", "tokens": 4096, "fin": 2048, "fout": 8192, "train": True},
        # a few rows, quantised on the way in
        {"name": "product_rows", "kind": "product", "dtype": "bf16", "tokens": 16, "fin": 2048, "fout": 8192, "train": False},
        # the tokens of an odd aspect bucket (60 x 67) on 4-bit operands, both directions
        {"name": "product_image", "kind": "product", "dtype": "bf16", "tokens": 4020, "fin": 2048, "fout": 8192, "train": True},
        # a text encoder's layer over padded 77-token captions
        {"name": "attn_text", "kind": "attention", "dtype": "bf16", "batch": 4, "heads": 12, "q": 77, "k": 77, "dim": 64,
         "buckets": 32, "distance": 128, "causal": False, "mask": True, "train": True},
        # the same over padded 512-token prompts
        {"name": "attn_prompt", "kind": "attention", "dtype": "bf16", "batch": 4, "heads": 16, "q": 512, "k": 512, "dim": 64,
         "buckets": 32, "distance": 128, "causal": False, "mask": True, "train": True},
        # a causal decoder's layer over a long odd sequence
        {"name": "attn_long_causal", "kind": "attention", "dtype": "f16", "batch": 1, "heads": 8, "q": 4020, "k": 4020, "dim": 128,
         "buckets": 32, "distance": 128, "causal": True, "mask": False, "train": True},
        # an encoder kept in full precision
        {"name": "attn_f32", "kind": "attention", "dtype": "f32", "batch": 1, "heads": 16, "q": 1040, "k": 1040, "dim": 64,
         "buckets": 64, "distance": 256, "causal": False, "mask": False, "train": True},
        # one new token of each of eight sequences against their keys
        {"name": "attn_token", "kind": "attention", "dtype": "bf16", "batch": 8, "heads": 16, "q": 1, "k": 4096, "dim": 64,
         "buckets": 32, "distance": 128, "causal": True, "mask": True, "train": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):  # full-precision products count eightfold
    w = work(case)
    return w["flops"] * (8 if case["dtype"] == "f32" else 1) + w["bytes"] * 100


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(("quantize", "linear", "linear", "product", "attention", "attention", "attention"))
        half = rng.choice(("bf16", "f16"))
        any3 = rng.choice(("bf16", "f16", "f32"))
        if kind == "quantize":
            c = {"dtype": any3, "rows": _log(rng, 64, 16384), "cols": rng.choice((32 * _log(rng, 2, 256), _log(rng, 50, 8192)))}
        elif kind in ("linear", "product"):
            step = rng.choice((64, 64, 64, 8, 1))  # output widths are mostly multiples of 64
            c = {"dtype": half, "tokens": _log(rng, 1, 8192), "fin": 32 * _log(rng, 8, 256), "fout": _log(rng, 256, 8192) // step * step,
                 "train": rng.random() < 0.5}
        else:
            causal, train = rng.random() < 0.4, rng.random() < 0.7
            k = _log(rng, 24, 4096)
            c = {"dtype": any3, "batch": rng.randint(1, 8), "heads": rng.randint(1, 24), "q": k if train else rng.choice((k, 1, 1, rng.randint(1, 24))),
                 "k": k, "dim": rng.choice((32, 40, 64, 64, 64, 80, 128)), "buckets": rng.choice((32, 32, 64, 20)),
                 "distance": rng.choice((128, 128, 256, 100)), "causal": causal, "mask": rng.random() < 0.5, "train": train}
        c = {"kind": kind, **c}
        if _cost(c) <= most:
            return c


# ---- microscaled 4-bit floating point, in 32 bits -----------------------------------------------------------------
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _times_2(v, e):
    """v * 2^e, exactly wherever the result has no more bits than v: two factors, neither of them subnormal."""
    half = e // 2
    return v * ((half + 127) << 23).int().view(torch.float32) * ((e - half + 127) << 23).int().view(torch.float32)


def _blocks(x):
    """x [rows, cols] as fp32 [rows, blocks, 32], its last block filled up with zeros."""
    rows, cols = x.shape
    return torch.nn.functional.pad(x.float(), (0, -cols % 32)).view(rows, -1, 32)


def _quantize(x):
    """Codes [rows, blocks, 32] (0..15, bit 3 the sign) and exponents [rows, blocks] of x [rows, cols]."""
    b = _blocks(x)
    top = b.abs().amax(-1)
    e = torch.where(top > 0, torch.frexp(top).exponent - 3, -127).clamp(min=-127)  # floor(log2 top) - 2
    v = _times_2(b, -e.unsqueeze(-1))
    m = v.abs()
    code = (m > 0.25).int() + (m >= 0.75) + (m > 1.25) + (m >= 1.75) + (m > 2.5) + (m >= 3.5) + (m > 5.0)
    return code + 8 * torch.signbit(v), e


def _values(code, e, cols):
    """The fp32 values that codes and exponents stand for, [rows, cols]."""
    v = torch.tensor(_E2M1, device=code.device)[(code & 7).long()]
    v = torch.where(code >= 8, -v, v)
    return _times_2(v, e.unsqueeze(-1)).flatten(1)[:, :cols]


def _pack(code, e, cols):
    """As stored: two codes a byte, the even element low, [rows, ceil(cols / 2)]; a scale byte a block, [rows, blocks]."""
    c = code.flatten(1)
    return (c[:, 0::2] | (c[:, 1::2] << 4))[:, : (cols + 1) // 2].to(torch.uint8).contiguous(), (e + 127).to(torch.uint8)


def _unpack(packed, scale, cols):
    code = torch.stack((packed & 15, packed >> 4), -1).flatten(1).int()
    code = torch.nn.functional.pad(code, (0, scale.shape[1] * 32 - code.shape[1])).view(code.shape[0], -1, 32)
    return _values(code, scale.int() - 127, cols)


# ---- inputs -------------------------------------------------------------------------------------------------------
_GRADS = {"linear": ("x", "b"), "product": ("x", "b"), "attention": ("q", "k", "v", "table")}


def _inputs(case, seed):
    """Everything that a pass reads, from the seed alone: activations and output gradients ~ N(0, 1), weights ~ N(0, 0.02)
    with a scale of its own in each row, biases of a trained table's size, captions of different lengths."""
    dev = "cuda" if torch.cuda.is_available() else "cpu"
    g = torch.Generator(dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def r(*shape, scale=1.0):
        return torch.randn(shape, generator=g, device=dev).mul_(scale).to(dt)

    def weight(o, i):
        return r(o, i, scale=0.02) * torch.exp(torch.randn((o, 1), generator=g, device=dev) * 0.5).to(dt)

    if case["kind"] == "quantize":
        return {"x": weight(case["rows"], case["cols"])}
    if case["kind"] in ("linear", "product"):
        m, i, o = case["tokens"], case["fin"], case["fout"]
        codes, scale = _pack(*_quantize(weight(o, i)), i)
        t = {"x": r(m, i), "codes": codes, "scale": scale, "b": r(o, scale=0.02)}
        if case["train"]:
            t["g"] = r(m, o)
        return t
    n, h, d = case["batch"], case["heads"], case["dim"]  # token-major, as a model's projections leave them
    t = {"q": r(n, case["q"], h, d), "k": r(n, case["k"], h, d), "v": r(n, case["k"], h, d), "table": r(case["buckets"], h)}
    if case["mask"]:  # padded at the end
        length = torch.randint(max(1, case["k"] // 2), case["k"] + 1, (n, 1), generator=g, device=dev)
        t["mask"] = torch.arange(case["k"], device=dev) < length
    if case["train"]:
        t["g"] = r(n, case["q"], h, d)
    return t


def prepare(case, seed):
    t = _inputs(case, seed)
    if own:  # a program that uses the operators has its tensors on the framework's device
        path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "torch-vulkan_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        import torch_vulkan

        torch_vulkan.set_inline_backward()  # as a training loop on this device does once, on its own thread
        t = {k: v.cpu().to("vk") for k, v in t.items()}
        for n in _GRADS.get(case["kind"], ()) if case.get("train") else ():
            t[n].requires_grad_(True)
    return {"case": case, "t": t}


# ---- one pass -----------------------------------------------------------------------------------------------------
def run(state):
    case, t = state["case"], state["t"]
    return _own(case, t) if own else _plain(case, t)


def _own(case, t):
    import torch_vulkan as tv

    if case["kind"] == "quantize":
        codes, scale = tv.quantize_mxfp4(t["x"])
        return {"y": tv.dequant_mxfp4(codes, scale, DTYPES[case["dtype"]], cols=case["cols"])}
    if case["kind"] in ("linear", "product"):
        y = tv.mxfp4_linear(t["x"], t["codes"], t["scale"], t["b"], quantize_input=case["kind"] == "product")
    else:
        q, k, v = (t[n].transpose(1, 2) for n in "qkv")
        y = tv.relative_bias_attention(q, k, v, t["table"], key_mask=t.get("mask"), causal=case["causal"], max_distance=case["distance"],
                                       query_offset=_offset(case)).transpose(1, 2)
    if not case["train"]:
        return {"y": y}
    names = _GRADS[case["kind"]]
    return {"y": y.detach(), **{"d" + n: d for n, d in zip(names, torch.autograd.grad(y, [t[n] for n in names], t["g"]))}}


def _offset(case):
    """Position of the first query: new tokens come last."""
    return case["k"] - case["q"]


def _plain(case, t):
    dt = DTYPES[case["dtype"]]
    if case["kind"] == "quantize":
        return {"y": _values(*_quantize(t["x"]), case["cols"]).to(dt)}
    if case["kind"] in ("linear", "product"):
        w = _unpack(t["codes"], t["scale"], case["fin"])
        x = _values(*_quantize(t["x"]), case["fin"]) if case["kind"] == "product" else t["x"].float()
        out = {"y": (x @ w.t() + t["b"].float()).to(dt)}
        if case["train"]:
            g = t["g"].float()
            out.update(dx=(g @ w).to(dt), db=g.sum(0).to(dt))
        return out
    q, k, v = (t[n].float().transpose(1, 2).contiguous() for n in "qkv")
    off, nq, nk = _offset(case), case["q"], case["k"]
    dist = torch.arange(1 - nq, nk, device=q.device) - off  # of each diagonal j - i, from the bottom left corner
    bucket = _buckets(dist, case["buckets"], case["distance"], case["causal"])
    # a head's bias by diagonal, and the score matrix's view of it: row i reads from diagonal nq - 1 - i on
    bias = t["table"].float()[bucket].t().contiguous()
    at = torch.arange(nk, device=q.device) + (nq - 1 - torch.arange(nq, device=q.device)).unsqueeze(1)
    scale = 1.0 / math.sqrt(case["dim"])
    s = torch.matmul(q, k.transpose(2, 3).contiguous()) * scale + bias[:, at]
    seen = dist[at] <= 0 if case["causal"] else torch.ones_like(at, dtype=torch.bool)
    seen = seen & t["mask"][:, None, None, :] if "mask" in t else seen.expand(s.shape[0], 1, nq, nk)
    s = torch.where(seen, s, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = torch.matmul(p, v)
    out = {"y": o.transpose(1, 2).to(dt)}
    if case["train"]:
        do = t["g"].float().transpose(1, 2).contiguous()
        dp = torch.matmul(do, v.transpose(2, 3).contiguous())
        ds = p * (dp - (do * o).sum(-1, keepdim=True))
        out["dq"] = (torch.matmul(ds, k) * scale).transpose(1, 2).to(dt)
        out["dk"] = (torch.matmul(ds.transpose(2, 3).contiguous(), q) * scale).transpose(1, 2).to(dt)
        out["dv"] = torch.matmul(p.transpose(2, 3).contiguous(), do).transpose(1, 2).to(dt)
        # the sums over diagonals: each row shifted by one against the one below it, then summed in 64 bits
        by = torch.nn.functional.pad(ds.sum(0).flip(1), (0, nq)).flatten(1)[:, : -nq].view(-1, nq, nq + nk - 1).double().sum(1)
        hot = (bucket.unsqueeze(1) == torch.arange(case["buckets"], device=q.device)).double()
        out["dtable"] = (by @ hot).t().contiguous().to(dt)
    return out


def _buckets(dist, buckets, distance, causal):
    if causal:
        side, n, nb = 0, (-dist).clamp(min=0), buckets
    else:
        nb = buckets // 2
        side, n = (dist > 0).long() * nb, dist.abs()
    e = nb // 2
    far = torch.log(n.clamp(min=e).double() / e) / math.log(distance / e) * (nb - e)
    far = e + torch.floor(far + 1e-9).long()  # a border is reached where the logarithms meet
    return side + torch.where(n < e, n, far.clamp(max=nb - 1))


# ---- the same in 64 bits, from the definitions ----------------------------------------------------------------------
def _power(e):
    """2^e in 64 bits, for whole e in the normal range."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_mxfp4(x):
    """The nearest representable values of x [rows, cols], ties to the even code."""
    rows, cols = x.shape
    b = torch.zeros((rows, (cols + 31) // 32 * 32), dtype=torch.float64, device=x.device)
    b[:, :cols] = x.double()
    b = b.view(rows, -1, 32)
    top = b.abs().amax(-1, keepdim=True).contiguous()
    e = ((top.view(torch.int64) >> 52) - 1023 - 2).clamp(min=-127)
    unit = _power(e)
    v = b / unit
    step = torch.where(v.abs() < 2, 0.5, torch.where(v.abs() < 4, 1.0, 2.0))
    return ((torch.round(v / step) * step).clamp(-6, 6) * unit).reshape(rows, -1)[:, :cols]


def _exact_unpack(codes, scale, cols):
    c = torch.empty((codes.shape[0], 2 * codes.shape[1]), dtype=torch.int64, device=codes.device)
    c[:, 0::2], c[:, 1::2] = codes % 16, codes // 16
    exp, man = (c % 8) // 2, (c % 2).double()
    mag = torch.where(exp > 0, (1 + man / 2) * _power(exp - 1), man / 2)
    v = torch.where(c >= 8, -mag, mag)[:, :cols]
    return v * _power(scale.long() - 127).repeat_interleave(32, 1)[:, :cols]


def _exact_bucket(r, buckets, distance, causal):
    nb = buckets if causal else buckets // 2
    side = nb if not causal and r > 0 else 0
    n = max(-r, 0) if causal else abs(r)
    e = nb // 2
    if n < e:
        return side + n
    k = 0  # the most k <= nb - e - 1 with (n / e)^(nb - e) >= (distance / e)^k, in whole numbers
    while k + 1 < nb - e and n ** (nb - e) * e ** (k + 1) >= distance ** (k + 1) * e ** (nb - e):
        k += 1
    return side + e + k


def exact(case, seed):
    t = _inputs(case, seed)
    if case["kind"] == "quantize":
        return {"y": _exact_mxfp4(t["x"])}
    if case["kind"] in ("linear", "product"):
        w = _exact_unpack(t["codes"], t["scale"], case["fin"])
        x = _exact_mxfp4(t["x"]) if case["kind"] == "product" else t["x"].double()
        out = {"y": torch.addmm(t["b"].double(), x, w.t())}
        if case["train"]:
            out.update(dx=torch.mm(t["g"].double(), w), db=t["g"].double().sum(0))
        return out
    nq, nk, off, scale = case["q"], case["k"], _offset(case), case["dim"] ** -0.5
    dev = t["q"].device
    of = torch.tensor([_exact_bucket(r - off, case["buckets"], case["distance"], case["causal"]) for r in range(1 - nq, nk)], device=dev)
    i, j = torch.arange(nq, device=dev).view(-1, 1), torch.arange(nk, device=dev).view(1, -1)
    where = of[j - i + nq - 1]
    gone = (j > i + off) if case["causal"] else torch.zeros_like(where, dtype=torch.bool)
    out = {"y": torch.empty(t["q"].shape, dtype=torch.float64, device=dev)}
    if case["train"]:
        out.update({"d" + n: torch.zeros(t[n].shape, dtype=torch.float64, device=dev) for n in ("q", "k", "v", "table")})
    for b in range(case["batch"]):
        no = gone | ~t["mask"][b].view(1, -1) if "mask" in t else gone
        for h in range(case["heads"]):
            q, k, v, table = t["q"][b, :, h].double(), t["k"][b, :, h].double(), t["v"][b, :, h].double(), t["table"][:, h].double()
            p = torch.softmax((torch.mm(q, k.t()) * scale + table[where]).masked_fill(no, -math.inf), -1)
            out["y"][b, :, h] = o = torch.mm(p, v)
            if case["train"]:
                g = t["g"][b, :, h].double()
                ds = p * (torch.mm(g, v.t()) - (g * o).sum(-1, keepdim=True))
                out["dq"][b, :, h], out["dk"][b, :, h], out["dv"][b, :, h] = torch.mm(ds, k) * scale, torch.mm(ds.t(), q) * scale, torch.mm(p.t(), g)
                out["dtable"][:, h] += torch.bincount(where.flatten(), ds.flatten(), case["buckets"])
    return out


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case):
    e = SIZE[case["dtype"]]
    if case["kind"] == "quantize":  # read, packed, and written back
        n = case["rows"] * case["cols"]
        return {"bytes": 2 * e * n + case["rows"] * ((case["cols"] + 1) // 2 + (case["cols"] + 31) // 32), "flops": 10 * n}
    if case["kind"] in ("linear", "product"):
        m, i, o, t = case["tokens"], case["fin"], case["fout"], 1 + case["train"]
        return {"bytes": t * e * (m * i + m * o + o) + o * i // 2 + o * (i // 32), "flops": t * 2 * m * i * o}
    n, h, q, k, d = (case[x] for x in ("batch", "heads", "q", "k", "dim"))
    seen = q * k - q * (q - 1) // 2 if case["causal"] else q * k  # pairs, whatever the padding
    side = 4 if case["train"] else 2  # q, k, v, o, and their gradients
    return {"bytes": e * (n * h * d * (q + k) * side + side // 2 * case["buckets"] * h) + (n * k if case["mask"] else 0),
            "flops": (7 if case["train"] else 2) * 2 * n * h * seen * d}
