"""Attention with a learned relative position bias against its definition in float64, with masks, causal forms, offsets and
odd sizes, and its gradients against the formula's, which the first test holds against differences.

Tolerances, per element (u = finfo(dtype).eps / 2; f = 2^-24, fp32's):
  * logits: fp32 sums of D exact products off by at most ds = D f scale |q| |k| (+ the bias's and the logsumexp's own
    rounding), so P is off by a factor of at most ep = 4 (max ds + 4 f (1 + max |s|));
  * o: (ep + u) P |v| for P (rounded to the type) and one rounding, u |o|;
  * delta = rowsum(o dO) from the stored o: edelta = |dO| (error of o); dP: D f |dO| |v|;
  * dS: P (edelta + edP) + ep |dS|; dq, dk, dv: that through |k|, |q|, |dO| with u more for the rounded P and dS, one
    rounding; the table's gradient: its sum over the bucket, fp32 summation n f, one rounding.
f16 adds half its smallest subnormal for every rounded P, dS and output.  Sums over n terms add n f of their size."""

import math

import numpy as np
import pytest
import torch

import torch_vulkan
from torch_vulkan import abi

vk = torch.device("vk")
HALF = [torch.bfloat16, torch.float16]
DTYPES = [torch.float32] + HALF


def bucket(r, buckets, distance, causal):
    """The definition, in whole numbers."""
    nb = buckets if causal else buckets // 2
    side = nb if not causal and r > 0 else 0
    n = max(-r, 0) if causal else abs(r)
    e = nb // 2
    if n < e:
        return side + n
    t = 0
    while t + 1 < nb - e and n ** (nb - e) * e ** (t + 1) >= distance ** (t + 1) * e ** (nb - e):
        t += 1
    return side + e + t


def pairs(c):
    """Bucket of every pair [Sq, Sk] and whether its key may be seen [B, Sq, Sk]."""
    r = np.arange(c["Sk"])[None, :] - np.arange(c["Sq"])[:, None] - c["off"]
    lo = int(r.min())
    of = np.array([bucket(x, c["buckets"], c["distance"], c["causal"]) for x in range(lo, int(r.max()) + 1)])
    seen = np.broadcast_to(r <= 0 if c["causal"] else np.ones_like(r, bool), (c["B"], c["Sq"], c["Sk"])).copy()
    if c["mask"] is not None:
        seen &= c["mask"][:, None, :]
    seen &= ~np.isin(of[r - lo], c.get("hide", []))
    return of[r - lo], seen


def inputs(c, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)

    def r(*shape):
        return torch.randn(shape, generator=g).to(dtype)

    B, H, D = c["B"], c["H"], c["D"]
    return {"q": r(B, H, c["Sq"], D), "k": r(B, H, c["Sk"], D), "v": r(B, H, c["Sk"], D), "table": r(c["buckets"], H), "g": r(B, H, c["Sq"], D)}


def oracle(t, c, dtype):
    """Float64 results and what they may be off by."""
    q, k, v, table, g = (t[n].double().numpy() for n in ("q", "k", "v", "table", "g"))
    of, seen = pairs(c)
    seen = seen[:, None]
    if c["mask"] is not None:  # what a masked key holds plays no part
        k, v = (np.where(c["mask"][:, None, :, None], x, 0.0) for x in (k, v))
    scale = c["scale"] if c["scale"] is not None else 1 / math.sqrt(c["D"])
    T = lambda x: x.swapaxes(-1, -2)  # noqa: E731
    s = scale * (q @ T(k)) + table.T[:, of][None]
    s = np.where(seen, s, -np.inf)
    m = s.max(-1, keepdims=True)
    p = np.exp(s - np.where(np.isfinite(m), m, 0.0))
    z = p.sum(-1, keepdims=True)
    p = np.divide(p, z, out=np.zeros_like(p), where=z > 0)
    o = p @ v
    dp = g @ T(v)
    ds = p * (dp - (g * o).sum(-1, keepdims=True))
    res = {"o": o, "q": scale * (ds @ k), "k": scale * (T(ds) @ q), "v": T(p) @ g}
    sums = ds.sum(0).reshape(c["H"], -1)
    res["table"] = np.stack([np.bincount(of.ravel(), x, c["buckets"]) for x in sums], 1)

    f, info = 2.0**-24, torch.finfo(dtype)
    u, tiny = info.eps / 2, info.smallest_normal * info.eps / 2
    A = np.abs
    fin = np.where(seen, A(s), 0.0)
    ds_err = c["D"] * f * scale * float((A(q) @ T(A(k))).max(initial=0.0))
    ep = 4 * (ds_err + 4 * f * (1 + float(fin.max(initial=0.0))))
    n = max(c["Sq"], c["Sk"])
    up = u + n * f
    rp = up if dtype != torch.float32 else n * f  # P and dS are rounded in 16 bits only
    nothing = tiny if dtype == torch.float16 else 0.0
    tol = {"o": (ep + rp) * (p @ A(v)) + nothing * A(v).sum(-2, keepdims=True)}
    tol["o"] = 1.1 * (tol["o"] + u * A(o)) + tiny
    edp = (A(g) * tol["o"]).sum(-1, keepdims=True) + c["D"] * f * ((A(g) @ T(A(v))) + (A(g) * A(o)).sum(-1, keepdims=True))
    eds = p * edp + ep * A(ds)
    r = eds + rp * A(ds)
    tol["q"] = 1.1 * (scale * (r @ A(k) + nothing * A(k).sum(-2, keepdims=True)) + u * A(res["q"])) + tiny
    tol["k"] = 1.1 * (scale * (T(r) @ A(q) + nothing * A(q).sum(-2, keepdims=True)) + u * A(res["k"])) + tiny
    tol["v"] = 1.1 * ((ep + rp) * (T(p) @ A(g)) + nothing * A(g).sum(-2, keepdims=True) + u * A(res["v"])) + tiny
    terms = c["B"] * c["Sq"] * c["Sk"]
    loose = (eds + min(terms, 4096) * f * A(ds)).sum(0).reshape(c["H"], -1)  # sums of at most 4096 in a row, then in levels
    tol["table"] = 1.1 * (np.stack([np.bincount(of.ravel(), x, c["buckets"]) for x in loose], 1) + u * A(res["table"])) + tiny
    return res, tol


def case(B=1, H=2, Sq=64, Sk=64, D=64, buckets=32, distance=128, causal=False, off=0, mask=None, scale=None, seed=0):
    g = np.random.default_rng(seed)
    m = None
    if mask == "random":
        m = g.random((B, Sk)) < 0.6
    elif mask == "tail":
        m = np.arange(Sk)[None] < g.integers(1, Sk + 1, (B, 1))
    elif mask == "empty":  # the first sequence has no key at all
        m = g.random((B, Sk)) < 0.5
        m[0] = False
    elif mask == "one":
        m = np.zeros((B, Sk), bool)
        m[np.arange(B), g.integers(0, Sk, B)] = True
    elif mask == "late":  # only the last keys
        m = np.broadcast_to(np.arange(Sk)[None] >= Sk - 3, (B, Sk)).copy()
    return dict(B=B, H=H, Sq=Sq, Sk=Sk, D=D, buckets=buckets, distance=distance, causal=causal, off=off, mask=m, scale=scale)


CASES = {
    "one_pair": case(Sq=1, Sk=1, D=8), "one_key": case(Sq=40, Sk=1), "one_query": case(Sq=1, Sk=33, off=32),
    "tile": case(Sq=32, Sk=32, D=32), "below": case(Sq=31, Sk=63), "above": case(Sq=33, Sk=65, D=40), "odd": case(B=2, H=3, Sq=77, Sk=77),
    "far": case(Sq=300, Sk=420, buckets=20, distance=100, off=50), "few_buckets": case(Sq=70, Sk=150, buckets=4, distance=3),
    "wide": case(H=1, Sq=200, Sk=1500, D=16, buckets=512, distance=1024, off=700), "causal": case(Sq=200, Sk=200, causal=True, D=72),
    "causal_few": case(Sq=150, Sk=150, causal=True, buckets=2, distance=2), "causal_cache": case(B=2, Sq=5, Sk=300, causal=True, off=295),
    "causal_empty_rows": case(Sq=100, Sk=100, causal=True, off=-40), "causal_all_seen": case(Sq=20, Sk=50, causal=True, off=500),
    "causal_none": case(Sq=20, Sk=50, causal=True, off=-20), "beyond": case(Sq=50, Sk=50, off=4000), "behind": case(Sq=50, Sk=50, off=-4000),
    "random": case(B=3, Sq=100, Sk=200, mask="random"), "tail": case(B=4, Sq=130, Sk=130, mask="tail"), "empty": case(B=2, Sq=70, Sk=90, mask="empty"),
    "one_left": case(B=3, Sq=70, Sk=300, mask="one"), "late": case(B=2, Sq=64, Sk=500, mask="late", D=128),
    "causal_masked": case(B=3, Sq=140, Sk=140, causal=True, mask="random"), "d1": case(Sq=20, Sk=40, D=1), "d100": case(Sq=70, Sk=70, D=100),
    "d128": case(Sq=160, Sk=257, D=128, scale=0.3), "d96": case(Sq=65, Sk=130, D=96, scale=1.0), "steep": case(Sq=64, Sk=64, scale=3.0),
    "flat": case(Sq=64, Sk=64, scale=1e-3), "groups2": case(B=4, H=64, Sq=50, Sk=70, D=24), "groups4": case(B=8, H=64, Sq=70, Sk=40, D=16),
    "groups4_causal": case(B=8, H=64, Sq=70, Sk=70, D=16, causal=True, mask="tail"), "split": case(B=1, H=1, Sq=1, Sk=5000, off=4999, causal=True),
    "split_masked": case(B=2, H=3, Sq=9, Sk=3000, off=2991, mask="tail"), "split_empty": case(B=2, H=1, Sq=3, Sk=2100, mask="empty"),
    "wide_d128": case(H=2, Sq=40, Sk=300, D=128, buckets=64, distance=1024, off=200),
    "groups2_d128": case(B=2, H=64, Sq=100, Sk=90, D=80, mask="tail"), "groups4_d128": case(B=8, H=64, Sq=40, Sk=70, D=72),
    "few_d128": case(B=2, H=2, Sq=2, Sk=700, D=128, off=698, causal=True), "split_d112": case(B=2, H=1, Sq=1, Sk=3001, D=112, off=3000, mask="tail"),
}


def tensors(t, c):
    out = {n: x.to(vk) for n, x in t.items()}
    out["mask"] = None if c["mask"] is None else torch.from_numpy(c["mask"]).to(vk)
    return out


def call(t, c, **kw):
    return torch_vulkan.relative_bias_attention(t["q"], t["k"], t["v"], t["table"], key_mask=t["mask"], causal=c["causal"], scale=c["scale"],
                                                max_distance=c["distance"], query_offset=c["off"], **kw)


def close(got, ref, tol, what):
    d = np.abs(got.detach().cpu().double().numpy() - ref)
    assert d.shape == ref.shape and (d <= tol).all(), (what, float(np.nanmax(d / tol)), np.unravel_index(np.nanargmax(d / tol), d.shape), int(np.isnan(d).sum()))


def grads(t, c, g=None):
    leaves = [t[n].detach().requires_grad_() for n in ("q", "k", "v", "table")]
    y = call({**t, **dict(zip(("q", "k", "v", "table"), leaves))}, c)
    return y, dict(zip(("q", "k", "v", "table"), torch.autograd.grad(y, leaves, t["g"] if g is None else g)))


@pytest.mark.parametrize("name", ["odd", "causal_empty_rows", "few_buckets", "random"])
def test_the_formula_is_the_derivative(name):
    """The oracle's gradients against central differences of its forward pass, in float64 (truncation and rounding 1e-6)."""
    c = dict(CASES[name])
    t = {n: x.double() for n, x in inputs(c, torch.float32).items()}
    res, _ = oracle(t, c, torch.float32)
    rng = np.random.default_rng(0)
    for n in ("q", "k", "v", "table"):
        way = torch.from_numpy(rng.standard_normal(t[n].shape))
        h = 1e-5
        up, down = (float((oracle({**t, n: t[n] + x * way}, c, torch.float32)[0]["o"] * t["g"].numpy()).sum()) for x in (h, -h))
        want = float((res[n] * way.numpy()).sum())
        assert abs((up - down) / (2 * h) - want) <= 1e-6 * (1 + np.abs(res[n] * way.numpy()).sum())


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("buckets,distance", [(32, 128), (64, 256), (20, 100), (4, 2), (4, 3), (16, 16), (32, 17), (128, 1024), (256, 1000), (34, 50)])
def test_borders_are_the_definitions(buckets, distance, causal):
    import ctypes

    nb = buckets if causal else buckets // 2
    lib = ctypes.CDLL(abi._LIB_PATH)
    start = (ctypes.c_uint16 * 256)()
    got = lib.hrt_attn_rel_buckets(buckets, distance, int(causal), start)
    if distance <= nb // 2:
        assert got == -1
        return
    assert got == nb
    of = [bucket(-n, buckets, distance, causal) for n in range(1100)]
    for n in range(1100):
        assert of[n] == max(k for k in range(nb) if start[k] <= n)


def test_borders_refused():
    import ctypes

    lib, start = ctypes.CDLL(abi._LIB_PATH), (ctypes.c_uint16 * 256)()
    for buckets, distance, causal in ((1, 128, 1), (257, 512, 1), (3, 128, 0), (2, 128, 0), (514, 1024, 0), (32, 1025, 0), (32, 8, 0), (32, 16, 1), (-4, 9, 0), (0, 0, 0)):
        assert lib.hrt_attn_rel_buckets(buckets, distance, causal, start) == -1


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="vk tensor"):
        torch_vulkan.relative_bias_attention(*(torch.zeros(1, 1, 4, 8) for _ in range(3)), torch.zeros(32, 1))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", list(CASES))
def test_forward_and_gradients(name, dtype):
    c = CASES[name]
    t = inputs(c, dtype)
    if c["mask"] is not None:  # masked keys and values hold anything
        bad = torch.tensor([float("nan"), float("inf"), -float("inf")], dtype=dtype)
        at = torch.from_numpy(~c["mask"])[:, None, :, None]
        for n in ("k", "v"):
            t[n] = torch.where(at, bad[torch.arange(c["Sk"]) % 3][None, None, :, None], t[n])
    ref, tol = oracle(t, c, dtype)
    d = tensors(t, c)
    close(call(d, c), ref["o"], tol["o"], "o")
    y, got = grads(d, c)
    close(y, ref["o"], tol["o"], "o")
    for n, x in got.items():
        assert x.dtype == dtype
        close(x, ref[n], tol[n], n)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("low", [float("-inf"), "lowest"])
@pytest.mark.parametrize("far", [True, False])
@pytest.mark.parametrize("Sq,Sk,off", [(300, 300, 0), (3, 700, 697), (40, 2500, 2000)])
def test_a_table_that_hides(Sq, Sk, off, far, low, dtype):
    """Hidden buckets, the last of each direction (whole tiles) or nearer ones; every query sees others.  The oracle masks their
    pairs: f16's lowest value is an ordinary bias, but weighs exp(-65504 + 50) = 0 beside any other."""
    c = case(B=2, H=2, Sq=Sq, Sk=Sk, D=64, off=off, buckets=8, distance=16)
    hide = [3, 7] if far else [0, 5, 6]
    c["hide"] = hide
    t = inputs(c, dtype)
    ref, tol = oracle({**t, "table": t["table"].index_fill(0, torch.tensor(hide), 0.0)}, c, dtype)
    t["table"][hide] = torch.finfo(dtype).min if low == "lowest" else low
    d = tensors(t, c)
    close(call(d, c), ref["o"], tol["o"], "o")
    y, got = grads(d, c)
    close(y, ref["o"], tol["o"], "o")
    for n, x in got.items():
        close(x, ref[n], tol[n], n)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Sq", [1, 200])
def test_a_table_that_hides_everything(Sq, dtype):
    c = case(B=1, H=2, Sq=Sq, Sk=600, D=32, off=200)
    t = inputs(c, dtype)
    t["table"].fill_(float("-inf"))
    y, got = grads(tensors(t, c), c)
    assert not y.detach().cpu().any() and not any(x.cpu().any() for x in got.values())


@pytest.mark.gpu
def test_views_are_read_in_place_or_copied():
    """Token-major, head-broadcast, offset and strided operands give what contiguous ones do, gradients included."""
    c = case(B=2, H=3, Sq=70, Sk=70, D=64, mask="tail")
    t = tensors(inputs(c, torch.bfloat16), c)
    y0, g0 = grads(t, c)
    B, H, S, D = t["q"].shape
    forms = {
        "token_major": lambda x: x.transpose(1, 2).contiguous().transpose(1, 2),
        "wider_rows": lambda x: torch.cat([x, x], 3)[..., :D],
        "odd_offset": lambda x: torch.cat([torch.zeros(5, dtype=x.dtype, device=vk), x.flatten()])[5:].view(x.shape),
        "d_strided": lambda x: x.transpose(2, 3).contiguous().transpose(2, 3),
        "seq_strided": lambda x: torch.stack([x, x], 3)[:, :, :, 0],
    }
    for name, f in forms.items():
        y, g = grads({**t, **{n: f(t[n]) for n in "qkv"}}, c, f(t["g"]))
        assert torch.equal(y.cpu(), y0.cpu()), name
        for n in g:
            assert torch.equal(g[n].cpu(), g0[n].cpu()), (name, n)
    # one key head and one value head for all queries' heads: the gradient is the sum of the heads'
    one = {n: t[n][:, :1].detach() for n in "kv"}
    full = {**t, **{n: x.expand(B, H, S, D) for n, x in one.items()}}
    _, per_head = grads({**t, **{n: x.expand(B, H, S, D).contiguous() for n, x in one.items()}}, c)
    leaves = {n: x.clone().requires_grad_() for n, x in one.items()}
    y = call({**full, **{n: x.expand(B, H, S, D) for n, x in leaves.items()}}, c)
    y.backward(t["g"])
    for n, x in leaves.items():
        assert torch.equal(x.grad.cpu(), per_head[n].sum(1, keepdim=True).cpu()), n
    # one mask row for every sequence; a table that is not contiguous; a gradient broadcast from one value
    m = t["mask"][:1]
    want = call({**t, "mask": m.expand(B, S).contiguous()}, c).cpu()
    assert torch.equal(call({**t, "mask": m}, c).cpu(), want) and torch.equal(call({**t, "mask": m.expand(B, S)}, c).cpu(), want)
    assert torch.equal(call({**t, "table": t["table"].t().contiguous().t()}, c).cpu(), y0.cpu())
    ones = torch.ones((), dtype=torch.bfloat16, device=vk).expand(B, H, S, D)
    assert torch.equal(grads(t, c, ones)[1]["q"].cpu(), grads(t, c, ones.contiguous())[1]["q"].cpu())


@pytest.mark.gpu
def test_only_what_is_asked_for():
    c = case(B=1, H=2, Sq=40, Sk=50)
    t = tensors(inputs(c, torch.float16), c)
    _, all_of = grads(t, c)
    for n in ("q", "k", "v", "table"):
        leaf = t[n].detach().requires_grad_()
        (g,) = torch.autograd.grad(call({**t, n: leaf}, c), leaf, t["g"])
        assert torch.equal(g.cpu(), all_of[n].cpu()), n
    with torch.no_grad():
        assert not call({**t, "q": t["q"].requires_grad_()}, c).requires_grad


@pytest.mark.gpu
def test_nothing_to_attend_to():
    for B, Sq, Sk in ((0, 4, 4), (1, 0, 4), (1, 4, 0)):
        t = {"q": torch.ones(B, 2, Sq, 8), "k": torch.ones(B, 2, Sk, 8), "v": torch.ones(B, 2, Sk, 8), "table": torch.ones(32, 2)}
        leaves = {n: x.to(vk).requires_grad_() for n, x in t.items()}
        y = torch_vulkan.relative_bias_attention(*leaves.values())
        assert y.shape == (B, 2, Sq, 8) and not y.detach().cpu().any()
        y.sum().backward()
        assert all(x.grad.shape == x.shape and not x.grad.cpu().any() for x in leaves.values())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_same_bits_every_run(dtype):
    c = case(B=2, H=4, Sq=300, Sk=300, causal=True, mask="tail")
    t = tensors(inputs(c, dtype), c)
    y0, g0 = grads(t, c)
    for _ in range(5):
        y, g = grads(t, c)
        assert torch.equal(y.cpu(), y0.cpu()) and all(torch.equal(g[n].cpu(), g0[n].cpu()) for n in g)


@pytest.mark.gpu
def test_recorded_forward_and_backward():
    """Recorded while an eager graph of the same leaves lives; replayed between eager calls."""
    torch_vulkan.set_inline_backward()
    try:
        rt, out = abi.Runtime(), {}
        c = case(B=2, H=2, Sq=90, Sk=90, mask="tail")
        t = tensors(inputs(c, torch.bfloat16), c)
        leaves = {n: t[n].requires_grad_() for n in ("q", "k", "v", "table")}
        alive = call(t, c)

        def run():
            y = call(t, c)
            out["r"] = [y.detach(), *torch.autograd.grad(y, list(leaves.values()), t["g"])]

        run()
        want = [x.cpu() for x in out["r"]]
        gid = rt.graph(run)
        for _ in range(3):
            for x in out["r"]:
                x.zero_()
            rt.graph_launch(gid)
            assert all(torch.equal(x.cpu(), w) for x, w in zip(out["r"], want))
            again = torch.autograd.grad(call(t, c), list(leaves.values()), t["g"])
            assert all(torch.equal(x.cpu(), w) for x, w in zip(again, want[1:]))
        assert all(torch.equal(x.cpu(), w) for x, w in zip(torch.autograd.grad(alive, list(leaves.values()), t["g"]), want[1:]))
        rt.graph_destroy(gid)
    finally:
        torch_vulkan.set_inline_backward(False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("B,H,Sq,Sk,D", [(2, 3, 77, 77, 64), (1, 2, 40, 333, 128), (1, 3, 9, 3000, 40), (1, 2, 3, 100, 72), (1, 1, 1, 3000, 64), (16, 32, 70, 50, 16)])
def test_what_the_outputs_rounding_left(B, H, Sq, Sk, D, dtype):
    """Queries and a table of zeros: o is the mean of v, P = 1 exactly, so o + o_lo is off by two roundings in a row and the fp32
    sum's, and so is delta."""
    g = torch.Generator().manual_seed(Sk)
    q, v, do = torch.zeros(B, Sq, H, D, dtype=dtype), torch.randn((B, Sk, H, D), generator=g).to(dtype), torch.randn((B, Sq, H, D), generator=g).to(dtype)
    o, lo, dq = (torch.full((B, Sq, H, D), float("nan"), dtype=dtype, device=vk) for _ in range(3))
    lse, delta, ws = (torch.empty(n, device=vk) for n in (B * H * Sq, B * H * Sq, 1 << 18))
    t = {"q": q, "k": v, "v": v, "dout": do, "table": torch.zeros(32, H, dtype=dtype)}
    t = {n: x.to(vk) for n, x in t.items()}
    a = abi.AttnRelArgs(B=B, H=H, Sq=Sq, Sk=Sk, D=D, buckets=32, max_distance=128, scale=1.0, ws_floats=1 << 18, **{n: x.data_ptr() for n, x in t.items()},
                        o=o.data_ptr(), o_lo=lo.data_ptr(), lse=lse.data_ptr(), delta=delta.data_ptr(), dq=dq.data_ptr(), ws=ws.data_ptr())
    for n, S in (("q", Sq), ("k", Sk), ("v", Sk), ("do", Sq)):
        setattr(a, f"{n}_sb", S * H * D), setattr(a, f"{n}_sh", D), setattr(a, f"{n}_ss", H * D)
    tag = {torch.bfloat16: "bf16", torch.float16: "f16"}[dtype]
    for which in ("fwd", "dq"):
        abi.Runtime().dispatch(f"attn_rel_{which}_{tag}", a)
    mean, size = v.double().mean(1, keepdim=True), v.double().abs().mean(1, keepdim=True)  # [B, 1, H, D]
    u, tiny = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    tol = (1.1 * (u * u * mean.abs() + (Sk + 4) * 2.0**-24 * size) + tiny).expand(B, Sq, H, D)
    got = o.cpu().double() + lo.cpu().double()
    assert ((got - mean).abs() <= tol).all() and (lo.cpu().double().abs() <= 1.01 * u * o.cpu().double().abs() + tiny).all()
    ref = (mean * do.double()).sum(-1).transpose(1, 2)
    tol = (tol * do.double().abs()).sum(-1).transpose(1, 2) + 2 * D * 2.0**-24 * (1.01 * mean * do.double()).abs().sum(-1).transpose(1, 2)
    assert ((delta.cpu().double().view(B, H, Sq) - ref).abs() <= tol).all()


@pytest.mark.gpu
def test_one_query_over_rows_past_31_bits():
    """Keys and values 32 KiB apart, 2.3 GB from first to last, shared by so many heads that their range is not divided."""
    H, Sk, D = 1024, 70000, 64
    g = torch.Generator().manual_seed(1)
    kv, q, table = (torch.randn(s, generator=g).bfloat16() for s in ((Sk, 2 * D), (1, H, 1, D), (32, H)))
    block = torch.empty(Sk, 16384, dtype=torch.bfloat16, device=vk)
    block[:, : 2 * D] = kv.to(vk)
    k, v = (block[:, i * D:(i + 1) * D].view(1, 1, Sk, D).expand(1, H, Sk, D) for i in range(2))
    y = torch_vulkan.relative_bias_attention(q.to(vk), k, v, table.to(vk), causal=True, query_offset=Sk - 1).cpu()
    some = [0, 517, 1023]
    c = case(H=3, Sq=1, Sk=Sk, D=D, causal=True, off=Sk - 1)
    t = {"q": q[:, some], "table": table[:, some], "g": torch.zeros(1, 3, 1, D).bfloat16()}
    t |= {n: kv[:, i * D:(i + 1) * D].reshape(1, 1, Sk, D).expand(1, 3, Sk, D) for i, n in enumerate("kv")}
    ref, tol = oracle(t, c, torch.bfloat16)
    close(y[:, some], ref["o"], tol["o"], "o")


@pytest.mark.gpu
def test_without_room_for_the_key_ranges():
    """The forward of few rows goes on without its workspace, in the plain order of its sums."""
    c = CASES["split_masked"]
    t = inputs(c, torch.bfloat16)
    ref, tol = oracle(t, c, torch.bfloat16)
    d = tensors(t, c)
    o, lse = torch.empty(2, 9, 3, 64, dtype=torch.bfloat16, device=vk), torch.empty(2, 3, 9, device=vk)
    a = abi.AttnRelArgs(B=2, H=3, Sq=9, Sk=3000, D=64, buckets=32, max_distance=128, scale=0.125, q_off=2991, mask_sb=3000,
                        **{n: d[n].data_ptr() for n in ("q", "k", "v", "table", "mask")}, o=o.data_ptr(), lse=lse.data_ptr())
    for n in "qkv":
        for s, x in zip("bhs", d[n].stride()):
            setattr(a, f"{n}_s{s}", x)
    abi.Runtime().dispatch("attn_rel_fwd_bf16", a)
    close(o.transpose(1, 2), ref["o"], tol["o"], "o")


@pytest.mark.gpu
def test_refusals():
    c = case(B=2, H=2, Sq=8, Sk=8, D=16)
    t = tensors(inputs(c, torch.bfloat16), c)
    f = torch_vulkan.relative_bias_attention
    q, k, v, table = (t[n] for n in ("q", "k", "v", "table"))
    ok = torch.ones(2, 8, dtype=torch.bool, device=vk)
    for args, kw, text in (((q, k.float(), v, table), {}, "one type"), ((q, k, v, table.float()), {}, "one type"), ((q, k.cpu(), v, table), {}, "vk"),
                           ((q[0], k, v, table), {}, "B, H, S, D"), ((q, k[:, :1], v[:, :1], table), {}, "as many heads"), ((q, k, v[:, :, :4], table), {}, "k and v"),
                           ((q, k, v, table[:, :1]), {}, "buckets"), ((q, k, v, table[:31]), {}, "even"), ((q, k, v, table[:2]), {}, "even"),
                           ((q, k, v, table), dict(max_distance=8), "max_distance"), ((q, k, v, table), dict(max_distance=2000), "max_distance"),
                           ((q, k, v, table), dict(scale=0.0), "scale"), ((q, k, v, table), dict(scale=-1.0), "scale"), ((q, k, v, table), dict(scale=float("nan")), "scale"),
                           ((q, k, v, table), dict(key_mask=ok[:, :4]), "key_mask"), ((q, k, v, table), dict(key_mask=ok.to(torch.uint8)), "key_mask"),
                           ((q, k, v, table), dict(key_mask=ok.cpu()), "key_mask"), ((q, k, v, table), dict(query_offset=1 << 50), "query_offset"),
                           ((q.long(), k.long(), v.long(), table.long()), {}, "float")):
        with pytest.raises(RuntimeError, match=text):
            f(*args, **kw)
    big = torch.zeros(1, 1, 2, 136, dtype=torch.bfloat16, device=vk)
    with pytest.raises(RuntimeError, match="D must"):
        f(big, big, big, table[:, :1])
    x = q.detach().requires_grad_()
    (g,) = torch.autograd.grad(f(q, k, v, table).sum() + f(x, k, v, table).sum(), x)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(f(x, k, v, table).sum(), x, create_graph=True)
    # the C ABI checks for itself
    rt, out = abi.Runtime(), torch.empty(2, 8, 2, 16, dtype=torch.bfloat16, device=vk)
    lse = torch.empty(2, 2, 8, device=vk)

    def args(**kw):
        a = abi.AttnRelArgs(B=2, H=2, Sq=8, Sk=8, D=16, buckets=32, max_distance=128, scale=0.25, q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(),
                            table=table.data_ptr(), o=out.data_ptr(), lse=lse.data_ptr(), delta=lse.data_ptr(), dout=q.data_ptr())
        for n in ("q", "k", "v", "do"):
            a.__setattr__(f"{n}_sb", 256), a.__setattr__(f"{n}_sh", 128), a.__setattr__(f"{n}_ss", 16)
        for n, x in kw.items():
            setattr(a, n, x)
        return a

    for kw, text in ((dict(D=12), "16-byte pieces"), (dict(D=136), "D <= 128"), (dict(buckets=33), "buckets"), (dict(q=q.data_ptr() + 2), "aligned"),
                     (dict(k_ss=12), "16 bytes"), (dict(Sk=1 << 20), "k"), (dict(scale=0.0), "scale"), (dict(lse=0), "lse"), (dict(mask=ok.data_ptr(), mask_sb=1 << 30), "mask"),
                     (dict(v_sh=-8), "non-negative"), (dict(B=0), "B, H"), (dict(k_ss=1 << 30), "apart")):
        with pytest.raises(RuntimeError, match=text):
            rt.dispatch("attn_rel_fwd_bf16", args(**kw))
    with pytest.raises(RuntimeError, match="workspace"):
        rt.dispatch("attn_rel_dq_bf16", args(dtable=table.data_ptr()))
    with pytest.raises(RuntimeError, match="dk"):
        rt.dispatch("attn_rel_dkdv_bf16", args())


@pytest.mark.gpu
def test_a_block_on_a_frozen_four_bit_base():
    """The layer that these operators are for: frozen 4-bit projections with adapters around attention whose bias is trained.
    Forward and all gradients against the same block in float64 (u = 2^-8; intermediates are rounded to bf16 nine times on
    the longest path, products average the roundings out: 9 u of the largest value)."""
    import torch.nn.functional as F

    B, S, H, D, r = 2, 77, 4, 64, 8
    W = H * D
    g = torch.Generator().manual_seed(3)

    def rand(*shape, scale=1.0):
        return (torch.randn(shape, generator=g) * scale).to(torch.bfloat16)

    x, go, table = rand(B, S, W), rand(B, S, W), rand(32, H)
    packed = {n: torch_vulkan.quantize_mxfp4(rand(W, W, scale=W**-0.5)) for n in "qkvo"}
    adapters = {n: (rand(r, W, scale=W**-0.5), rand(W, r, scale=0.3)) for n in "qkvo"}
    mask = torch.arange(S)[None] < torch.tensor([[77], [40]])

    def block(x, table, adapters, linear, attend):
        def proj(n, y):
            a, b = adapters[n]
            return linear(n, y) + F.linear(F.linear(y, a), b)

        q, k, v = (proj(n, x).view(B, S, H, D).transpose(1, 2) for n in "qkv")
        return x + proj("o", attend(q, k, v, table).transpose(1, 2).reshape(B, S, W))

    def run(cast, linear, attend):
        leaves = [cast(x), cast(table)] + [cast(t) for n in "qkvo" for t in adapters[n]]
        for t in leaves:
            t.requires_grad_()
        y = block(leaves[0], leaves[1], {n: leaves[2 + 2 * i:4 + 2 * i] for i, n in enumerate("qkvo")}, linear, attend)
        return [y, *torch.autograd.grad(y, leaves, cast(go))]

    def attend64(q, k, v, table):
        of, _ = pairs(dict(B=B, Sq=S, Sk=S, off=0, buckets=32, distance=128, causal=False, mask=None))
        s = q @ k.transpose(2, 3) / math.sqrt(D) + table.t()[:, torch.from_numpy(of)]
        return torch.softmax(s.masked_fill(~mask[:, None, None], -math.inf), -1) @ v

    dense = {n: torch_vulkan.dequant_mxfp4(*packed[n], torch.float64) for n in "qkvo"}
    want = run(lambda t: t.double(), lambda n, y: y @ dense[n].t(), attend64)
    on = {n: [t.to(vk) for t in packed[n]] for n in "qkvo"}
    m = mask.to(vk)
    got = run(lambda t: t.detach().to(vk), lambda n, y: torch_vulkan.mxfp4_linear(y, *on[n]),
              lambda q, k, v, table: torch_vulkan.relative_bias_attention(q, k, v, table, key_mask=m))
    for a, b in zip(got, want):
        a = a.detach().cpu().double()
        assert float((a - b).abs().max()) <= 9 * 2.0**-8 * float(b.abs().max())
    assert not {n for n in torch_vulkan.fallback_counts() if not n.startswith("aten::_local")}, torch_vulkan.fallback_counts()


def test_argument_block_matches_the_header(tmp_path):
    import ctypes
    import os
    import subprocess

    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "hrt_ops.h"', 'int main(void) { printf("size %zu\\n", sizeof(hrt_attn_rel_args));']
    lines += [f'printf("{f} %zu\\n", offsetof(hrt_attn_rel_args, {f}));' for f, _ in abi.AttnRelArgs._fields_]
    (tmp_path / "l.c").write_text("\n".join(lines + ["return 0; }"]))
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    subprocess.run(["gcc", "-std=c11", "-I", include, str(tmp_path / "l.c"), "-o", str(tmp_path / "l")], check=True)
    for line in subprocess.run([str(tmp_path / "l")], stdout=subprocess.PIPE, text=True, check=True).stdout.splitlines():
        f, n = line.split()
        assert int(n) == (ctypes.sizeof(abi.AttnRelArgs) if f == "size" else getattr(abi.AttnRelArgs, f).offset), f


@pytest.mark.gpu
def test_forward_mode_is_refused():
    """A tangent is never dropped: neither without nor with a gradient wanted."""
    import torch.autograd.forward_ad as fwd

    c = case(B=1, H=2, Sq=8, Sk=8, D=16)
    t = tensors(inputs(c, torch.bfloat16), c)
    with fwd.dual_level():
        for n in ("q", "k", "v", "table"):
            for wants in (False, True):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call({**t, n: fwd.make_dual(t[n].detach().requires_grad_(wants), torch.ones_like(t[n]))}, c)
        y = call({**t, "q": t["q"].detach().requires_grad_()}, c)  # nor that of an incoming gradient
        with pytest.raises(RuntimeError, match="forward-mode"):
            y.backward(fwd.make_dual(t["g"], t["g"]))
    assert call(t, c).shape == t["q"].shape


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 20, 100])
def test_in_place_operations_on_the_output(D):
    """The backward pass reads the output, so that one changed in place is refused there, in autograd's own words.  One that no gradient
    goes through may be changed, and one whose rows are no whole 16-byte pieces, which is a copy."""
    c = case(B=2, H=2, Sq=40, Sk=40, D=D)
    t = tensors(inputs(c, torch.bfloat16), c)
    leaf = t["q"].detach().requires_grad_()
    out = call({**t, "q": leaf}, c)
    want = torch.autograd.grad(out * 2, leaf, t["g"])[0].cpu()
    with torch.no_grad():
        free = call(t, c)
        assert torch.equal(free.add_(free).cpu(), (out.detach() * 2).cpu())
    y = call({**t, "q": leaf}, c).mul_(2)  # not forbidden as a view's
    assert torch.equal(y.detach().cpu(), (out.detach() * 2).cpu())
    if D % 8 == 0:
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(y, leaf, t["g"])
    else:
        assert torch.equal(torch.autograd.grad(y, leaf, t["g"])[0].cpu(), want)
    assert y.transpose(1, 2).is_contiguous()  # token-major


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,H,Sq,Sk,D,off,mask", [(1, 2, 40, 200, 64, 60, None), (2, 2, 1, 300, 64, 99, None), (1, 2, 9, 3000, 40, 1000, None), (2, 3, 70, 90, 128, -3, None),
                                                  (2, 2, 33, 97, 32, 7, "random"), (1, 1, 20, 50, 64, -20, None), (8, 64, 70, 100, 16, 5, None), (2, 64, 100, 150, 80, 0, None)])
def test_keys_after_the_last_query_are_not_read(B, H, Sq, Sk, D, off, mask, dtype):
    """A cache longer than what has been written to it: a causal form sees no key behind its last query, whatever stands there."""
    c = case(B=B, H=H, Sq=Sq, Sk=Sk, D=D, causal=True, off=off, mask=mask)
    t = inputs(c, dtype)
    seen = max(Sq + off, 0)
    ref, tol = oracle(t, c, dtype)
    for n in "kv":
        t[n][:, :, seen:] = torch.tensor([float("nan"), float("inf"), -float("inf")], dtype=dtype)[torch.arange(Sk - seen) % 3][:, None]
    d = tensors(t, c)
    close(call(d, c), ref["o"], tol["o"], "o")
    y, got = grads(d, c)
    close(y, ref["o"], tol["o"], "o")
    for n, x in got.items():
        close(x, ref[n], tol[n], n)


@pytest.mark.gpu
@pytest.mark.parametrize("off", [-(1 << 63), (1 << 63) - 1, (1 << 40) + 1, -(1 << 40) - 1])
def test_offsets_out_of_range_are_refused(off):
    """With and without rows: the check is the call's own."""
    for Sq in (4, 0):
        t = [torch.zeros(1, 1, n, 8, device=vk) for n in (Sq, 4, 4)]
        with pytest.raises(RuntimeError, match="relative_bias_attention: query_offset out of range"):
            torch_vulkan.relative_bias_attention(*t, torch.zeros(32, 1, device=vk), query_offset=off)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,H,Sq,Sk,D,off,mask", [(1, 2, 100, 100, 64, -40, None), (2, 3, 300, 200, 128, -133, "random"), (8, 64, 70, 40, 16, -33, None), (1, 2, 20, 50, 64, -20, None)])
def test_queries_before_the_first_key_touch_no_gradient(B, H, Sq, Sk, D, off, mask, dtype):
    """A query that causal leaves no key: whatever stands in it and in its output's gradient, k, v and table get nothing of it."""
    c = case(B=B, H=H, Sq=Sq, Sk=Sk, D=D, causal=True, off=off, mask=mask)
    t = inputs(c, dtype)
    none = min(-off, Sq)
    t["g"][:, :, :none] = 0
    ref, tol = oracle(t, c, dtype)
    for n in "qg":
        t[n][:, :, :none] = torch.tensor([float("nan"), float("inf"), -float("inf")], dtype=dtype)[torch.arange(none) % 3][:, None]
    y, got = grads(tensors(t, c), c)
    close(y, ref["o"], tol["o"], "o")
    for n, x in got.items():
        close(x, ref[n], tol[n], n)
