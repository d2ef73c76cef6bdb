"""Rotary positions of several axes against the formula in float64.

Tolerances.  The turn is reduced in fp64 to an eighth and handed over in fp32, its sine and cosine are off by at most 2^-22; two
products and a sum round three times, 2^-24 each, and the output once: (|a| + |b|) (2^-22 + 3 2^-24) and finfo.eps / 2 of the
result (half the smallest subnormal of f16).  Far positions add the fp64 angle's own rounding, 2 turns 2^-52 of a radian each."""

import numpy as np
import pytest
import torch
import torch.nn.functional as F

import torch_vulkan
from torch_vulkan import abi

vk = torch.device("vk")
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
SUB = {torch.bfloat16: 2.0**-134, torch.float16: 2.0**-25, torch.float32: 2.0**-150}


def f64(t):
    return t.detach().cpu().double().numpy()


def turned(x, pos, freqs, sections, interleaved, back=False):
    """The formula, and the sum of magnitudes that its roundings are relative to."""
    x, pos, f = f64(x), f64(pos), f64(freqs)
    P = sum(sections)
    axis = np.repeat(np.arange(len(sections)), sections)
    angle = pos[..., axis] * f * (-1 if back else 1)  # [(B,) S, P]
    angle = angle[:, None] if angle.ndim == 3 else angle
    one, two = (slice(0, 2 * P, 2), slice(1, 2 * P, 2)) if interleaved else (slice(0, P), slice(P, 2 * P))
    a, b = x[..., one], x[..., two]
    y, size = x.copy(), np.zeros_like(x)
    y[..., one], y[..., two] = a * np.cos(angle) - b * np.sin(angle), b * np.cos(angle) + a * np.sin(angle)
    far = np.abs(angle) * 2.0**-51
    size[..., one] = size[..., two] = (np.abs(a) + np.abs(b)) * (2.0**-22 + 3 * 2.0**-24 + far)
    return y, size


def check(got, x, pos, freqs, sections, interleaved, back=False):
    want, tol = turned(x, pos, freqs, sections, interleaved, back)
    dtype = x.dtype
    err = np.abs(f64(got) - want)
    tol = tol + torch.finfo(dtype).eps / 2 * np.abs(want) + SUB[dtype]
    assert got.dtype == dtype and (err <= tol).all(), float(np.max(err / tol))
    P = sum(sections)
    assert torch.equal(got.detach().cpu()[..., 2 * P :], x[..., 2 * P :])


def grid(sizes):
    return torch.stack(torch.meshgrid(*(torch.arange(n) for n in sizes), indexing="ij"), -1).view(-1, len(sizes))


def data(B, Hq, Hk, S, D, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn((B, h, S, D), generator=g).to(dtype) for h in (Hq, Hk, Hq, Hk)]


# heads of every piece width (whole, half, single), one head and many, parts that stay, wide heads in rounds
CASES = [(1, 4, 4, (1, 6, 5), 128, (22, 21, 21)), (2, 3, 1, (2, 3, 3), 64, (8, 12, 12)), (1, 5, 5, (7,), 80, (20,)), (2, 2, 2, (4, 5), 96, (16, 8)), (1, 1, 2, (3, 3), 10, (2, 3)),
         (1, 2, 2, (9,), 7, (3,)), (3, 8, 2, (1,), 128, (64,)), (1, 16, 4, (2, 2, 2, 3), 72, (9, 9, 9, 9)), (1, 2, 1, (5,), 2, (1,)), (1, 3, 3, (6,), 1024, (300,)), (1, 1, 1, (4,), 1000, (499,)),
         (1, 2, 2, (3, 4), 64, (0, 32)), (2, 40, 40, (1, 8, 8), 128, (22, 21, 21)), (5, 2, 2, (17, 60), 32, (8, 8))]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("case", CASES)
def test_against_the_formula(case, interleaved, dtype):
    B, Hq, Hk, sizes, D, sections = case
    pos, freqs = grid(sizes), torch_vulkan.rotary_frequencies(sections, 10000.0)
    q, k, gq, gk = data(B, Hq, Hk, len(pos), D, dtype, D + B)
    Q, K = q.to(vk).requires_grad_(), k.to(vk).requires_grad_()
    out = torch_vulkan.rotary_embedding(Q, K, pos.to(vk), freqs.to(vk), sections, interleaved)
    for o, x in zip(out, (q, k)):
        check(o, x, pos, freqs, sections, interleaved)
        assert o.transpose(1, 2).is_contiguous()
    grads = torch.autograd.grad(out, (Q, K), (gq.to(vk), gk.to(vk)))
    for d, g in zip(grads, (gq, gk)):
        check(d, g, pos, freqs, sections, interleaved, back=True)
    alone = torch_vulkan.rotary_embedding(k.to(vk), None, pos.to(vk), freqs.to(vk), sections, interleaved)
    assert torch.equal(alone.cpu(), out[1].detach().cpu())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [torch.int32, torch.int64, torch.float32])
def test_positions(kind):
    """One set for all, one for each sequence, views; fractions; far and negative ones."""
    sections, freqs = (4, 6, 6), torch_vulkan.rotary_frequencies((4, 6, 6), (10000.0, 500.0, 1e6))
    g = torch.Generator().manual_seed(2)
    q, k, _, _ = data(3, 2, 2, 11, 40, torch.float32, 3)
    pos = torch.randint(-(1 << 24), 1 << 24, (3, 11, 3), generator=g)
    pos = (pos / 8 if kind == torch.float32 else pos).to(kind)
    wide = torch.zeros(3, 22, 5, dtype=kind)
    wide[:, ::2, 1:4] = pos
    turn = lambda p: torch_vulkan.rotary_embedding(q.to(vk), k.to(vk), p, freqs.to(vk), sections)  # noqa: E731
    for p, ref in ((pos.to(vk), pos), (wide.to(vk)[:, ::2, 1:4], pos), (pos[1].to(vk), pos[1]), (pos[1:2].to(vk), pos[1]), (pos[1:2].to(vk).expand(3, 11, 3), pos[1]),
                   (pos[:, :1].to(vk).expand(3, 11, 3), pos[:, :1].expand(3, 11, 3)), (pos.permute(2, 0, 1).contiguous().to(vk).permute(1, 2, 0), pos)):
        for got, x in zip(turn(p), (q, k)):
            check(got, x, ref, freqs, sections, False)
    if kind == torch.int64:
        far = pos * (1 << 16)
        for got, x in zip(turn(far.to(vk)), (q, k)):
            check(got, x, far, freqs, sections, False)
    if kind == torch.float32:
        pos[1, 3, 0] = float("inf")
        got = turn(pos.to(vk))[0].cpu()
        hit = torch.zeros(3, 2, 11, 40, dtype=torch.bool)
        hit[1, :, 3, :4] = hit[1, :, 3, 16:20] = True
        assert torch.isnan(got[hit]).all() and torch.isfinite(got[~hit]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(dtype):
    sections, B, S, H, D = (10, 11, 11), 2, 12, 4, 64
    pos, freqs = grid((2, 3, 2)).to(vk), torch_vulkan.rotary_frequencies((10, 11, 11)).to(vk)
    q, k, gq, gk = data(B, H, H, S, D, dtype, 9)
    want = [t.cpu() for t in torch_vulkan.rotary_embedding(q.to(vk), k.to(vk), pos, freqs, sections)]
    proj = torch.zeros(B, S, 3, H, D + 3, dtype=dtype)  # one projection of queries, keys and values
    proj[:, :, 0, :, 1 : D + 1], proj[:, :, 1, :, 1 : D + 1] = q.transpose(1, 2), k.transpose(1, 2)
    proj = proj.to(vk)
    for a, b in ((proj[:, :, 0, :, 1 : D + 1].transpose(1, 2), proj[:, :, 1, :, 1 : D + 1].transpose(1, 2)),
                 (q.transpose(1, 2).contiguous().to(vk).transpose(1, 2), k.to(vk)), (q.transpose(2, 3).contiguous().to(vk).transpose(2, 3), k.permute(3, 2, 1, 0).contiguous().to(vk).permute(3, 2, 1, 0))):
        A, C = a.detach().requires_grad_(), b.detach().requires_grad_()
        got = torch_vulkan.rotary_embedding(A, C, pos, freqs, sections)
        assert all(torch.equal(x.detach().cpu(), y) for x, y in zip(got, want))
        dq, dk = torch.autograd.grad(got, (A, C), (gq.transpose(2, 3).contiguous().to(vk).transpose(2, 3), gk[:, :1].to(vk).expand(B, H, S, D)))
        wq, wk = torch.autograd.grad(torch_vulkan.rotary_embedding(A, C, pos, freqs, sections), (A, C), (gq.to(vk), gk[:, :1].expand(B, H, S, D).contiguous().to(vk)))
        assert torch.equal(dq.cpu(), wq.cpu()) and torch.equal(dk.cpu(), wk.cpu())
    one = torch_vulkan.rotary_embedding(q[:1, :1].to(vk).expand(B, H, S, D), k.to(vk), pos, freqs, sections)
    assert torch.equal(one[0].cpu(), want[0][:1, :1].expand(B, H, S, D))


@pytest.mark.gpu
def test_gradients_of_one_and_of_gradients():
    sections, pos, freqs = (5, 3), grid((3, 4)), torch_vulkan.rotary_frequencies((5, 3))
    q, k, gq, gk = data(2, 3, 2, 12, 20, torch.float32, 1)
    P, Fr = pos.to(vk), freqs.to(vk)
    Q, K, G, GK = (t.to(vk).requires_grad_() for t in (q, k, gq, gk))
    out = torch_vulkan.rotary_embedding(Q, K, P, Fr, sections)
    (dk,) = torch.autograd.grad(out[1], K, gk.to(vk), retain_graph=True)  # the keys alone
    check(dk, gk, pos, freqs, sections, False, back=True)
    dq, dk = torch.autograd.grad(out, (Q, K), (G, GK), create_graph=True)
    hq, hk = torch.autograd.grad((dq, dk), (G, GK), (q.to(vk), k.to(vk)))  # the turn itself again
    assert torch.equal(hq.cpu(), out[0].detach().cpu()) and torch.equal(hk.cpu(), out[1].detach().cpu())
    out = torch_vulkan.rotary_embedding(Q, k.to(vk), P, Fr, sections)
    (dq,) = torch.autograd.grad(out[0], Q, gq.to(vk))
    check(dq, gq, pos, freqs, sections, False, back=True)
    out = torch_vulkan.rotary_embedding(q.to(vk), K, P, Fr, sections)
    (dk,) = torch.autograd.grad(out[1], K, gk.to(vk))
    check(dk, gk, pos, freqs, sections, False, back=True)
    # against differences: the map is linear, so one difference of any size is the derivative
    step = torch.randn(q.shape, generator=torch.Generator().manual_seed(8))
    a, t1 = turned(q.double() + step.double(), pos, freqs, sections, False)
    b, t2 = turned(q, pos, freqs, sections, False)
    want = ((a - b) * f64(gq)).sum()
    tol = ((t1 + t2 + 2.0**-23 * (np.abs(a) + np.abs(b))) * np.abs(f64(gq))).sum()
    assert abs((f64(dq) * f64(step)).sum() - want) <= tol
    # in place on an output
    out = torch_vulkan.rotary_embedding(Q, K, P, Fr, sections)
    out[0].mul_(2)
    (dq2,) = torch.autograd.grad(out[0], Q, gq.to(vk))
    assert torch.equal(dq2.cpu(), 2 * dq.cpu())


@pytest.mark.gpu
def test_nothing_to_do():
    freqs, pos = torch_vulkan.rotary_frequencies((4,)).to(vk), torch.zeros(3, 1, dtype=torch.int64).to(vk)
    q = torch.randn(2, 2, 3, 8).to(vk)
    for a, b, p in ((q[:0], q[:0], pos), (q[:, :, :0], q[:, :, :0], pos[:0]), (q[:, :0], q, pos), (q, q[:, :0], pos), (q[:, :0], q[:, :0], pos), (q[:, :0], None, pos)):
        out = torch_vulkan.rotary_embedding(a, b, p, freqs, (4,))
        out = out if b is not None else (out,)
        for o, x in zip(out, (a, b)):
            assert torch.equal(o.cpu(), x.cpu())  # position 0: no turn


@pytest.mark.gpu
def test_refusals():
    q, k, _, _ = (t.to(vk) for t in data(2, 4, 2, 6, 16, torch.bfloat16, 1))
    pos, freqs = grid((2, 3)).to(vk), torch_vulkan.rotary_frequencies((4, 4)).to(vk)
    rot = torch_vulkan.rotary_embedding
    for match, call in [("vk tensor", lambda: rot(q.cpu(), k, pos, freqs, (4, 4))), ("q must", lambda: rot(q[0], k, pos, freqs, (4, 4))), ("q must", lambda: rot(q.int(), k, pos, freqs, (4, 4))),
                        ("k must", lambda: rot(q, k.float(), pos, freqs, (4, 4))), ("k must", lambda: rot(q, k[:, :, :3], pos, freqs, (4, 4))),
                        ("sections", lambda: rot(q, k, pos, freqs, ())), ("sections", lambda: rot(q, k, pos, freqs, (2, 2, 2, 1, 1))), ("section", lambda: rot(q, k, pos, freqs, (-1, 9))),
                        ("sections", lambda: rot(q, k, pos, freqs, (5, 4))), ("sections", lambda: rot(q, k, pos, freqs, (0, 0))), ("freqs", lambda: rot(q, k, pos, freqs[:7], (4, 4))),
                        ("freqs", lambda: rot(q, k, pos, freqs.float(), (4, 4))), ("freqs", lambda: rot(q, k, pos, freqs.cpu(), (4, 4))),
                        ("positions", lambda: rot(q, k, pos.double(), freqs, (4, 4))), ("positions", lambda: rot(q, k, pos.cpu(), freqs, (4, 4))),
                        ("positions", lambda: rot(q, k, pos[:5], freqs, (4, 4))), ("positions", lambda: rot(q, k, pos[:, :1], freqs, (4, 4))),
                        ("positions", lambda: rot(q, k, pos.expand(3, 6, 2), freqs, (4, 4))),
                        ("no gradient", lambda: rot(q, k, pos.float().requires_grad_(), freqs, (4, 4))), ("no gradient", lambda: rot(q, k, pos, freqs.detach().requires_grad_(), (4, 4)))]:
        with pytest.raises(RuntimeError, match=match):
            call()
    import torch.autograd.forward_ad as fwd

    with fwd.dual_level():
        for args in ((fwd.make_dual(q, q), k), (q, fwd.make_dual(k, k))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                rot(*args, pos, freqs, (4, 4))
        y = rot(q.detach().requires_grad_(), None, pos, freqs, (4, 4))
        with pytest.raises(RuntimeError, match="forward-mode"):
            y.backward(fwd.make_dual(torch.ones_like(y), torch.ones_like(y)))


def test_frequencies_and_cpu_refusals():
    f = torch_vulkan.rotary_frequencies((22, 21, 0), (10000.0, 500.0, 7.0))
    assert f.dtype == torch.float64 and f.shape == (43,) and f[0] == f[22] == 1.0
    assert torch.allclose(f[:22], 10000.0 ** (-2 * torch.arange(22, dtype=torch.float64) / 44), rtol=1e-14, atol=0)
    with pytest.raises(RuntimeError, match="theta"):
        torch_vulkan.rotary_frequencies((4, 4), (1e4,))
    with pytest.raises(RuntimeError, match="section"):
        torch_vulkan.rotary_frequencies(())
    with pytest.raises(RuntimeError, match="vk tensor"):
        torch_vulkan.rotary_embedding(torch.zeros(1, 1, 2, 4), None, torch.zeros(2, 1), f, (2,))


@pytest.mark.gpu
def test_replayed_graph():
    rt, out = abi.Runtime(), {}
    sections, pos, freqs = (22, 21, 21), grid((2, 8, 9)).to(vk), torch_vulkan.rotary_frequencies((22, 21, 21)).to(vk)
    q, k, gq, gk = (t.to(vk) for t in data(2, 4, 4, 144, 128, torch.bfloat16, 8))
    Q, K = q.detach().requires_grad_(), k.detach().requires_grad_()

    def run():
        with torch.autograd.set_multithreading_enabled(False):
            o = torch_vulkan.rotary_embedding(Q, K, pos, freqs, sections)
            return *(t.detach() for t in o), *torch.autograd.grad(o, (Q, K), (gq, gk))

    eager = [t.cpu() for t in run()]

    def record():
        out["y"] = run()

    gid = rt.graph(record)
    for _ in range(3):
        for t in out["y"]:
            t.zero_()
        rt.graph_launch(gid)
        assert all(torch.equal(a.cpu(), b) for a, b in zip(out["y"], eager))
        assert all(torch.equal(a.cpu(), b) for a, b in zip(run(), eager))
    rt.graph_destroy(gid)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    far = torch.zeros((1 << 31) + 8192, dtype=torch.bfloat16, device=vk)
    sections, pos, freqs = (5, 3), grid((2, 3)).to(vk), torch_vulkan.rotary_frequencies((5, 3)).to(vk)
    q, k, _, _ = data(3, 2, 2, 6, 24, torch.bfloat16, 12)
    view = far.as_strided((3, 2, 6, 24), (1 << 30, 1 << 11, 24, 1))
    view.copy_(q.to(vk))
    for a, b in ((view, k.to(vk)), (k.to(vk), view)):
        got = torch_vulkan.rotary_embedding(a, b, pos, freqs, sections)
        want = torch_vulkan.rotary_embedding(a.contiguous(), b.contiguous(), pos, freqs, sections)
        assert all(torch.equal(x.cpu(), y.cpu()) for x, y in zip(got, want))
    del far, view
    S = (1 << 31) // (128 * 64) + 5  # outputs past 2^31 elements
    one = torch.ones(1, 1, 1, 64, dtype=torch.bfloat16, device=vk).expand(1, 128, S, 64)
    y = torch_vulkan.rotary_embedding(one, None, torch.zeros(S, 1, dtype=torch.int32, device=vk), freqs, (8,))
    assert (y[:, :, -3:].cpu() == 1).all()


# ---- the operators of a block on an 8-bit base together -----------------------------------------------------------------
class Block(torch.nn.Module):
    """Self-attention and MLP of a transformer block on frozen 8-bit weights with trained adapters: residual norms, 8-bit products,
    normed and turned queries and keys, attention."""

    def __init__(self, dim, heads, rank=4):
        super().__init__()
        self.heads, self.hd = heads, dim // heads
        P = torch.nn.Parameter
        self.n1, self.n2, self.nq, self.nk = P(torch.ones(dim)), P(torch.ones(dim)), P(torch.ones(self.hd)), P(torch.ones(self.hd))
        for name, o, i in (("qkv", 3 * dim, dim), ("out", dim, dim), ("up", 2 * dim, dim), ("down", dim, 2 * dim)):
            w = torch.randn(o, i) * i**-0.5
            codes, scale = torch_vulkan.quantize_int8_rows(w)
            self.register_buffer(name + "_w", codes)
            self.register_buffer(name + "_s", scale)
            self.register_parameter(name + "_a", P(torch.randn(rank, i) * i**-0.5))
            self.register_parameter(name + "_b", P(torch.randn(o, rank) * 0.02))

    def lin(self, name, x, plain):
        w, s, a, b = (getattr(self, name + p) for p in ("_w", "_s", "_a", "_b"))
        if plain:  # the values of both sides in 64 bits, the rounding of x passed straight through
            q = x.detach()
            top = q.abs().amax(-1, keepdim=True)
            q = torch.round(q * 127 / top) * (top / 127)
            base = (x + (q - x).detach()) @ (w.double() * s.unsqueeze(-1).double()).t()
        else:
            base = torch_vulkan.int8_linear(x, w, s)
        return base + (x @ a.t()) @ b.t()

    def forward(self, x, r, pos, freqs, sections, plain=False):
        def norm(x, w, r=None):
            if not plain:
                return torch_vulkan.rms_norm(x, w, residual=r)
            h = x if r is None else x + r
            y = h / torch.sqrt(h.pow(2).mean(-1, keepdim=True) + 1e-6) * w
            return y if r is None else (y, h)

        B, S, D = x.shape
        y, r = norm(x, self.n1, r)
        q, k, v = self.lin("qkv", y, plain).view(B, S, 3, self.heads, self.hd).unbind(2)
        q, k, v = norm(q, self.nq).transpose(1, 2), norm(k, self.nk).transpose(1, 2), v.transpose(1, 2)
        if plain:
            angle = pos.double()[:, torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections))] * freqs

            def turn(x):
                a, b = x.chunk(2, -1)
                return torch.cat((a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()), -1)

            q, k = turn(q), turn(k)
        else:
            q, k = torch_vulkan.rotary_embedding(q, k, pos, freqs, sections)
        o = F.scaled_dot_product_attention(q, k, v).transpose(1, 2).reshape(B, S, D)
        y, r = norm(self.lin("out", o, plain), self.n2, r)
        return r + self.lin("down", F.silu(self.lin("up", y, plain)), plain)


@pytest.mark.gpu
def test_a_block_on_an_8_bit_base():
    """Forward and backward against the same block in float64 on the CPU.  Every intermediate is stored in bf16 (2^-9 relative), some
    twenty roundings deep, and codes near a border may differ by one step of a 127th: 2e-2 of the output's and 4e-2 of a
    gradient's norm bounds their sum (20 x 2^-9 if none cancelled is 4e-2)."""
    torch.manual_seed(0)
    B, dim, heads, sizes = 2, 256, 2, (1, 9, 7)
    sections = (22, 21, 21)
    pos, freqs = grid(sizes), torch_vulkan.rotary_frequencies(sections)
    block = Block(dim, heads)
    S = len(pos)
    x, r, g = (torch.randn(B, S, dim).bfloat16() for _ in range(3))
    for p in block.parameters():
        p.data = p.data.bfloat16().float()  # both sides start from the same values
    import copy

    on = copy.deepcopy(block).to(vk)
    for p in on.parameters():
        p.data = p.data.to(torch.bfloat16)
    ref = copy.deepcopy(block)
    for p in ref.parameters():
        p.data = p.data.double()
    X, R = x.to(vk).requires_grad_(), r.to(vk).requires_grad_()
    y = on(X, R, pos.to(vk), freqs.to(vk), sections)
    y.backward(g.to(vk))
    x64, r64 = x.double().requires_grad_(), r.double().requires_grad_()
    want = ref(x64, r64, pos, freqs, sections, plain=True)
    want.backward(g.double())
    rel = lambda a, b: float((a.detach().cpu().double() - b).norm() / b.norm())  # noqa: E731
    assert rel(y, want.detach()) < 2e-2
    for a, b in ((X.grad, x64.grad), (R.grad, r64.grad)):
        assert rel(a, b) < 4e-2
    for (n, a), (_, b) in zip(on.named_parameters(), ref.named_parameters()):
        assert rel(a.grad, b.grad) < 4e-2, n
    names = torch_vulkan.kernel_counts()
    for n in ("rms_norm", "rms_norm_backward", "int8_linear", "int8_linear_backward", "rotary_embedding", "rotary_embedding_backward"):
        assert names.get("torch_vulkan::" + n, 0) >= 1, n
    # the same block while sampling: 8-bit rows out of the norm, the same codes as the layer's own
    with torch.no_grad():
        h = torch_vulkan.rms_norm(X, on.n1, residual=R)
        q, s, h8 = torch_vulkan.rms_norm_int8(X, on.n1, residual=R)
        a = torch_vulkan.int8_linear(h[0], on.qkv_w, on.qkv_s)
        b = torch_vulkan.int8_linear(q, on.qkv_w, on.qkv_s, x_scale=s)
    assert torch.equal(h[1].cpu(), h8.cpu())
    assert rel(b, a.cpu().double()) < 1e-2  # the layer's rows went through bf16 first
