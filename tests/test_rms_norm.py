"""Root-mean-square norm against the formula in float64.

Tolerances, u = 2^-24 and e = finfo.eps / 2 of the type.  The sum of squares adds non-negative terms: a lane takes at most 32 of
them (a 256th of the row where it is longer than that) and tree steps follow, so it is off by at most n u relative, n = 48 +
D / 256, its root by half of it; the mean, eps, root, quotient and the two products round six times.  y adds its own rounding.
Backward: n = h rstd from the kept h, which with a residual was rounded to its type (e); the mean of d n is off by (n + 4) u + e of
the mean of |d n|; three more roundings and the output's.  dw: each term e + 10 u, the sum over the rows at most rows + 80
roundings."""

import ctypes
import threading

import numpy as np
import pytest
import torch

import torch_vulkan
from torch_vulkan import abi

vk = torch.device("vk")
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
SUB = {torch.bfloat16: 2.0**-134, torch.float16: 2.0**-25, torch.float32: 2.0**-150}
U = 2.0**-24


def f64(t):
    return t.detach().cpu().double().numpy()


def steps(D):
    return 48 + D / 256


def norm(x, w, r, eps):
    h = f64(x) + (f64(r) if r is not None else 0.0)
    size = np.sqrt((h * h).mean(-1, keepdims=True) + eps)
    return h / size * (f64(w) if w is not None else 1.0), h, size


def within(got, want, tol, dtype):
    tol = tol + torch.finfo(dtype).eps / 2 * np.abs(want) + SUB[dtype]
    assert got.dtype == dtype and tuple(got.shape) == want.shape
    err = np.abs(f64(got) - want)
    assert (err <= tol).all(), float(np.max(err / tol))


def gradients(x, w, r, gy, gh, eps):
    """dx (the residual's too), dw, and their tolerances without the last rounding."""
    _, h, size = norm(x, None, r, eps)
    D = h.shape[-1]
    n, d = h / size, (f64(gy) if gy is not None else 0.0) * (f64(w) if w is not None else 1.0) + np.zeros_like(h)
    dot, dots = (d * n).mean(-1, keepdims=True), np.abs(d * n).mean(-1, keepdims=True)
    g2 = f64(gh) if gh is not None else 0.0
    dx = (d - n * dot) / size + g2
    e = torch.finfo(x.dtype).eps / 2 if r is not None else 0.0
    c = (steps(D) + 8) * U
    tol = (np.abs(d) * c + np.abs(n) * dots * (2 * e + 3 * c)) / size + 2 * U * (np.abs(dx) + np.abs(g2))
    t = (f64(gy) if gy is not None else 0.0) * n
    rows = int(np.prod(h.shape[:-1]))
    t, size_t = t.reshape(rows, D), np.abs(t).reshape(rows, D).sum(0)
    return dx, tol, t.sum(0), size_t * (e + c + (rows + 80) * U)


def data(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x, r, gy, gh = (torch.randn(shape, generator=g).to(dtype) for _ in range(4))
    w = (1 + 0.2 * torch.randn((shape[-1],), generator=g)).to(dtype)
    return x, w, r, gy, gh


# every sharing of a row out over lanes, both sides of its borders, odd widths, passes
SHAPES = [(1, 1), (3, 7), (5, 64), (70, 65), (33, 128), (5, 129), (2, 3, 200), (40, 256), (3, 257), (9, 500), (6, 512), (5, 1000), (2, 1025), (1030, 1000), (1100, 2048),
          (7, 2048), (4, 2050), (3, 4096), (5, 4100), (2, 8192), (3, 8200), (2, 20001), (600, 40), (2500, 130)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_against_the_formula(shape, dtype):
    x, w, r, gy, gh = data(shape, dtype, sum(shape))
    eps = 1e-5
    X, W, R = (t.to(vk).requires_grad_() for t in (x, w, r))
    c = (steps(shape[-1]) / 2 + 6) * U
    for weight in (W, None):
        y, h = torch_vulkan.rms_norm(X, weight, residual=R, eps=eps)
        want, h64, _ = norm(x, w if weight is not None else None, r, eps)
        within(y, want, np.abs(want) * (c + U), dtype)
        assert torch.equal(h.detach().cpu(), (x.float() + r.float()).to(dtype))
        grads = torch.autograd.grad((y, h), [t for t in (X, R, weight) if t is not None], (gy.to(vk), gh.to(vk)))
        dx, tol, dw, wtol = gradients(x, w if weight is not None else None, r, gy, gh, eps)
        within(grads[0], dx, tol, dtype)
        assert torch.equal(grads[0].cpu(), grads[1].cpu())
        if weight is not None:
            within(grads[2], dw, wtol, dtype)
        y = torch_vulkan.rms_norm(X, weight, eps=eps)
        want, _, _ = norm(x, w if weight is not None else None, None, eps)
        within(y, want, np.abs(want) * c, dtype)
        grads = torch.autograd.grad(y, [t for t in (X, weight) if t is not None], gy.to(vk))
        dx, tol, dw, wtol = gradients(x, w if weight is not None else None, None, gy, None, eps)
        within(grads[0], dx, tol, dtype)
        if weight is not None:
            within(grads[1], dw, wtol, dtype)


@pytest.mark.gpu
def test_gradients_against_differences():
    """The directional derivative of <y, gy> + <h, gh> by central differences of the formula in float64 (truncation and rounding
    below 1e-7 of the terms' sizes at this step)."""
    x, w, r, gy, gh = data((6, 40), torch.float32, 5)
    vx, vw, vr, _, _ = data((6, 40), torch.float32, 6)
    X, W, R = (t.to(vk).requires_grad_() for t in (x, w, r))
    y, h = torch_vulkan.rms_norm(X, W, residual=R)
    got = [f64(t) for t in torch.autograd.grad((y, h), (X, W, R), (gy.to(vk), gh.to(vk)))]

    def value(t):
        a, b, c = x.double() + t * vx.double(), w.double() + t * vw.double(), r.double() + t * vr.double()
        yy, hh, _ = norm(a, b, c, 1e-6)
        return float((yy * f64(gy)).sum() + (hh * f64(gh)).sum())

    step = 1e-4
    want = (value(step) - value(-step)) / (2 * step)
    have = sum(float((a * f64(b)).sum()) for a, b in zip(got, (vx, vw, vr)))
    _, tol, _, wtol = gradients(x, w, r, gy, gh, 1e-6)
    size = np.abs(got[0] * f64(vx)).sum() + np.abs(got[1] * f64(vw)).sum() + np.abs(got[2] * f64(vr)).sum()
    allowed = ((tol + U * np.abs(got[0])) * (np.abs(f64(vx)) + np.abs(f64(vr)))).sum() + ((wtol + U * np.abs(got[1])) * np.abs(f64(vw))).sum() + 1e-7 * size
    assert abs(have - want) <= allowed


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_eight_bit_rows(shape, dtype):
    """A code is within half a step of the unrounded quotient, and the quotient off by the norm's rounding and three more."""
    x, w, r, _, _ = data(shape, dtype, 1 + sum(shape))
    for weight, res in ((w, r), (None, None), (w, None)):
        out = torch_vulkan.rms_norm_int8(x.to(vk), weight.to(vk) if weight is not None else None, residual=res.to(vk) if res is not None else None, eps=1e-5)
        want, h, _ = norm(x, weight, res, 1e-5)
        codes, scale = f64(out[0]), f64(out[1])
        top = np.abs(want).max(-1)
        c = (steps(shape[-1]) / 2 + 8) * U
        assert out[0].dtype == torch.int8 and (np.abs(scale - top / 127) <= (top / 127) * (c + U)).all()
        q = 127 * want / top[..., None]
        assert (np.abs(codes - q) <= 0.5 + np.abs(q) * (2 * c + 3 * U)).all()
        assert (np.abs(codes).max(-1) == 127).all()
        assert len(out) == (3 if res is not None else 2)
        if res is not None:
            assert torch.equal(out[2].cpu(), (x.float() + res.float()).to(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(dtype):
    """Heads inside a projection, transposed and cut views, expanded residuals, rows behind more dimensions than are read in place."""
    x, w, r, gy, gh = data((2, 6, 4, 80), dtype, 3)
    W = w.to(vk)
    base = torch.zeros(2, 6, 3, 4, 85, dtype=dtype)
    base[:, :, 1, :, 3:83] = x
    five = torch.zeros(3, 2, 9, 5, 90, dtype=dtype)
    five[1:, :, 3:9:2, :4, :80] = x.view(2, 2, 3, 4, 80)
    views = [(x.to(vk), x), (base.to(vk)[:, :, 1, :, 3:83], x), (x.transpose(1, 2).contiguous().to(vk).transpose(1, 2), x),
             (x.transpose(2, 3).contiguous().to(vk).transpose(2, 3), x), (x[:, :1].to(vk).expand(2, 6, 4, 80), x[:, :1].expand(2, 6, 4, 80)),
             (five.to(vk)[1:, :, 3:9:2, :4, :80], x.view(2, 2, 3, 4, 80)), (x[0, 0, 0].to(vk), x[0, 0, 0])]
    for view, ref in views:
        want = torch_vulkan.rms_norm(ref.contiguous().to(vk), W).cpu()
        assert torch.equal(torch_vulkan.rms_norm(view, W).cpu(), want)
        res, g = r.flatten()[: ref.numel()].view(ref.shape), gy.flatten()[: ref.numel()].view(ref.shape)
        X, R = view.detach().requires_grad_(), res.to(vk).requires_grad_()
        C = ref.contiguous().to(vk).requires_grad_()
        for a, b in ((X, R), (R, X)):
            c, d = (C, R) if a is X else (R, C)
            got = torch_vulkan.rms_norm(a, W, residual=b)
            wanted = torch_vulkan.rms_norm(c, W, residual=d)
            gv = g.to(vk) if g.dim() < 2 else g.transpose(-1, -2).contiguous().to(vk).transpose(-1, -2)
            dg = torch.autograd.grad(got[0], (X, R), gv)
            dw = torch.autograd.grad(wanted[0], (C, R), g.to(vk))
            assert all(torch.equal(p.detach().cpu(), q.detach().cpu()) for p, q in zip((*got, *dg), (*wanted, *dw)))
            q8, w8 = torch_vulkan.rms_norm_int8(view, W), torch_vulkan.rms_norm_int8(ref.contiguous().to(vk), W)
            assert all(torch.equal(p.cpu(), q.cpu()) for p, q in zip(q8, w8))


@pytest.mark.gpu
def test_outputs_that_are_not_all_used():
    x, w, r, gy, gh = data((5, 48), torch.float32, 4)
    X, W, R = (t.to(vk).requires_grad_() for t in (x, w, r))
    y, h = torch_vulkan.rms_norm(X, W, residual=R)
    dx, dw = torch.autograd.grad(h, (X, W), gh.to(vk), allow_unused=True, retain_graph=True)  # the residual's way alone
    assert torch.equal(dx.cpu(), gh) and (dw is None or dw.cpu().abs().sum() == 0)
    (dr,) = torch.autograd.grad(y, R, gy.to(vk), retain_graph=True)
    want, tol, dw64, wtol = gradients(x, w, r, gy, None, 1e-6)
    within(dr, want, tol, torch.float32)
    (dw,) = torch.autograd.grad(y, W, gy.to(vk))
    within(dw, dw64, wtol, torch.float32)
    # a residual and an input that are one tensor; gradients that accumulate
    y, h = torch_vulkan.rms_norm(X, W, residual=X)
    (gy.to(vk) * y).sum().backward()
    first = X.grad.cpu().clone()
    want, tol, _, _ = gradients(x, w, x, gy, None, 1e-6)
    within(X.grad, 2 * want, 2 * tol + 2 * U * np.abs(want), torch.float32)
    y, h = torch_vulkan.rms_norm(X, W, residual=R)
    ((gy.to(vk) * y).sum() + (gh.to(vk) * h).sum()).backward()
    want, tol, _, _ = gradients(x, w, r, gy, gh, 1e-6)
    within(R.grad, want, tol, torch.float32)
    within(X.grad, f64(first) + want, tol + 2 * U * (np.abs(f64(first)) + np.abs(want)), torch.float32)


@pytest.mark.gpu
def test_rows_that_are_not_finite_or_zero():
    x, w, r, gy, gh = data((6, 130), torch.bfloat16, 8)
    x[1, 3], x[2, 5], x[4], r[4] = float("nan"), float("inf"), 0, 0
    X, W, R = (t.to(vk).requires_grad_() for t in (x, w, r))
    y, h = torch_vulkan.rms_norm(X, W, residual=R)
    (dx,) = torch.autograd.grad((y, h), X, (gy.to(vk), gh.to(vk)))
    rest = [0, 3, 5]
    assert torch.isnan(y.detach().cpu()[1]).all() and torch.isnan(y.detach().cpu()[2, 5]) and y.detach().cpu()[4].abs().sum() == 0
    want, tol, _, _ = gradients(x, w, r, gy, gh, 1e-6)
    within(dx[rest], want[rest], tol[rest], torch.bfloat16)
    within(dx[4], want[4], tol[4], torch.bfloat16)  # zeros: d / sqrt(eps) + gh
    q, s, _ = torch_vulkan.rms_norm_int8(X.detach(), W.detach(), residual=R.detach())
    s = s.cpu()
    assert torch.isnan(s[1:3]).all() and s[4] == 0 and q.cpu()[4].abs().sum() == 0 and torch.isfinite(s[rest]).all()
    z = torch.zeros(3, 130).to(vk)
    assert torch.isnan(torch_vulkan.rms_norm(z, eps=0.0).cpu()).all()  # 0 / 0, as the formula has it
    assert torch.isnan(torch_vulkan.rms_norm_int8(z, eps=0.0)[1].cpu()).all()


@pytest.mark.gpu
def test_nothing_to_do():
    X = torch.zeros(0, 16).to(vk).requires_grad_()
    W = torch.ones(16).to(vk).requires_grad_()
    y, h = torch_vulkan.rms_norm(X, W, residual=torch.zeros(0, 16).to(vk))
    dx, dw = torch.autograd.grad(y.sum() + h.sum(), (X, W))
    assert y.shape == h.shape == dx.shape == (0, 16) and dw.cpu().abs().sum() == 0
    q, s = torch_vulkan.rms_norm_int8(X.detach())
    assert q.shape == (0, 16) and s.shape == (0,)


@pytest.mark.gpu
def test_refusals():
    x, w, r, _, _ = (t.to(vk) for t in data((4, 24), torch.bfloat16, 1))
    X = x.detach().requires_grad_()
    n, n8 = torch_vulkan.rms_norm, torch_vulkan.rms_norm_int8
    for f in (n, n8):
        for match, call in [("float32", lambda: f(x.to(torch.int32))), ("last dimension", lambda: f(x[:, :0])), ("last dimension", lambda: f(x[0, 0])),
                            ("weight", lambda: f(x, w.float())), ("weight", lambda: f(x, w[:3])), ("weight", lambda: f(x, w.cpu())), ("residual", lambda: f(x, w, r[:2])),
                            ("residual", lambda: f(x, w, r.float())), ("residual", lambda: f(x, w, r[:1])), ("eps", lambda: f(x, w, eps=-1.0)),
                            ("eps", lambda: f(x, w, eps=float("nan"))), ("vk tensor", lambda: f(x.cpu()))]:
            with pytest.raises(RuntimeError, match=match):
                call()
    with pytest.raises(RuntimeError, match="has no gradient"):
        n8(X, w)
    with torch.no_grad():
        assert n8(X, w)[0].shape == (4, 24)
    y = n(X, w)
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(y.sum(), X, create_graph=True)
    y, h = n(X, w, residual=r)
    h.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()
    y, h = n(X, w, residual=r)
    y.mul_(2)  # y is not kept
    y.sum().backward()


def test_cpu_refusal():
    with pytest.raises(RuntimeError, match="vk tensor"):
        torch_vulkan.rms_norm(torch.zeros(2, 4))
    with pytest.raises(RuntimeError, match="vk tensor"):
        torch_vulkan.rms_norm_int8(torch.zeros(2, 4))


@pytest.mark.gpu
def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fwd

    x, w, r, _, _ = (t.to(vk) for t in data((4, 24), torch.float32, 1))
    with fwd.dual_level():
        for f in (torch_vulkan.rms_norm, torch_vulkan.rms_norm_int8):
            for args in ((fwd.make_dual(x, x), w, r), (x, fwd.make_dual(w, w), r), (x, w, fwd.make_dual(r, r))):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    f(*args)
        y = torch_vulkan.rms_norm(x.detach().requires_grad_(), w)
        with pytest.raises(RuntimeError, match="forward-mode"):
            y.backward(fwd.make_dual(torch.ones_like(y), torch.ones_like(y)))


@pytest.mark.gpu
def test_autocast_runs_it_in_fp32():
    x, w, r, _, _ = data((4, 24), torch.float32, 1)
    xb = x.bfloat16()
    with torch.autocast("vk", dtype=torch.bfloat16):
        y, h = torch_vulkan.rms_norm(xb.to(vk), w.to(vk), residual=r.to(vk))
        q, s, h8 = torch_vulkan.rms_norm_int8(xb.to(vk), w.to(vk), residual=r.to(vk))
    want = torch_vulkan.rms_norm(xb.float().to(vk), w.to(vk), residual=r.to(vk))
    assert torch.equal(y.cpu(), want[0].cpu()) and torch.equal(h.cpu(), want[1].cpu()) and torch.equal(h8.cpu(), want[1].cpu())
    assert torch.equal(q.cpu(), torch_vulkan.rms_norm_int8(xb.float().to(vk), w.to(vk), residual=r.to(vk))[0].cpu())


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 2048), (900, 300), (2500, 128)])
def test_replayed_graph(shape):
    rt, out = abi.Runtime(), {}
    x, w, r, gy, gh = (t.to(vk) for t in data(shape, torch.bfloat16, 8))
    X, W, R = (t.detach().requires_grad_() for t in (x, w, r))

    def run():
        with torch.autograd.set_multithreading_enabled(False):
            y, h = torch_vulkan.rms_norm(X, W, residual=R)
            grads = torch.autograd.grad((y, h), (X, W, R), (gy, gh))
        return y.detach(), h.detach(), *grads, *torch_vulkan.rms_norm_int8(x, w, residual=r)[:2]

    eager = [t.cpu() for t in run()]

    def record():
        out["y"] = run()

    gid = rt.graph(record)
    for _ in range(3):
        for t in out["y"]:
            t.zero_()
        rt.graph_launch(gid)
        assert all(torch.equal(a.cpu(), b) for a, b in zip(out["y"], eager))
        assert all(torch.equal(a.cpu(), b) for a, b in zip(run(), eager))  # eager work between the replays, the same bits
    rt.graph_destroy(gid)


@pytest.mark.gpu
def test_two_threads():
    x, w, r, gy, _ = (t.to(vk) for t in data((700, 520), torch.float16, 2))
    want = [t.cpu() for t in torch_vulkan.rms_norm(x, w, residual=r)]
    bad = []

    def work():
        X, W = x.detach().requires_grad_(), w.detach().requires_grad_()
        for _ in range(20):
            y, h = torch_vulkan.rms_norm(X, W, residual=r)
            torch.autograd.grad(y, (X, W), gy)
            if not (torch.equal(y.detach().cpu(), want[0]) and torch.equal(h.detach().cpu(), want[1])):
                bad.append(1)

    threads = [threading.Thread(target=work) for _ in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Rows, heads and outputs that begin more than 2^31 elements into their tensors."""
    far = torch.zeros((1 << 31) + 8192, dtype=torch.bfloat16, device=vk)
    x, w, r, gy, gh = data((3, 2, 136), torch.bfloat16, 12)
    view = far.as_strided((3, 2, 136), (1 << 30, 1 << 12, 1))  # the last row lies 2^31 + 2^12 in
    view.copy_(x.to(vk))
    X, C, W, R = view.detach().requires_grad_(), x.to(vk).requires_grad_(), w.to(vk).requires_grad_(), r.to(vk)
    for a in (torch_vulkan.rms_norm_int8(view, W.detach(), residual=R), torch_vulkan.rms_norm_int8(R, W.detach(), residual=view)):
        b = torch_vulkan.rms_norm_int8(C.detach(), W.detach(), residual=R)
        assert all(torch.equal(p.cpu(), q.cpu()) for p, q in zip(a, b))
    a, b = torch_vulkan.rms_norm(X, W), torch_vulkan.rms_norm(C, W)
    assert torch.equal(a.detach().cpu(), b.detach().cpu())
    for p, q in zip(torch.autograd.grad(a, (X, W), gy.to(vk)), torch.autograd.grad(b, (C, W), gy.to(vk))):
        assert torch.equal(p.cpu(), q.cpu())
    assert all(torch.equal(p.cpu(), q.cpu()) for p, q in zip(torch_vulkan.quantize_int8_rows(view), torch_vulkan.quantize_int8_rows(x.to(vk))))
    del far, view, X, a
    n = (1 << 31) // 4096 + 3  # outputs past 2^31 elements
    y = torch_vulkan.rms_norm(torch.ones(1, 4096, dtype=torch.bfloat16, device=vk).expand(n, 4096), None, eps=0.0)
    q, s = torch_vulkan.rms_norm_int8(torch.ones(1, 4096, dtype=torch.bfloat16, device=vk).expand(n, 4096), None, eps=0.0)
    assert (y[-4:].cpu() == 1).all() and (q[-4:].cpu() == 127).all() and (s[-4:].cpu() == torch.tensor(1.0) / 127).all()
    z = torch_vulkan.dequant_int8_rows(q, s)
    assert (z[-4:].cpu() == 1).all()


@pytest.mark.gpu
def test_two_graphs_and_a_live_eager_one():
    """Two recordings of the same leaves, replayed in turn, with gradients that accumulate, while an eager graph of them lives."""
    rt = abi.Runtime()
    x, w, r, gy, gh = (t.to(vk) for t in data((1500, 264), torch.float32, 8))
    X, W = x.detach().requires_grad_(), w.detach().requires_grad_()
    live = torch_vulkan.rms_norm(X, W)

    def step(g):
        with torch.autograd.set_multithreading_enabled(False):
            torch_vulkan.rms_norm(X, W, residual=r)[0].backward(g)

    want = []
    for g in (gy, gh):
        X.grad = W.grad = None
        step(g)
        want.append((X.grad.cpu(), W.grad.cpu()))
    step(gy)  # gradients exist: what is recorded adds to them
    held = X.grad, W.grad
    ids = [rt.graph(lambda g=g: step(g)) for g in (gy, gh)]
    assert X.grad is held[0] and W.grad is held[1]
    for i in (0, 1, 1, 0):
        X.grad.zero_(), W.grad.zero_()
        rt.graph_launch(ids[i])
        assert torch.equal(X.grad.cpu(), want[i][0]) and torch.equal(W.grad.cpu(), want[i][1])
    X.grad = W.grad = None
    live.backward(gy)
    (dx, dw) = torch.autograd.grad(torch_vulkan.rms_norm(X, W), (X, W), gy)
    assert torch.equal(X.grad.cpu(), dx.cpu()) and torch.equal(W.grad.cpu(), dw.cpu())
    for i in ids:
        rt.graph_destroy(i)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(5, 64), (3, 7), (5, 1000), (9, 2048), (3, 8192), (2, 20001)])
def test_the_block_writes_h_without_a_residual(shape, dtype):
    """r 0 in the argument block: h = x, written where h_out asks for it, beside y and beside 8-bit rows."""
    rt, (rows, D) = abi.Runtime(), shape
    x, w, _, _, _ = data(shape, dtype, 4)
    suffix = {torch.float32: "f32", torch.bfloat16: "bf16", torch.float16: "f16"}[dtype]
    X, W, Y, H = x.to(vk), w.to(vk), torch.zeros(shape, dtype=dtype, device=vk), torch.full(shape, 7.0, dtype=dtype, device=vk)
    Q, S = torch.zeros(shape, dtype=torch.int8, device=vk), torch.zeros(rows, device=vk)
    xs = (abi.i64 * 3)(D, 0, 0)
    for out in (dict(y=Y.data_ptr()), dict(q=Q.data_ptr(), scale=S.data_ptr())):
        for h in (H.data_ptr(), 0):
            H.fill_(7.0)
            rt.dispatch("rms_fwd_" + suffix, abi.RmsArgs(x=X.data_ptr(), w=W.data_ptr(), h_out=h, rows=rows, D=D, n1=1, n2=1, xs=xs, eps=1e-6, **out))
            assert torch.equal(H.cpu(), x if h else torch.full(shape, 7.0, dtype=dtype))
    assert torch.equal(Y.cpu(), torch_vulkan.rms_norm(X, W).cpu())
    q, s = torch_vulkan.rms_norm_int8(X, W)
    assert torch.equal(Q.cpu(), q.cpu()) and torch.equal(S.cpu(), s.cpu())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(7, 130), (1030, 264), (7, 4100), (7, 20001), (70000, 7)])
def test_the_residuals_way_is_its_own(shape, dtype):
    """Where h alone is used its gradient goes through as it is, rows that have no norm among them, and the weight's is zero."""
    x, w, r, _, gh = data(shape, dtype, 9)
    x[1, 3], x[2, 5], x[4], r[4], w[6] = float("nan"), float("inf"), 0, 0, float("inf")
    for weight in (w.to(vk).requires_grad_(), None):
        X, R = x.to(vk).requires_grad_(), r.to(vk).requires_grad_()
        for g in (gh.to(vk), gh.t().contiguous().to(vk).t(), gh[:, :1].to(vk).expand(shape)):
            h = torch_vulkan.rms_norm(X, weight, residual=R, eps=0.0)[1]
            grads = torch.autograd.grad(h, [t for t in (X, R, weight) if t is not None], g)
            assert torch.equal(grads[0].cpu(), g.cpu()) and torch.equal(grads[1].cpu(), g.cpu())
            assert weight is None or (grads[2].shape == w.shape and (grads[2].cpu() == 0).all())
    X, R = x.to(vk).requires_grad_(), r.to(vk).requires_grad_()
    torch_vulkan.rms_norm(X, None, residual=R, eps=0.0)[1].backward(gh.to(vk))
    X.grad.add_(1)  # two gradients, not one tensor
    assert torch.equal(R.grad.cpu(), gh)


@pytest.mark.gpu
def test_an_eps_that_fp32_does_not_hold():
    """Taken as 0 it would make NaN of rows of zeros, where the formula has 0."""
    x = torch.zeros(3, 40).to(vk)
    for f in (torch_vulkan.rms_norm, torch_vulkan.rms_norm_int8):
        with pytest.raises(RuntimeError, match="eps"):
            f(x, eps=1e-46)
        assert (f(x, eps=2e-45)[0].cpu() == 0).all()


# sums of the weight's gradient over more rows than the strips take: every sharing with a workspace, several rows to a workgroup of the
# passes too
MANY_ROWS = [(1100, 2052), (1100, 2056), (1100, 4096), (1100, 4100), (1030, 8200), (1030, 8201), (600, 16400), (1200, 16401)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", MANY_ROWS)
def test_many_wide_rows_against_the_formula(shape, dtype):
    test_against_the_formula(shape, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1500, 264), (1500, 520), (600, 16400)])
def test_two_threads_with_workspaces(shape):
    """Gradients whose sums go through a workspace, from two threads at once: one thread's bits."""
    x, w, r, gy, _ = (t.to(vk) for t in data(shape, torch.float16, 2))

    def gradients_of():
        X, W = x.detach().requires_grad_(), w.detach().requires_grad_()
        y, _ = torch_vulkan.rms_norm(X, W, residual=r)
        return torch.autograd.grad(y, (X, W), gy)

    want, bad = [t.cpu() for t in gradients_of()], []

    def work():
        for _ in range(10):
            if not all(torch.equal(a.cpu(), b) for a, b in zip(gradients_of(), want)):
                bad.append(1)

    threads = [threading.Thread(target=work) for _ in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_the_backward_block_without_gy(dtype):
    """dx = gh and dw = 0, with nothing else given, and zeros where there is no gh either; no workspace is asked for."""
    rt, (rows, D) = abi.Runtime(), (1100, 70)
    suffix, code = {torch.float32: ("f32", 0), torch.bfloat16: ("bf16", 1), torch.float16: ("f16", 2)}[dtype]
    gh = data((rows, D), dtype, 4)[4].to(vk)
    for g in (gh, None):
        dx, dw = torch.ones(rows, D, dtype=dtype, device=vk), torch.ones(D, dtype=dtype, device=vk)
        a = abi.RmsBwdArgs(gh=g.data_ptr() if g is not None else 0, dx=dx.data_ptr(), dw=dw.data_ptr(), rows=rows, D=D, n1=1, n2=1, ghs=(abi.i64 * 3)(D, 0, 0))
        assert rt.lib.hrt_rms_workspace(ctypes.byref(a), code) == 0
        rt.dispatch("rms_bwd_" + suffix, a)
        assert torch.equal(dx.cpu(), gh.cpu() if g is not None else torch.zeros(rows, D, dtype=dtype)) and (dw.cpu() == 0).all()
    with pytest.raises(RuntimeError, match="h"):
        a.gy = gh.data_ptr()
        rt.dispatch("rms_bwd_" + suffix, a)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(64, 96), (64, 97), (64, 5), (700, 264), (1030, 130), (1100, 2048), (1100, 4100), (64, 8201), (600, 16400), (520, 16403)])
def test_the_weights_gradient_of_an_unrounded_sum(shape, dtype):
    """Rows in pairs of equal gradients of opposite sign and of sums that round alike: the weight's gradient is what rounding takes
    from the sums.  It is left within a 512th of half the type's last place (2^-16, 2^-19 of the value; a subnormal sum within half
    its last place, 2^-25 in f16), for which the header's tolerance has e, and is tested against the formula with that bound."""
    rows, D = shape
    g = torch.Generator().manual_seed(rows + D)
    e = torch.finfo(dtype).eps
    h = (torch.randint(-512, 513, (rows // 2, D), generator=g).float() / 256 + torch.randint(0, 2, (rows // 2, D), generator=g).float() * 4).to(dtype)
    rest = (h.double().abs() * (torch.rand(rows // 2, D, generator=g).double() - 0.5) * 0.9 * e / 2).to(dtype)  # below half of any last place
    x, r = torch.stack((h, h), 1).view(rows, D), torch.stack((rest, torch.zeros_like(rest)), 1).view(rows, D)
    gy = torch.randn(rows // 2, D, generator=g).to(dtype)
    gy = torch.stack((gy, -gy), 1).view(rows, D)
    w = (1 + 0.2 * torch.randn(D, generator=g)).to(dtype)
    X, W, R = (t.to(vk).requires_grad_() for t in (x, w, r))
    y, hh = torch_vulkan.rms_norm(X, W, residual=R)
    if dtype != torch.float32:
        assert torch.equal(hh.detach().cpu(), x)
    dx, dw = torch.autograd.grad(y, (X, W), gy.to(vk))
    want, _, dw64, _ = gradients(x, w, r, gy, None, 1e-6)
    n, _, size = norm(x, None, r, 1e-6)
    left = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-16, torch.float16: 2.0**-19}[dtype]
    terms = np.abs(f64(gy)) * (np.abs(n) * (left + (steps(D) + 8 + 10 + rows + 80) * U) + (2.0**-25 / size if dtype == torch.float16 else 0.0))
    within(dw, dw64, terms.sum(0), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES[1:])
@pytest.mark.parametrize("D", [5, 64, 97, 1000, 4100, 16403])
def test_what_rounding_takes_from_a_sum(D, dtype):
    """h and its rests give the fp32 sum within half a 256th of the type's last place (a whole one where that is half the last place up),
    at both ends of the exponent range, beside rows that are not finite; refused where there is nothing to round."""
    rt, rows = abi.Runtime(), 9
    suffix, bits = ("bf16", 16) if dtype == torch.bfloat16 else ("f16", 13)  # fp32 patterns in a last place
    g = torch.Generator().manual_seed(D)
    big = torch.finfo(dtype).max
    size = torch.tensor([1.0, 2.0**-10, 2.0**-13, 300.0, big / 8, 1.0, 1.0, 1.0, 2.0**-30 if dtype == torch.bfloat16 else 2.0**-5]).unsqueeze(1)
    x, r = (torch.randn(rows, D, generator=g) * size).to(dtype), (torch.randn(rows, D, generator=g) * size / 64).to(dtype)
    x[5, 3], x[6, 1], x[7], r[7] = float("inf"), float("nan"), big, big * 2.0**-10  # the last: a sum that rounds to an infinity, or to the largest
    x[8, :2], r[8, :2] = 0, 0
    pitch = (D + 7) // 8 * 8
    X, R, Y, H = x.to(vk), r.to(vk), torch.zeros(rows, D, dtype=dtype, device=vk), torch.zeros(rows, D, dtype=dtype, device=vk)
    rest = torch.full((rows, pitch), 7, dtype=torch.int8, device=vk)
    xs = (abi.i64 * 3)(D, 0, 0)
    args = dict(x=X.data_ptr(), y=Y.data_ptr(), rows=rows, D=D, n1=1, n2=1, xs=xs, rs=xs, eps=1e-6)
    rt.dispatch("rms_fwd_" + suffix, abi.RmsArgs(r=R.data_ptr(), h_out=H.data_ptr(), h_rest=rest.data_ptr(), **args))
    s, h = x.float() + r.float(), H.cpu()
    assert torch.equal(torch.nan_to_num(h.float()), torch.nan_to_num(s.to(dtype).float())) and (rest.cpu()[:, D:] == 0).all()
    back = (h.float().view(torch.int32) + (rest.cpu()[:, :D].int() << (bits - 8))).view(torch.float32)
    fine = h.isfinite()
    normal = fine & (h.float().abs() >= 2.0**-14)
    assert torch.equal(back[~fine].isnan(), s[~fine].isnan()) and not back[~fine].isfinite().any()
    off = (back.double() - s.double()).abs()
    assert (off[normal] <= s.double().abs()[normal] * 2.0 ** (bits - 8 - 23)).all()
    assert (off[fine] <= (h.double() - s.double()).abs()[fine] + s.double().abs()[fine] * 2.0 ** (bits - 8 - 23)).all()
    for bad in (dict(r=R.data_ptr(), h_rest=rest.data_ptr()), dict(h_out=H.data_ptr(), h_rest=rest.data_ptr()),
                dict(r=R.data_ptr(), h_out=H.data_ptr(), h_rest=rest.data_ptr() + 4)):
        with pytest.raises(RuntimeError, match="h_rest"):
            rt.dispatch("rms_fwd_" + suffix, abi.RmsArgs(**bad, **args))
    with pytest.raises(RuntimeError, match="h_rest"):
        rt.dispatch("rms_bwd_f32", abi.RmsBwdArgs(gy=X.data_ptr(), h=X.data_ptr(), rstd=Y.data_ptr(), dx=Y.data_ptr(), h_rest=rest.data_ptr(), rows=1, D=2, n1=1, n2=1))
