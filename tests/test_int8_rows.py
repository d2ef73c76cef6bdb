"""8-bit rows and products: packing against its definition in whole numbers, products against float64 products of the values that
the packed operands stand for.

Tolerances.  Codes are exact; a scale is one fp32 division (correctly rounded: equal to numpy's), a value read back one fp32
product, rounded once more to its type.  A product's sum of integers is exact; its conversion to fp32, the two scales and the
bias round four times, 2^-24 each of what they round (scaled sum, or scaled sum plus bias), and the output once (finfo.eps / 2
relative, half the smallest subnormal of f16).  A gradient's sum over N runs over weights rounded to 16 bits (eps / 2 each; half
the smallest subnormal of f16) and rounds at most N times in fp32."""

import numpy as np
import pytest
import torch

import torch_vulkan
from torch_vulkan import abi

vk = torch.device("vk")
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
HALF = DTYPES[1:]
SUB = {torch.bfloat16: 2.0**-134, torch.float16: 2.0**-25, torch.float32: 2.0**-150}  # half the smallest subnormal


def f64(t):
    return t.detach().cpu().double().numpy()


def packed(x):
    """Codes and fp32 scales from the definition.  127 x and the border (2 n + 1) top / 2 are compared as whole numbers."""
    x = f64(x)
    top = np.abs(x).max(-1, keepdims=True)
    ok = np.isfinite(top) & (top > 0)
    safe = np.where(ok, top, 1.0)
    n = np.rint(np.where(ok, x, 0.0) * 127 / safe)
    # products of a 24-bit by an 8- or 9-bit number: exact, and so is the sign of their difference
    d = 127 * np.where(ok, x, 0.0) - n * safe
    n = n + (2 * d > safe) - (2 * d < -safe)
    n = np.where((2 * np.abs(d) == safe) & (n % 2 == 1), n + np.sign(d), n)
    with np.errstate(invalid="ignore", over="ignore"):
        scale = np.where(np.isfinite(top), top.astype(np.float32) / np.float32(127), np.float32(np.nan)).astype(np.float32)
        # a step of which 127 are finite in fp32: the neighbour below where the nearest is not one
        scale = np.where(np.isinf(scale * np.float32(127)), np.nextafter(scale, np.float32(0)), scale)
    return n.astype(np.int8), scale[..., 0]


def sample(rows, cols, dtype, seed):
    """Rows of very different sizes; every third row on rounding borders (multiples of top / 254), one of zeros."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, cols), generator=g) * torch.exp2(torch.randint(-10, 10, (rows, 1), generator=g).float())
    edge = torch.randint(-254, 255, (rows, cols), generator=g).float() / 128
    edge[:, 0] = 127 / 64
    x = torch.where(torch.arange(rows).unsqueeze(1) % 3 == 1, edge, x)
    x[rows // 2] = 0
    return x.to(dtype)


def same(got, want):
    codes, scale = (t.cpu().numpy() for t in got)
    assert codes.dtype == np.int8 and scale.dtype == np.float32
    assert np.array_equal(codes, want[0]) and np.array_equal(scale, want[1], equal_nan=True)


SHAPES = [(1, 1), (3, 7), (5, 16), (4, 33), (7, 127), (6, 128), (2, 130), (9, 256), (5, 500), (9, 1000), (2, 1025), (1030, 2048), (33, 4100), (3, 8192), (2, 8200), (2, 20000)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_cpu_form_follows_the_definition(shape, dtype):
    x = sample(*shape, dtype, sum(shape))
    got = torch_vulkan.quantize_int8_rows(x)
    same(got, packed(x))
    for out in DTYPES:
        y = torch_vulkan.dequant_int8_rows(*got, out)
        assert torch.equal(y, (got[0].float() * got[1].unsqueeze(-1)).to(out))


def extremes():
    """Both ends of the exponent range, infinities, NaN, subnormals."""
    f = torch.finfo(torch.float32)
    rows = [[f.max, 1.0], [f.tiny, f.tiny * 3], [f.smallest_normal / 4, 1e-40], [2.0**-149, 0.0], [float("inf"), 1.0], [float("nan"), 1.0], [-f.max, f.max / 254],
            [-0.0, 0.0], [2.0**-100, 2.0**-101], [2.0**100, 2.0**99], [2.0**101, -(2.0**20)], [1e-36, 1e-37], [3e38, -2e38]]
    x = torch.zeros(len(rows), 40)
    for i, r in enumerate(rows):
        x[i, 3:5] = torch.tensor(r)
    return x


def test_cpu_extremes():
    x = extremes()
    same(torch_vulkan.quantize_int8_rows(x), packed(x))


def test_cpu_refusals():
    c, s = torch_vulkan.quantize_int8_rows(torch.randn(4, 70))
    with pytest.raises(RuntimeError, match="without the last dimension"):
        torch_vulkan.dequant_int8_rows(c, s[:3])
    with pytest.raises(RuntimeError, match="int8"):
        torch_vulkan.dequant_int8_rows(c.int(), s)
    with pytest.raises(RuntimeError, match="float32"):
        torch_vulkan.quantize_int8_rows(torch.zeros(4, 4, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="vk tensor"):
        torch_vulkan.int8_linear(torch.zeros(4, 70), c, s)


def test_argument_blocks_match_the_header(tmp_path):
    """abi's blocks of the 8-bit, norm and rotary kernels lay their fields out as include/hrt_ops.h does."""
    import ctypes
    import os
    import subprocess

    blocks = {"hrt_i8_rows_args": abi.I8RowsArgs, "hrt_i8_mm_args": abi.I8MmArgs, "hrt_i8_linear_back_args": abi.I8LinearBackArgs, "hrt_rms_args": abi.RmsArgs, "hrt_rms_bwd_args": abi.RmsBwdArgs,
              "hrt_rotary_args": abi.RotaryArgs}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "hrt_ops.h"', "int main(void) {"]
    for c, py in blocks.items():
        lines.append(f'  printf("{c} size %zu\\n", sizeof({c}));')
        lines += [f'  printf("{c} {f} %zu\\n", offsetof({c}, {f}));' for f, _ in py._fields_]
    (tmp_path / "l.c").write_text("\n".join(lines + ["  return 0; }"]))
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    subprocess.run(["gcc", "-std=c11", "-I", include, str(tmp_path / "l.c"), "-o", str(tmp_path / "l")], check=True)
    got = [l.split() for l in subprocess.run([str(tmp_path / "l")], stdout=subprocess.PIPE, text=True, check=True).stdout.splitlines()]
    for c, f, n in got:
        assert int(n) == (ctypes.sizeof(blocks[c]) if f == "size" else getattr(blocks[c], f).offset), (c, f)


def test_the_order_that_the_products_barriers_count_on():
    """Stage 0 is issued before a fence and later stages behind it, and in a step X behind a fence behind W, at its start or spread."""
    import os
    import re

    kernels = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "torch-vulkan_amd", "csrc", "kernels")
    text = re.sub(r"//[^\n]*", "", open(os.path.join(kernels, "i8_gemm.hip")).read())
    zero, one = "(std::integral_constant<int, 0>(), 0);", "(std::integral_constant<int, 1>(), 1);"
    for first, later in ((f"stage_x{zero}", f"stage_w{one}"), (f"stage_w{zero}", f"stage_x{one}"), (f"stage_w{zero}", f"stage_w{one}"),
                         ("stage_w(IW(), ks + WR - 1);", "stage_x(IX(), ks + XR - 1);")):
        between = text[text.index(first) : text.index(later)]
        assert text.count(first) == text.count(later) == 1 and "issue_order_fence();" in between
    assert re.search(r"if \(c == IPW\) issue_order_fence\(\);\s*if \(c < IPW\) \{\s*if \(more_w\) copy_w\(.*?\} else \{\s*if \(more_x\) copy_x\(", text, re.S)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_packing_is_exact(shape, dtype):
    x = sample(*shape, dtype, 1 + sum(shape))
    got = torch_vulkan.quantize_int8_rows(x.to(vk))
    want = packed(x)
    same(got, want)
    for out in DTYPES:
        y = torch_vulkan.dequant_int8_rows(*got, out)
        assert torch.equal(y.cpu(), (torch.from_numpy(want[0]).float() * torch.from_numpy(want[1]).unsqueeze(-1)).to(out))


def all_quotients(dtype):
    """Rows whose largest value takes every mantissa (every 31st in f16), with every other mantissa over the nine binades in which
    codes are not 0; in fp32 the values next to every border of random rows."""
    if dtype == torch.float32:
        g = torch.Generator().manual_seed(5)
        top = (torch.rand(200, 1, generator=g) + 1) * torch.exp2(torch.randint(-60, 60, (200, 1), generator=g).float())
        edge = (top.double() * torch.arange(1, 254, 2) / 254).float()
        x = torch.cat([edge, torch.nextafter(edge, torch.zeros(1)), torch.nextafter(edge, torch.full((1,), 2.0**80))], -1)
    else:
        n = {torch.bfloat16: 128, torch.float16: 1024}[dtype]
        man = 1 + torch.arange(n) / n
        top = man[:: 1 if n == 128 else 31].unsqueeze(-1)
        x = (man * torch.exp2(-torch.arange(9.0)).unsqueeze(-1)).flatten().expand(len(top), -1)
        x = torch.where(x <= top, x, torch.zeros(()))
    x = torch.cat([top, x], -1)
    return torch.cat([x, -x]).to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_every_quotient(dtype):
    x = all_quotients(dtype)
    same(torch_vulkan.quantize_int8_rows(x.to(vk)), packed(x))
    same(torch_vulkan.quantize_int8_rows(x), packed(x))


@pytest.mark.gpu
def test_extremes_on_the_device():
    x = extremes()
    got = torch_vulkan.quantize_int8_rows(x.to(vk))
    same(got, packed(x))
    y = torch_vulkan.dequant_int8_rows(*got, torch.float32).cpu()
    bad = ~torch.isfinite(x).all(-1)
    assert torch.isnan(y[bad]).all() and torch.isfinite(y[~bad]).all()


@pytest.mark.gpu
def test_packing_of_views():
    x = sample(12, 4096, torch.bfloat16, 3)
    base = x.to(vk)
    for view, ref in ((base[:, 8:1032], x[:, 8:1032]), (base[:, 3:100], x[:, 3:100]), (base.t(), x.t()), (base[:1].expand(5, 4096), x[:1].expand(5, 4096)),
                      (base.view(3, 4, 4096), x.view(3, 4, 4096)), (base.view(3, 4, 4096).transpose(0, 1), x.view(3, 4, 4096).transpose(0, 1)), (base[0], x[0]),
                      (base[:0], x[:0]), (base[:, :0], x[:, :0])):
        got, want = torch_vulkan.quantize_int8_rows(view), torch_vulkan.quantize_int8_rows(ref)
        assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])
        assert torch.equal(torch_vulkan.dequant_int8_rows(*got).cpu(), torch_vulkan.dequant_int8_rows(*want))
    codes, scale = torch_vulkan.quantize_int8_rows(base)
    for cv, sv in ((codes[:, 5:77], scale), (codes.t()[:12], scale), (codes[::2], scale[::2])):
        assert torch.equal(torch_vulkan.dequant_int8_rows(cv, sv).cpu(), torch_vulkan.dequant_int8_rows(cv.cpu(), sv.cpu()))


# ---- the linear layer -------------------------------------------------------------------------------------------------
def operands(M, N, K, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((M, K), generator=g).to(dtype)
    w = torch.randint(-127, 128, (N, K), generator=g, dtype=torch.int8)
    s = torch.rand((N,), generator=g) * 2e-3 + 1e-5
    b = torch.randn((N,), generator=g).to(dtype)
    return x, w, s, b


def product(codes, scale, w, s, b):
    y = (codes.astype(np.float64) @ f64(w).T) * scale.astype(np.float64)[:, None] * f64(s)
    return y, (y + f64(b) if b is not None else y)


def check_forward(got, y, want, dtype):
    tol = torch.finfo(dtype).eps / 2 * np.abs(want) + SUB[dtype] + 1.01 * 2.0**-24 * (3 * np.abs(y) + np.abs(want))
    assert got.dtype == dtype and tuple(got.shape) == want.shape
    assert (np.abs(f64(got) - want) <= tol).all(), np.max(np.abs(f64(got) - want) / tol)


def check_back(got, g, w, s, dtype):
    v = f64(w) * f64(s)[:, None]
    want, size = f64(g) @ v, np.abs(f64(g)) @ np.abs(v)
    e = torch.finfo(dtype).eps / 2
    tol = e * np.abs(want) + SUB[dtype] + size * (1.01 * e + (len(v) + 1) * 2.0**-24) + np.abs(f64(g)).sum(-1, keepdims=True) * SUB[dtype]
    assert (np.abs(f64(got) - want) <= tol).all(), np.max(np.abs(f64(got) - want) / tol)


# every tile and both sides of its borders, rows, odd widths, ends of K inside a line and inside a piece of 16
# (the tile of 128 x 128, and the loops of all tiles: LONG_PRODUCTS)
PRODUCTS = [(1, 16, 16), (1, 1, 1), (2, 8, 144), (16, 48, 2064), (16, 100, 128), (17, 64, 1024), (32, 40, 1040), (33, 136, 320), (64, 64, 512), (77, 130, 272),
            (130, 256, 400), (129, 129, 128), (257, 264, 1000), (300, 512, 77), (5, 33, 50), (200, 2056, 656), (1, 4096, 4096), (20, 512, 9000), (308, 72, 4112),
            (3, 40, 2720), (3, 24, 4096), (4, 24, 4112), (8, 24, 2048), (7, 24, 1040), (5, 24, 1024), (3, 24, 1008), (4, 8, 512), (8, 24, 2064), (1, 24, 16384), (1, 8, 16400), (2, 8, 8192), (700, 2048, 512), (1500, 4096, 256), (4100, 2048, 144)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("M,N,K", PRODUCTS)
def test_linear(M, N, K, dtype):
    x, w, s, b = operands(M, N, K, dtype, M + N + K)
    codes, scale = packed(x)
    X, W, S, B = (t.to(vk) for t in (x, w, s, b))
    y, want = product(codes, scale, w, s, b)
    check_forward(torch_vulkan.int8_linear(X, W, S, B), y, want, dtype)
    y, want = product(codes, scale, w, s, None)
    check_forward(torch_vulkan.int8_linear(X, W, S), y, want, dtype)
    got = torch_vulkan.int8_linear(torch.from_numpy(codes).to(vk), W, S, x_scale=torch.from_numpy(scale).to(vk), out_dtype=dtype)
    check_forward(got, y, want, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 16, 40, 300, 1100])
def test_sums_at_their_largest(M):
    """All codes at 127 and -127 (-128 among the weights), at the longest K: whole sums of 31 bits."""
    K = 131056
    x = torch.ones((M, K), dtype=torch.int8) * 127
    w = torch.full((24, K), -128, dtype=torch.int8)
    w[::2] = 127
    xs, s = torch.linspace(0.5, 2, M), torch.linspace(1e-3, 2e-3, 24)
    y = (127.0 * K) * torch.where(torch.arange(24) % 2 == 0, 127.0, -128.0).double().numpy() * f64(xs)[:, None] * f64(s)
    got = torch_vulkan.int8_linear(x.to(vk), w.to(vk), s.to(vk), x_scale=xs.to(vk), out_dtype=torch.bfloat16)
    check_forward(got, y, y, torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("M,N,K", [(1, 16, 16), (37, 136, 320), (5, 33, 50), (308, 256, 512), (130, 72, 1000), (1030, 512, 264)])
def test_gradients(M, N, K, dtype):
    x, w, s, b = operands(M, N, K, dtype, 7)
    g = torch.randn((M, N), generator=torch.Generator().manual_seed(3)).to(dtype)
    X, B = x.to(vk).requires_grad_(), b.to(vk).requires_grad_()
    dx, db = torch.autograd.grad(torch_vulkan.int8_linear(X, w.to(vk), s.to(vk), B), (X, B), g.to(vk))
    check_back(dx, g, w, s, dtype)
    want = f64(g).sum(0)
    assert (np.abs(f64(db) - want) <= torch.finfo(dtype).eps / 2 * np.abs(want) + SUB[dtype] + M * 2.0**-24 * np.abs(f64(g)).sum(0)).all()
    # one of the two alone, and the bias under an int8 x
    (dx2,) = torch.autograd.grad(torch_vulkan.int8_linear(X, w.to(vk), s.to(vk)), (X,), g.to(vk))
    (db2,) = torch.autograd.grad(torch_vulkan.int8_linear(x.to(vk), w.to(vk), s.to(vk), B), (B,), g.to(vk))
    codes, scale = torch_vulkan.quantize_int8_rows(x.to(vk))
    (db3,) = torch.autograd.grad(torch_vulkan.int8_linear(codes, w.to(vk), s.to(vk), B, x_scale=scale, out_dtype=dtype), (B,), g.to(vk))
    assert torch.equal(dx2.cpu(), dx.cpu()) and torch.equal(db2.cpu(), db.cpu()) and torch.equal(db3.cpu(), db.cpu())


@pytest.mark.gpu
def test_the_gradients_gradient():
    """dx = g W is linear in g: its gradient is h W^T, and that one's k W again."""
    M, N, K, dtype = 37, 136, 320, torch.bfloat16
    x, w, s, b = operands(M, N, K, dtype, 23)
    r = torch.Generator().manual_seed(4)
    g, k = (torch.randn((M, N), generator=r).to(dtype) for _ in range(2))
    h = torch.randn((M, K), generator=r).to(dtype)
    X, G, H = (t.to(vk).requires_grad_() for t in (x, g, h))
    (dx,) = torch.autograd.grad(torch_vulkan.int8_linear(X, w.to(vk), s.to(vk), b.to(vk)), X, G, create_graph=True)
    check_back(dx, g, w, s, dtype)
    (gh,) = torch.autograd.grad(dx, G, H, create_graph=True)
    v = f64(w) * f64(s)[:, None]
    e, size = torch.finfo(dtype).eps / 2, np.abs(f64(h)) @ np.abs(v).T
    assert (np.abs(f64(gh) - f64(h) @ v.T) <= e * np.abs(f64(h) @ v.T) + size * (1.01 * e + (K + 1) * 2.0**-24)).all()
    (gk,) = torch.autograd.grad(gh, H, k.to(vk))
    check_back(gk, k, w, s, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
def test_layouts(dtype):
    x, w, s, b = operands(24, 72, 320, dtype, 11)
    want = torch_vulkan.int8_linear(x.to(vk), w.to(vk), s.to(vk), b.to(vk)).cpu()
    wide_x, wide_w = torch.zeros(24, 333, dtype=dtype), torch.zeros(144, 352, dtype=torch.int8)
    wide_x[:, 5:325], wide_w[::2, 16:336] = x, w
    off_w = torch.zeros(72, 321, dtype=torch.int8)
    off_w[:, 1:] = w
    for X in (x.to(vk), wide_x.to(vk)[:, 5:325], x.t().contiguous().to(vk).t(), x.view(2, 3, 4, 320).to(vk), x.view(4, 6, 320).transpose(0, 1).contiguous().to(vk).transpose(0, 1)):
        for W in (w.to(vk), wide_w.to(vk)[::2, 16:336], off_w.to(vk)[:, 1:], w.t().contiguous().to(vk).t()):
            got = torch_vulkan.int8_linear(X, W, torch.stack((s, s), 1).to(vk)[:, 0], b.to(vk))
            assert got.shape == (*X.shape[:-1], 72) and torch.equal(got.cpu().view(24, 72), want)
    one = torch_vulkan.int8_linear(x[0].to(vk), w.to(vk), s.to(vk), b.to(vk))
    assert one.shape == (72,) and torch.equal(one.cpu(), want[0])
    codes, scale = torch_vulkan.quantize_int8_rows(x[0].to(vk))
    one = torch_vulkan.int8_linear(codes, w.to(vk), s.to(vk), b.to(vk), x_scale=scale, out_dtype=dtype)
    assert scale.shape == () and torch.equal(one.cpu(), want[0])
    codes, scale = torch_vulkan.quantize_int8_rows(x.view(4, 6, 320).to(vk))
    got = torch_vulkan.int8_linear(codes.transpose(0, 1), w.to(vk), s.to(vk), b.to(vk), x_scale=scale.transpose(0, 1), out_dtype=dtype)
    assert torch.equal(got.transpose(0, 1).cpu().reshape(24, 72), want)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 5, 20, 100, 300])
def test_scales_and_bias_off_their_lines(M):
    """Slices of longer vectors, which do not begin on 16 bytes; rows given with scales of their own."""
    x, w, s, b = operands(M, 64, 320, torch.float16, 17)
    X, W = x.to(vk), w.to(vk)
    want = torch_vulkan.int8_linear(X, W, s.to(vk), b.to(vk)).cpu()
    codes, scale = torch_vulkan.quantize_int8_rows(X)
    for k in (1, 2, 3):
        S, B = torch.cat([torch.ones(k), s]).to(vk)[k:], torch.cat([torch.ones(k).half(), b]).to(vk)[k:]
        xs = torch.cat([torch.ones(k), scale.cpu()]).to(vk)[k:]
        assert torch.equal(torch_vulkan.int8_linear(X, W, S, B).cpu(), want)
        assert torch.equal(torch_vulkan.int8_linear(codes, W, S, B, x_scale=xs, out_dtype=torch.float16).cpu(), want)
        assert torch.equal(torch_vulkan.dequant_int8_rows(W, S).cpu(), torch_vulkan.dequant_int8_rows(w, s))


@pytest.mark.gpu
def test_nothing_to_do():
    x, w, s, b = (t.to(vk) for t in operands(4, 24, 32, torch.bfloat16, 1))
    assert torch_vulkan.int8_linear(x[:0], w, s, b).shape == (0, 24)
    assert torch_vulkan.int8_linear(x, w[:0], s[:0], b[:0]).shape == (4, 0)
    assert torch.equal(torch_vulkan.int8_linear(x[:, :0], w[:, :0], s, b).cpu(), b.cpu().expand(4, 24))
    assert torch_vulkan.int8_linear(x[:, :0], w[:, :0], s).cpu().abs().sum() == 0
    X, B = x[:0].detach().requires_grad_(), b.detach().requires_grad_()
    dx, db = torch.autograd.grad(torch_vulkan.int8_linear(X, w, s, B).sum(), (X, B))
    assert dx.shape == (0, 32) and db.cpu().abs().sum() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("M", [3, 40, 300])
def test_what_is_not_finite_stays_in_its_row_and_column(M):
    x, w, s, b = operands(M, 72, 320, torch.bfloat16, 9)
    want = torch_vulkan.int8_linear(x.to(vk), w.to(vk), s.to(vk), b.to(vk)).cpu()
    x[1, 5], s[7] = float("inf"), float("nan")
    x[2] = 0
    got = torch_vulkan.int8_linear(x.to(vk), w.to(vk), s.to(vk), b.to(vk)).cpu()
    hit = torch.zeros(M, 72, dtype=torch.bool)
    hit[1], hit[:, 7] = True, True
    assert torch.isnan(got[hit]).all() and torch.isfinite(got[~hit]).all()
    rest = ~hit
    rest[2] = False
    assert torch.equal(got[rest], want[rest]) and torch.equal(got[2][~hit[2]], b[~hit[2]])


@pytest.mark.gpu
def test_refusals():
    x, w, s, b = (t.to(vk) for t in operands(4, 24, 32, torch.bfloat16, 1))
    c, cs = torch_vulkan.quantize_int8_rows(x)
    lin = torch_vulkan.int8_linear
    for match, call in [("vk tensor", lambda: lin(x.float(), w, s)), ("vk device", lambda: lin(x, w.cpu(), s)), ("int8", lambda: lin(x, w.float(), s)),
                        ("float32", lambda: lin(x, w, s.bfloat16())), ("last dimension", lambda: lin(x, w, s[:3])), (r"\[N, K\]", lambda: lin(x[:, :16], w, s)),
                        ("bias", lambda: lin(x, w, s, b.half())), ("bias", lambda: lin(x, w, s, b[:3])), ("x_scale", lambda: lin(c, w, s)),
                        ("x_scale", lambda: lin(x, w, s, x_scale=cs)), ("x's scale", lambda: lin(c, w, s, x_scale=cs[:2])),
                        ("out_dtype", lambda: lin(c, w, s, x_scale=cs, out_dtype=torch.float32)), ("out_dtype", lambda: lin(x, w, s, out_dtype=torch.float16)),
                        ("no gradient", lambda: lin(x, w, s.detach().requires_grad_())), ("no gradient", lambda: lin(c, w, s, x_scale=cs.detach().requires_grad_())),
                        ("131056", lambda: lin(torch.zeros(1, 131072, dtype=torch.bfloat16).to(vk), torch.zeros(1, 131072, dtype=torch.int8).to(vk), s[:1])),
                        ("last dimension", lambda: torch_vulkan.dequant_int8_rows(c, cs[:2])), ("out_dtype", lambda: torch_vulkan.dequant_int8_rows(c, cs, torch.int32)),
                        ("float32", lambda: torch_vulkan.quantize_int8_rows(c))]:
        with pytest.raises(RuntimeError, match=match):
            call()


@pytest.mark.gpu
def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fwd

    x, w, s, b = (t.to(vk) for t in operands(4, 64, 96, torch.bfloat16, 1))
    with fwd.dual_level():
        for wants in (False, True):
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch_vulkan.int8_linear(fwd.make_dual(x.detach().requires_grad_(wants), torch.ones_like(x)), w, s, b)
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch_vulkan.int8_linear(x, w, s, fwd.make_dual(b.detach().requires_grad_(wants), torch.ones_like(b)))
        y = torch_vulkan.int8_linear(x.detach().requires_grad_(), w, s, b)
        with pytest.raises(RuntimeError, match="forward-mode"):
            y.backward(fwd.make_dual(torch.ones_like(y), torch.ones_like(y)))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(6, 96), (2, 3, 96), (96,), (0, 96), (6, 50)])
def test_in_place_operations_on_the_output(shape):
    x, w, s, b = operands(6, 64, shape[-1], torch.bfloat16, 31)
    n = int(np.prod(shape))
    W, S, X, B = w.to(vk), s.to(vk), x.flatten()[:n].view(shape).to(vk).requires_grad_(), b.to(vk).requires_grad_()
    A = torch.randn((*shape[:-1], 64), generator=torch.Generator().manual_seed(6)).bfloat16().to(vk).requires_grad_()

    def run(add):
        y = add(torch_vulkan.int8_linear(X, W, S, B), A)
        y = add(y, y * 2)
        return [y, *torch.autograd.grad(y, [X, B, A], torch.ones_like(y))]

    for a, c in zip(run(lambda y, z: y.add_(z)), run(lambda y, z: y + z)):
        assert torch.equal(a.detach().cpu(), c.detach().cpu())


@pytest.mark.gpu
def test_autocast_runs_it_in_its_type():
    x, w, s, b = operands(6, 64, 96, torch.float32, 2)
    X, B = x.to(vk).requires_grad_(), b.to(vk).requires_grad_()
    g = torch.ones(6, 64)
    for dtype in HALF:
        with torch.autocast("vk", dtype=dtype):
            y = torch_vulkan.int8_linear(X, w.to(vk), s.to(vk), B)
            c, cs = torch_vulkan.quantize_int8_rows(X.detach().to(dtype))
            z = torch_vulkan.int8_linear(c, w.to(vk), s.to(vk), B.detach(), x_scale=cs)
            o = torch_vulkan.int8_linear(c, w.to(vk), s.to(vk), B.detach(), x_scale=cs, out_dtype=torch.float16)
        assert y.dtype == z.dtype == dtype and o.dtype == torch.float16
        want = torch_vulkan.int8_linear(x.to(dtype).to(vk), w.to(vk), s.to(vk), b.to(dtype).to(vk))
        assert torch.equal(y.detach().cpu(), want.cpu()) and torch.equal(z.cpu(), want.cpu())
        dx, db = torch.autograd.grad(y, (X, B), g.to(dtype).to(vk))
        assert dx.dtype == db.dtype == torch.float32
        check_back(dx, g, w, s, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 20, 200])
def test_replayed_graph(M):
    rt, out = abi.Runtime(), {}
    x, w, s, b = (t.to(vk) for t in operands(M, 512, 2000, torch.bfloat16, 8))
    g = torch.randn((M, 512), generator=torch.Generator().manual_seed(1)).bfloat16().to(vk)
    X = x.detach().requires_grad_()

    def run():
        with torch.autograd.set_multithreading_enabled(False):
            y = torch_vulkan.int8_linear(X, w, s, b)
            (dx,) = torch.autograd.grad(y, X, g)
        return y.detach(), dx

    eager = [t.cpu() for t in run()]

    def record():
        out["y"] = run()

    gid = rt.graph(record)
    for _ in range(3):
        for t in out["y"]:
            t.zero_()
        rt.graph_launch(gid)
        assert all(torch.equal(a.cpu(), b_) for a, b_ in zip(out["y"], eager))
        assert all(torch.equal(a.cpu(), b_) for a, b_ in zip(run(), eager))
    rt.graph_destroy(gid)


@pytest.mark.gpu
@pytest.mark.parametrize("K", [64, 1040, 2048])
@pytest.mark.parametrize("M", [1, 2, 3, 4, 7, 8])
def test_few_rows_where_they_lie(M, K):
    """Rows that the product quantises itself: off their lines, apart, repeated, of zeros, not finite; the codes of the packed rows."""
    x, w, s, b = operands(M, 40, K, torch.bfloat16, K)
    x[M // 2, 5:] = 0
    if M > 2:
        x[1], x[2, 7] = 0, float("nan")
    codes, scale = torch_vulkan.quantize_int8_rows(x)
    W, S, B = w.to(vk), s.to(vk), b.to(vk)
    want = torch_vulkan.int8_linear(codes.to(vk), W, S, B, x_scale=scale.to(vk)).cpu()
    wide = torch.full((2 * M, K + 13), 1e4, dtype=torch.bfloat16)
    wide[::2, 3 : K + 3] = x
    for X in (x.to(vk), wide.to(vk)[::2, 3 : K + 3]):
        got = torch_vulkan.int8_linear(X, W, S, B).cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))
    one = torch_vulkan.int8_linear(x[:1].to(vk).expand(M, K), W, S, B).cpu()
    assert torch.equal(torch.nan_to_num(one), torch.nan_to_num(want[:1].expand(M, 40)))


@pytest.mark.gpu
def test_rows_far_apart():
    """8-bit rows 2^30 bytes apart are copied together first, 16-bit ones are quantised where they lie."""
    x, w, s, b = operands(3, 24, 64, torch.bfloat16, 3)
    far = torch.zeros((1 << 31) + 4096, dtype=torch.int8, device=vk)
    wide = far.as_strided((3, 64), (1 << 30, 1))
    wide.copy_(w[:3].to(vk))
    got = torch_vulkan.int8_linear(x.to(vk), wide, s[:3].to(vk), b[:3].to(vk))
    assert torch.equal(got.cpu(), torch_vulkan.int8_linear(x.to(vk), w[:3].to(vk), s[:3].to(vk), b[:3].to(vk)).cpu())
    assert torch.equal(torch_vulkan.dequant_int8_rows(wide, s[:3].to(vk)).cpu(), torch_vulkan.dequant_int8_rows(w[:3], s[:3]))
    G = torch.randn((3, 3), generator=torch.Generator().manual_seed(1)).bfloat16().to(vk)
    X = x.to(vk).requires_grad_()
    (dx,) = torch.autograd.grad(torch_vulkan.int8_linear(X, wide, s[:3].to(vk)), X, G)
    (want,) = torch.autograd.grad(torch_vulkan.int8_linear(X, w[:3].to(vk), s[:3].to(vk)), X, G)
    assert torch.equal(dx.cpu(), want.cpu())
    del far, wide
    far = torch.zeros((1 << 31) + 4096, dtype=torch.bfloat16, device=vk)
    wide = far.as_strided((3, 64), (1 << 30, 1))
    wide.copy_(x.to(vk))
    got = torch_vulkan.int8_linear(wide, w.to(vk), s.to(vk), b.to(vk))
    assert torch.equal(got.cpu(), torch_vulkan.int8_linear(x.to(vk), w.to(vk), s.to(vk), b.to(vk)).cpu())


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(20000, 72, 48), (3, 50000, 32), (700, 20011, 16)])
def test_long_and_thin(M, N, K):
    x, w, s, b = operands(M, N, K, torch.bfloat16, 5)
    codes, scale = packed(x)
    y, want = product(codes, scale, w, s, b)
    X, B = x.to(vk).requires_grad_(), b.to(vk).requires_grad_()
    out = torch_vulkan.int8_linear(X, w.to(vk), s.to(vk), B)
    check_forward(out, y, want, torch.bfloat16)
    g = torch.randn((M, N), generator=torch.Generator().manual_seed(3)).bfloat16()
    dx, db = torch.autograd.grad(out, (X, B), g.to(vk))
    check_back(dx, g, w, s, torch.bfloat16)
    want = f64(g).sum(0)
    assert (np.abs(f64(db) - want) <= 2.0**-8 * np.abs(want) + M * 2.0**-24 * np.abs(f64(g)).sum(0)).all()


@pytest.mark.gpu
def test_an_expanded_gradient():
    x, w, s, b = operands(6, 24, 64, torch.bfloat16, 3)
    X, B = x.to(vk).requires_grad_(), b.to(vk).requires_grad_()
    dx, db = torch.autograd.grad(torch_vulkan.int8_linear(X, w.to(vk), s.to(vk), B).sum(), (X, B))
    check_back(dx, torch.ones(6, 24).bfloat16(), w, s, torch.bfloat16)
    assert (db.cpu() == 6).all()


@pytest.mark.gpu
@pytest.mark.parametrize("N", [72, 70])
@pytest.mark.parametrize("M", [1, 5, 12, 20, 40, 140, 300])
def test_far_scales_whose_product_is_near(M, N):
    """Sums of which one scale's share alone passes fp32's range, beside rows of ordinary size."""
    K = 320
    x, w, s, b = operands(M, N, K, torch.bfloat16, M)
    x[::2] *= 2.0**120
    x[::4] = x[::4].abs()  # codes of one sign: the largest sums
    w[:8] = w[:8].abs()
    x[0, :K] = 1e36
    codes, scale = packed(x)
    y, want = product(codes, scale, w, s, b)
    assert (np.abs(y).max() < 2.0**127) and (np.abs(codes.astype(np.float64) @ f64(w).T) * scale[:, None]).max() > 2.0**128
    X, W, S, B, C, XS = (t.to(vk) for t in (x, w, s, b, torch.from_numpy(codes), torch.from_numpy(scale)))
    check_forward(torch_vulkan.int8_linear(X, W, S, B), y, want, torch.bfloat16)
    check_forward(torch_vulkan.int8_linear(C, W, S, B, x_scale=XS), y, want, torch.bfloat16)
    near = (s * 2.0**-118).float()  # and an fp16 result under scales that all but cancel
    y, _ = product(codes, scale, w, near, None)
    y[1::2], want = 0, None
    got = torch_vulkan.int8_linear(C, W, near.to(vk), x_scale=XS, out_dtype=torch.float16)
    check_forward(got[::2], y[::2], y[::2], torch.float16)


def test_tangents_and_gradients_are_not_dropped_on_the_cpu():
    import torch.autograd.forward_ad as fwd

    x = torch.randn(4, 70)
    with fwd.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch_vulkan.quantize_int8_rows(fwd.make_dual(x, x))
        assert torch_vulkan.quantize_int8_rows(x)[0].shape == (4, 70)


@pytest.mark.gpu
def test_tangents_and_gradients_are_not_dropped():
    """Packing and unpacking refuse a tangent, and unpacking a scale whose gradient would be lost."""
    import torch.autograd.forward_ad as fwd

    x = torch.randn(4, 70).to(vk)
    c, s = torch_vulkan.quantize_int8_rows(x)
    with fwd.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch_vulkan.quantize_int8_rows(fwd.make_dual(x, x))
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch_vulkan.dequant_int8_rows(c, fwd.make_dual(s, s))
    wants = s.detach().requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient"):
        torch_vulkan.dequant_int8_rows(c, wants)
    with torch.no_grad():
        assert torch.equal(torch_vulkan.dequant_int8_rows(c, wants).cpu(), torch_vulkan.dequant_int8_rows(c, s).cpu())
    assert torch.equal(torch_vulkan.quantize_int8_rows(x.detach().requires_grad_())[0].cpu(), c.cpu())  # a weight at rest


@pytest.mark.gpu
def test_autocast_does_not_pass_over_a_named_type():
    x, w, s, b = (t.to(vk) for t in operands(6, 64, 96, torch.float16, 2))
    with torch.autocast("vk", dtype=torch.bfloat16):
        for out in (torch.float16, torch.float32):
            with pytest.raises(RuntimeError, match="out_dtype"):
                torch_vulkan.int8_linear(x, w, s, b, out_dtype=out)
        assert torch_vulkan.int8_linear(x, w, s, b, out_dtype=torch.bfloat16).dtype == torch.bfloat16


# Each tile at lengths of K that its loop takes in one round and in several, with as few and as many steps left behind it, whole lines
# of y and odd ends.
LONG_PRODUCTS = [(4100, 2056, 1024), (4090, 4095, 1616), (4100, 2056, 2064), (4090, 4095, 2200), (1500, 4104, 640), (2000, 2055, 880), (1500, 4104, 2064), (2000, 2055, 2050),
                 (1030, 2056, 1024), (700, 4101, 1616), (700, 4104, 2064), (1030, 2050, 2200), (500, 4101, 272), (520, 2056, 880), (700, 2050, 640), (1024, 2048, 2064),
                 (600, 2050, 2050), (130, 1032, 2048), (300, 1030, 3216), (130, 1032, 4112), (300, 1030, 4100)]


def test_products_reach_every_tile_and_its_loop():
    """By the plan itself: a change of its rule that leaves a tile, its unguarded loop or the steps behind it to no test fails here."""
    import ctypes

    plan = ctypes.CDLL(abi._LIB_PATH).hrt_i8_mm_plan
    plan.argtypes, plan.restype = [ctypes.c_void_p, ctypes.c_void_p], ctypes.c_int32
    seen = set()
    for M, N, K in PRODUCTS + LONG_PRODUCTS:
        rounds = ctypes.c_int64()
        args = abi.I8MmArgs(x_scale=4, M=M, N=N, K=(K + 15) // 16 * 16)  # rows are filled up to 16
        seen.add((plan(ctypes.byref(args), ctypes.byref(rounds)), N % 8 == 0, min(rounds.value, 2)))
    for tile in range(abi.I8_MM_TILES):
        for lines in (True, False):
            assert (tile, lines, 2) in seen
        for rounds in (0, 1):
            assert (tile, True, rounds) in seen or (tile, False, rounds) in seen
    assert {t for t, _, _ in seen} == {-1, *range(abi.I8_MM_TILES)}
    none = ctypes.c_int64(7)
    assert plan(None, None) == -1 and plan(ctypes.byref(abi.I8MmArgs()), ctypes.byref(none)) == -1 and none.value == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("M,N,K", LONG_PRODUCTS)
def test_long_products(M, N, K, dtype):
    test_linear(M, N, K, dtype)


def f16_quotients():
    """Rows under every f16 mantissa as the largest value, with every mantissa not above it in its own binade, where quotients come
    closest to a border (a 2^19th of their size), and the closest of the binades below."""
    man = 1 + torch.arange(1024) / 1024
    top = man.unsqueeze(-1)
    x = (man * torch.exp2(-torch.arange(9.0)).unsqueeze(-1)).flatten().expand(1024, -1)
    x = torch.cat([top, torch.where(x <= top, x, torch.zeros(()))], -1)
    return torch.cat([x, -x]).half()


def test_how_close_quotients_come_to_a_border():
    """254 a and k b of 11-bit a <= b, k odd, differ by 1 at least, of at most 254 x 2047: 2^-19, and 2^-32 for 24 bits."""
    a = torch.arange(1024, 2048, dtype=torch.int64)
    gap = 1.0
    for b in a.tolist():
        n = 254 * a[a <= b]
        k = n // b
        near = torch.minimum((n - (k - 1 + k % 2) * b).abs(), (n - (k + 1 + k % 2) * b).abs())
        gap = min(gap, float((near[near > 0] / n[near > 0]).min()))
    assert 2.0**-19 < gap < 2.0**-18


def test_every_f16_quotient_on_the_cpu():
    x = f16_quotients()[::7]
    same(torch_vulkan.quantize_int8_rows(x), packed(x))


@pytest.mark.gpu
def test_every_f16_quotient():
    x = f16_quotients()
    same(torch_vulkan.quantize_int8_rows(x.to(vk)), packed(x))
