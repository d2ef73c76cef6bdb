"""Microscaled 4-bit floating point: packing against the format's definition evaluated in 64 bits, products against
float64 products of the values that the packed operands stand for.

Tolerances.  Packing and unpacking are exact.  A product's output is rounded once (half a step of the output type,
finfo.eps / 2 relative, and half the smallest subnormal of f16); its fp32 sum of K exact products is off by at most K
roundings of the running sum's size, K 2^-24 sum |x| |w|, in any order."""

import numpy as np
import pytest
import torch

import torch_vulkan
from torch_vulkan import abi

vk = torch.device("vk")
E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def values(codes, scale, cols):
    """Float64 values of packed rows."""
    c, s = codes.cpu().numpy(), scale.cpu().numpy().astype(np.int64)
    code = np.stack((c & 15, c >> 4), -1).reshape(c.shape[0], 2 * c.shape[1])[:, :cols].astype(np.int64)
    v = E2M1[code & 7] * np.where(code & 8, -1.0, 1.0)
    two = np.where(s == 255, np.nan, np.ldexp(1.0, s - 127))
    return v * np.repeat(two, 32, axis=1)[:, :cols]


def rounded(x):
    """The values that packing keeps, from the definition: nearest multiple of the step around each value, ties to even."""
    x = x.double().cpu().numpy()
    rows, cols = x.shape
    b = np.zeros((rows, (cols + 31) // 32 * 32))
    b[:, :cols] = x
    b = b.reshape(rows, -1, 32)
    top = np.abs(b).max(-1, keepdims=True)
    with np.errstate(invalid="ignore"):
        e = np.maximum(np.frexp(np.where(np.isfinite(top), top, 1.0))[1] - 1 - 2, -127)
        e = np.where(top == 0, -127, e)
        unit = np.ldexp(1.0, e)
        v = b / unit
        step = np.where(np.abs(v) < 2, 0.5, np.where(np.abs(v) < 4, 1.0, 2.0))
        out = np.clip(np.rint(v / step) * step, -6, 6) * unit
    out = np.where(np.isfinite(top), out, np.nan)
    return out.reshape(rows, -1)[:, :cols]


def sample(rows, cols, dtype, seed):
    """Rows of very different sizes, with values that sit on every rounding border."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, cols), generator=g) * torch.exp2(torch.randint(-12, 12, (rows, 1), generator=g).float())
    border = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.96875, 0.0, -0.0])
    pick = border[torch.randint(0, len(border), (rows, cols), generator=g)] * (torch.randint(0, 2, (rows, cols), generator=g) * 2 - 1)
    x = torch.where(torch.arange(rows).unsqueeze(1) % 2 == 0, x, pick)
    x[rows // 2] = 0
    return x.to(dtype)


def same(a, b):
    return np.array_equal(a, b, equal_nan=True)


SHAPES = [(1, 1), (3, 31), (5, 32), (4, 33), (7, 64), (2, 100), (9, 1000), (64, 2048), (33, 4100)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_cpu_form_follows_the_definition(shape, dtype):
    x = sample(*shape, dtype, sum(shape))
    codes, scale = torch_vulkan.quantize_mxfp4(x)
    assert same(values(codes, scale, shape[1]), rounded(x))
    for out in DTYPES:
        y = torch_vulkan.dequant_mxfp4(codes, scale, out, cols=shape[1])
        assert torch.equal(y, torch.from_numpy(values(codes, scale, shape[1])).to(out))


def test_cpu_refusals():
    c, s = torch_vulkan.quantize_mxfp4(torch.randn(4, 70))
    with pytest.raises(RuntimeError, match="rows of 72 values"):
        torch_vulkan.dequant_mxfp4(c, s, cols=72)
    with pytest.raises(RuntimeError, match="uint8"):
        torch_vulkan.dequant_mxfp4(c.int(), s)
    with pytest.raises(RuntimeError, match="float32"):
        torch_vulkan.quantize_mxfp4(torch.zeros(4, 4, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="vk tensor"):
        torch_vulkan.mxfp4_linear(torch.zeros(4, 70), c, s)


def extremes():
    """Blocks at both ends of the exponent range, infinities, NaN, subnormals."""
    f = torch.finfo(torch.float32)
    rows = [[f.max, 1.0], [f.tiny, f.tiny * 3], [f.smallest_normal / 4, 1e-40], [2.0**-125, 2.0**-126], [float("inf"), 1.0],
            [float("nan"), 1.0], [-f.max, f.max / 16], [2.0**-149, 0.0], [-0.0, 0.0]]
    x = torch.zeros(len(rows), 64)
    for i, r in enumerate(rows):
        x[i, 3:5] = torch.tensor(r)
        x[i, 40] = i + 1.0  # the row's other block stays ordinary
    return x


def test_cpu_extremes():
    x = extremes()
    c, s = torch_vulkan.quantize_mxfp4(x)
    assert same(values(c, s, 64), rounded(x))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_packing_matches_the_cpu_form_bit_for_bit(shape, dtype):
    x = sample(*shape, dtype, 1 + sum(shape))
    want = torch_vulkan.quantize_mxfp4(x)
    got = torch_vulkan.quantize_mxfp4(x.to(vk))
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])
    for out in DTYPES:
        y = torch_vulkan.dequant_mxfp4(*got, out, cols=shape[1])
        assert torch.equal(y.cpu(), torch_vulkan.dequant_mxfp4(*want, out, cols=shape[1]))


@pytest.mark.gpu
def test_extremes_on_the_device():
    x = extremes()
    want = torch_vulkan.quantize_mxfp4(x)
    got = torch_vulkan.quantize_mxfp4(x.to(vk))
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])
    every = torch.arange(256, dtype=torch.uint8)  # all code pairs under all scales
    codes = every.view(1, 256).expand(256, 256).contiguous().view(-1, 16)
    scale = every.view(256, 1).expand(256, 16).contiguous().view(-1, 1)
    for out in DTYPES:
        y = torch_vulkan.dequant_mxfp4(codes.to(vk), scale.to(vk), out).cpu()
        assert same(y.double().numpy(), torch_vulkan.dequant_mxfp4(codes, scale, out).double().numpy())


@pytest.mark.gpu
def test_packing_of_views():
    x = sample(12, 4096, torch.bfloat16, 3)
    base = x.to(vk)
    for view, ref in ((base[:, 8:1032], x[:, 8:1032]), (base[:, 3:100], x[:, 3:100]), (base.t(), x.t()), (base[:1].expand(5, 4096), x[:1].expand(5, 4096)),
                      (base.view(3, 4, 4096), x.view(3, 4, 4096)), (base[0], x[0]), (base[:0], x[:0]), (base[:, :0], x[:, :0])):
        got, want = torch_vulkan.quantize_mxfp4(view), torch_vulkan.quantize_mxfp4(ref)
        assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])
        y = torch_vulkan.dequant_mxfp4(*got, torch.float16, cols=ref.shape[-1])
        assert torch.equal(y.cpu(), torch_vulkan.dequant_mxfp4(*want, torch.float16, cols=ref.shape[-1]))


def operands(M, N, K, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn((N, K), generator=g) * torch.exp(torch.randn((N, 1), generator=g)) * 0.05
    x = torch.randn((M, K), generator=g).to(dtype)
    return x, *torch_vulkan.quantize_mxfp4(w), torch.randn((N,), generator=g).to(dtype)


def check(y, ref, size, K, dtype):
    """y against float64 ref; size: sum |x| |w| of each output."""
    f = torch.finfo(dtype)
    # the rounding applies to the sum as it came out, hence the factor of 1.01 (K 2^-24 < 0.01)
    tol = 1.01 * (f.eps / 2) * np.abs(ref) + 1.01 * K * 2.0**-24 * size + f.smallest_normal * f.eps / 2
    err = np.abs(y.detach().cpu().double().numpy() - ref)
    assert y.dtype == dtype and (err <= tol).all(), (float((err / tol).max()), np.unravel_index(np.argmax(err / tol), err.shape))


# few rows and every tile, whole and ragged; K in whole and partial steps, scale rows of odd lengths
PRODUCTS = [(1, 64, 64), (1, 48, 96), (3, 17, 32), (16, 128, 2048), (17, 100, 320), (33, 1, 160), (64, 50, 1056), (65, 64, 64), (77, 70, 96),
            (200, 130, 320), (129, 300, 2080), (1000, 3001, 224), (1024, 3008, 128), (1537, 4000, 160), (4100, 4098, 96), (4096, 4096, 512)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES[1:])
@pytest.mark.parametrize("quantize", [False, True])
@pytest.mark.parametrize("M,N,K", PRODUCTS)
def test_linear(M, N, K, quantize, dtype):
    x, codes, scale, b = operands(M, N, K, dtype, M + N + K)
    w = values(codes, scale, K)
    xr = values(*torch_vulkan.quantize_mxfp4(x), K) if quantize else x.double().numpy()
    ref, size = xr @ w.T, np.abs(xr) @ np.abs(w).T
    X, C, S, B = (t.to(vk) for t in (x, codes, scale, b))
    check(torch_vulkan.mxfp4_linear(X, C, S, quantize_input=quantize), ref, size, K, dtype)
    bias = b.double().numpy()
    check(torch_vulkan.mxfp4_linear(X, C, S, B, quantize), ref + bias, size + np.abs(bias), K + 1, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES[1:])
@pytest.mark.parametrize("quantize", [False, True])
@pytest.mark.parametrize("M,N,K", [(7, 136, 4160), (16, 40, 2112), (1000, 1000, 1280), (2000, 2000, 1280), (2500, 2000, 1280), (2500, 2001, 1184),
                                   (1000, 8200, 1280), (1000, 8200, 1184)])
def test_linear_over_several_blocks_of_scales(M, N, K, quantize, dtype):
    """Every tile over more than 1024 values of K, and few rows over more than 2048; every 37th row is compared, and the last."""
    x, codes, scale, b = operands(M, N, K, dtype, M + N + K)
    some = sorted({*range(0, M, 37), M - 1})
    w, part = values(codes, scale, K), x[some]
    xr = values(*torch_vulkan.quantize_mxfp4(part), K) if quantize else part.double().numpy()
    bias = b.double().numpy()
    y = torch_vulkan.mxfp4_linear(*(t.to(vk) for t in (x, codes, scale, b)), quantize)
    check(y.cpu()[some], xr @ w.T + bias, np.abs(xr) @ np.abs(w).T + np.abs(bias), K + 1, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("quantize", [False, True])
@pytest.mark.parametrize("M,N,K", [(5, 40, 33), (70, 64, 100), (3, 8, 1), (4, 8, 0), (0, 8, 64), (4, 0, 64)])
def test_linear_of_rows_that_end_inside_a_block_and_of_nothing(M, N, K, quantize):
    x, codes, scale, b = operands(M, N, max(K, 1), torch.bfloat16, 9)
    x, codes, scale = x[:, :K], codes[:, : (K + 1) // 2], scale[:, : (K + 31) // 32]
    w = values(codes, scale, K)
    xr = values(*torch_vulkan.quantize_mxfp4(x), K) if quantize else x.double().numpy()
    y = torch_vulkan.mxfp4_linear(x.to(vk), codes.to(vk), scale.to(vk), b.to(vk), quantize)
    assert y.shape == (M, N)
    check(y, xr @ w.T + b.double().numpy(), np.abs(xr) @ np.abs(w).T + np.abs(b.double().numpy()), K + 1, torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [2, 80])
def test_linear_of_views(M):
    """Row strides, offsets that are not on 16 bytes, broadcast rows, leading dimensions, packed weights out of a larger block."""
    K, N = 96, 72
    x, codes, scale, b = operands(M, N, K, torch.float16, 5)
    C, S = codes.to(vk), scale.to(vk)
    wide = torch.zeros(M, K + 24, dtype=x.dtype)
    wide[:, 5:5 + K] = x
    big_c, big_s = torch.zeros(N * (K // 2) + 7, dtype=torch.uint8), torch.zeros(N * 3 + 1, dtype=torch.uint8)
    big_c[7:], big_s[1:] = codes.flatten(), scale.flatten()
    Cv, Sv = big_c.to(vk)[7:].view(N, K // 2), big_s.to(vk)[1:].view(N, 3)
    for quantize in (False, True):
        want = torch_vulkan.mxfp4_linear(x.to(vk), C, S, b.to(vk), quantize).cpu()
        for X in (wide.to(vk)[:, 5:5 + K], x.t().contiguous().to(vk).t(), x.to(vk)):
            assert torch.equal(torch_vulkan.mxfp4_linear(X, Cv, Sv, b.to(vk), quantize).cpu(), want)
        one = torch_vulkan.mxfp4_linear(x[:1].to(vk).expand(M, K), C, S, b.to(vk), quantize).cpu()
        assert torch.equal(one, want[:1].expand(M, N))
        lead = torch_vulkan.mxfp4_linear(x.view(2, M // 2, K).to(vk), C, S, b.to(vk), quantize).cpu()
        assert torch.equal(lead, want.view(2, M // 2, N))


@pytest.mark.gpu
@pytest.mark.parametrize("M", [8, 100])
def test_nan_stays_in_its_row_and_column(M):
    x, codes, scale, _ = operands(M, 96, 192, torch.bfloat16, 2)
    want = torch_vulkan.mxfp4_linear(x.to(vk), codes.to(vk), scale.to(vk), quantize_input=True).cpu()
    x[3, 70], scale[5, 1] = float("inf"), 255
    got = torch_vulkan.mxfp4_linear(x.to(vk), codes.to(vk), scale.to(vk), quantize_input=True).cpu()
    hit = torch.zeros(M, 96, dtype=torch.bool)
    hit[3], hit[:, 5] = True, True
    assert torch.isnan(got[hit]).all() and torch.equal(got[~hit], want[~hit])


@pytest.mark.gpu
@pytest.mark.parametrize("quantize", [False, True])
@pytest.mark.parametrize("M,N,K", [(1, 64, 64), (37, 130, 320), (300, 520, 96), (40, 64, 50)])
def test_gradients(M, N, K, quantize):
    """dx = g W and db = the sum of g: one rounding of an fp32 sum of exact products each."""
    dtype = torch.bfloat16
    x, codes, scale, b = operands(M, N, K, dtype, 17)
    g = torch.randn((M, N), generator=torch.Generator().manual_seed(1)).to(dtype)
    X, B = x.to(vk).requires_grad_(), b.to(vk).requires_grad_()
    y = torch_vulkan.mxfp4_linear(X, codes.to(vk), scale.to(vk), B, quantize)
    dx, db = torch.autograd.grad(y, (X, B), g.to(vk))
    w, g64 = values(codes, scale, K), g.double().numpy()
    check(dx, g64 @ w, np.abs(g64) @ np.abs(w), N, dtype)
    check(db, g64.sum(0), np.abs(g64).sum(0), M, dtype)
    # only what is asked for; a gradient broadcast from one value; leading dimensions
    X3 = x.view(1, M, K).to(vk).requires_grad_()
    torch_vulkan.mxfp4_linear(X3, codes.to(vk), scale.to(vk), quantize_input=quantize).sum().backward()
    check(X3.grad.view(M, K), np.ones((M, N)) @ w, np.ones((M, N)) @ np.abs(w), N, dtype)
    frozen = torch_vulkan.mxfp4_linear(x.to(vk), codes.to(vk), scale.to(vk), B, quantize)
    frozen.sum().backward()
    check(B.grad, np.full(N, float(M)), np.full(N, float(M)), M, dtype)
    with torch.no_grad():
        assert not torch_vulkan.mxfp4_linear(X, codes.to(vk), scale.to(vk), B, quantize).requires_grad


@pytest.mark.gpu
def test_refusals():
    x, codes, scale, b = (t.to(vk) for t in operands(4, 64, 96, torch.bfloat16, 1))
    call = torch_vulkan.mxfp4_linear
    for args, text in (((x.float(), codes, scale), "bfloat16 or float16"), ((x[:, :64], codes, scale), "rows of 64 values"),
                       ((x, codes.view(torch.int8), scale), "uint8"), ((x, codes, scale[:, :2]), "scales"), ((x, codes[:, :40], scale), "codes"),
                       ((x, codes, scale[:63]), "agree"), ((x, codes.cpu(), scale), "vk"), ((x, codes, scale, b[:63]), "bias"),
                       ((x, codes, scale, b.float()), "bias"), ((x, codes, scale, b.cpu()), "bias"), ((x, codes[0], scale[0]), "two")):
        with pytest.raises(RuntimeError, match=text):
            call(*args)
    with pytest.raises(RuntimeError, match="float32"):
        torch_vulkan.quantize_mxfp4(codes)
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        torch_vulkan.dequant_mxfp4(codes, scale, torch.float64)
    # the C ABI checks for itself
    rt, y = abi.Runtime(), torch.empty(4, 64, dtype=torch.bfloat16, device=vk)

    def args(**kw):
        a = abi.Mx4MmArgs(x=x.data_ptr(), w=codes.data_ptr(), w_scale=scale.data_ptr(), y=y.data_ptr(), M=4, N=64, K=96, x_sm=96)
        for k, v in kw.items():
            setattr(a, k, v)
        return a

    for kw, text in ((dict(K=80), "multiple of 32"), (dict(x_sm=100), "multiple of 8"), (dict(M=0), "empty"), (dict(x=x.data_ptr() + 2), "aligned"),
                     (dict(M=1 << 20), "x"), (dict(N=1 << 20), "w"), (dict(y=0), "y")):
        with pytest.raises(RuntimeError, match=text):
            rt.dispatch("mx4_mm_bf16", args(**kw))
    with pytest.raises(RuntimeError, match="codes"):
        rt.dispatch("mx4_quant_bf16", abi.Mx4Args(x=x.data_ptr(), codes=0, scale=scale.data_ptr(), rows=4, cols=96, x_sr=96))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES[1:])
@pytest.mark.parametrize("M,N,K", [(1, 8, 32), (3, 200, 96), (40, 64, 128), (31, 264, 160), (500, 2048, 4096), (500, 2000, 4128), (1500, 1000, 2080),
                                   (1010, 456, 8160), (8100, 456, 4064)])
def test_the_inputs_gradient_on_every_tile(M, N, K, dtype):
    """Whole and ragged tiles, stages of W's rows and blocks of its columns; every 37th row is compared, and the last."""
    _, codes, scale, _ = operands(1, N, K, dtype, M + N)
    g = torch.randn((M, N + 8), generator=torch.Generator().manual_seed(2)).to(dtype)
    some = sorted({*range(0, M, 37), M - 1})
    w, rows = values(codes, scale, K), g[some][:, 8:].double().numpy()
    x = torch.zeros(M, K, dtype=dtype).to(vk).requires_grad_()
    y = torch_vulkan.mxfp4_linear(x, codes.to(vk), scale.to(vk))
    for grad in (g.to(vk)[:, 8:], g[:, 8:].contiguous().to(vk)):  # rows further apart than they are long, and dense ones
        (dx,) = torch.autograd.grad(y, x, grad, retain_graph=True)
        check(dx.cpu()[some], rows @ w, np.abs(rows) @ np.abs(w), N, dtype)


@pytest.mark.gpu
def test_the_inputs_gradient_of_what_is_no_number():
    """A block of NaN reaches its 32 columns, an infinite gradient its row, nothing else."""
    M, N, K = 70, 72, 96
    _, codes, scale, _ = operands(1, N, K, torch.bfloat16, 4)
    g = torch.randn((M, N), generator=torch.Generator().manual_seed(3)).bfloat16()
    x = torch.zeros(M, K, dtype=torch.bfloat16).to(vk).requires_grad_()

    def back():
        return torch.autograd.grad(torch_vulkan.mxfp4_linear(x, codes.to(vk), scale.to(vk)), x, g.to(vk))[0].cpu()

    want = back()
    scale[5, 1], g[3, 70] = 255, float("nan")
    got = back()
    hit = torch.zeros(M, K, dtype=torch.bool)
    hit[:, 32:64], hit[3] = True, True
    assert torch.isnan(got[hit]).all() and torch.equal(got[~hit], want[~hit])


@pytest.mark.gpu
@pytest.mark.parametrize("M,quantize", [(1, False), (200, False), (1, True), (200, True)])
def test_replayed_graph(M, quantize):
    rt, out = abi.Runtime(), {}
    x, codes, scale, b = (t.to(vk) for t in operands(M, 512, 2048, torch.bfloat16, 8))

    def run():
        out["y"] = torch_vulkan.mxfp4_linear(x, codes, scale, b, quantize)

    run()
    want = out["y"].cpu()
    gid = rt.graph(run)
    for _ in range(3):
        out["y"].zero_()
        rt.graph_launch(gid)
        assert torch.equal(out["y"].cpu(), want)
        assert torch.equal(torch_vulkan.mxfp4_linear(x, codes, scale, b, quantize).cpu(), want)
    rt.graph_destroy(gid)


def test_argument_blocks_match_the_header(tmp_path):
    """abi.Mx4Args and abi.Mx4MmArgs lay their fields out as include/hrt_ops.h does."""
    import ctypes
    import os
    import subprocess

    blocks = {"hrt_mx4_args": abi.Mx4Args, "hrt_mx4_mm_args": abi.Mx4MmArgs}
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


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES[1:])
@pytest.mark.parametrize("quantize", [False, True])
@pytest.mark.parametrize("M,N,K", [(37, 136, 320), (3, 64, 96), (37, 130, 320), (5, 40, 50)])
def test_the_gradients_gradient(M, N, K, quantize, dtype):
    """dx = g W is linear in g, whichever product makes it: its gradient is h W^T, and that one's k W again."""
    x, codes, scale, b = operands(M, N, K, dtype, 23)
    r = torch.Generator().manual_seed(4)
    g, k = (torch.randn((M, N), generator=r).to(dtype) for _ in range(2))
    h, hb = torch.randn((M, K), generator=r).to(dtype), torch.randn((N,), generator=r).to(dtype)
    C, S, w = codes.to(vk), scale.to(vk), values(codes, scale, K)
    X, B, G, H = (t.to(vk).requires_grad_() for t in (x, b, g, h))
    f64 = lambda t: t.double().numpy()  # noqa: E731
    dx, db = torch.autograd.grad(torch_vulkan.mxfp4_linear(X, C, S, B, quantize), (X, B), G, create_graph=True)
    check(dx, f64(g) @ w, np.abs(f64(g)) @ np.abs(w), N, dtype)
    (gh,) = torch.autograd.grad(dx, G, H, create_graph=True)
    check(gh, f64(h) @ w.T, np.abs(f64(h)) @ np.abs(w).T, K, dtype)
    (gk,) = torch.autograd.grad(gh, H, k.to(vk))
    check(gk, f64(k) @ w, np.abs(f64(k)) @ np.abs(w), N, dtype)
    (gb,) = torch.autograd.grad(db, G, hb.to(vk))
    assert torch.equal(gb.cpu(), hb.expand(M, N))


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(37, 136, 320), (37, 130, 320), (5, 40, 50)])
def test_a_penalty_on_the_inputs_gradient(M, N, K):
    """d/dx of <(x W^T) W, h> is (h W^T) W: the calls that autograd makes are the ones that a program would make of them."""
    x, codes, scale, _ = operands(M, N, K, torch.bfloat16, 29)
    h = torch.randn((M, K), generator=torch.Generator().manual_seed(5)).bfloat16().to(vk)
    C, S, X = codes.to(vk), scale.to(vk), x.to(vk).requires_grad_()
    y = torch_vulkan.mxfp4_linear(X, C, S)
    (dx,) = torch.autograd.grad(y, X, y, create_graph=True)
    (got,) = torch.autograd.grad((dx * h).sum(), X, retain_graph=True)
    (want,) = torch.autograd.grad(y, X, torch_vulkan.mxfp4_linear(h, C, S))
    assert torch.equal(got.cpu(), want.cpu())


@pytest.mark.gpu
def test_forward_mode_is_refused():
    """A tangent is never dropped: neither without nor with a gradient wanted."""
    import torch.autograd.forward_ad as fwd

    x, codes, scale, b = (t.to(vk) for t in operands(4, 64, 96, torch.bfloat16, 1))
    with fwd.dual_level():
        for wants in (False, True):
            for quantize in (False, True):
                dual = fwd.make_dual(x.detach().requires_grad_(wants), torch.ones_like(x))
                with pytest.raises(RuntimeError, match="forward-mode"):
                    torch_vulkan.mxfp4_linear(dual, codes, scale, b, quantize)
                with pytest.raises(RuntimeError, match="forward-mode"):
                    torch_vulkan.mxfp4_linear(x, codes, scale, fwd.make_dual(b.detach().requires_grad_(wants), torch.ones_like(b)), quantize)
        y = torch_vulkan.mxfp4_linear(x.detach().requires_grad_(), codes, scale, b)  # nor that of an incoming gradient
        with pytest.raises(RuntimeError, match="forward-mode"):
            y.backward(fwd.make_dual(torch.ones_like(y), torch.ones_like(y)))
    assert torch_vulkan.mxfp4_linear(x, codes, scale, b).shape == (4, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("quantize", [False, True])
@pytest.mark.parametrize("shape,N", [((6, 96), 64), ((2, 3, 96), 64), ((96,), 64), ((6, 96), 50), ((2, 3, 50), 64), ((0, 96), 64)])
def test_in_place_operations_on_the_output(shape, N, quantize):
    """An adapter's output added to the layer's in place, in training and without gradients, as out of place."""
    K = shape[-1]
    x, codes, scale, b = operands(6, N, K, torch.bfloat16, 31)
    n = int(np.prod(shape))
    C, S, X = codes.to(vk), scale.to(vk), x.flatten()[:n].view(shape).to(vk).requires_grad_()
    B, A = b.to(vk).requires_grad_(), torch.randn((*shape[:-1], N), generator=torch.Generator().manual_seed(6)).bfloat16().to(vk).requires_grad_()

    def run(add, x, bias):
        y = add(torch_vulkan.mxfp4_linear(x, C, S, bias, quantize), A)
        y = add(y, y * 2)
        return [y, *torch.autograd.grad(y, [t for t in (x, bias, A) if t is not None and t.requires_grad], torch.ones_like(y))]

    for x_, bias in ((X, B), (X, None), (X.detach(), B), (X.detach(), None)):
        for a, w in zip(run(lambda y, z: y.add_(z), x_, bias), run(lambda y, z: y + z, x_, bias)):
            assert torch.equal(a.detach().cpu(), w.detach().cpu())
    y = torch_vulkan.mxfp4_linear(X, C, S, B, quantize)
    y.view(-1)[: y.numel() // 2].zero_()  # a view of it
    (dx,) = torch.autograd.grad(y, X, torch.ones_like(y))
    assert dx.shape == X.shape
