"""MI355X-native "vk" device for PyTorch: the torch_vulkan API over HIP and hand-written gfx950 kernels.

`import torch_vulkan` loads the C++ shim (which registers the PrivateUse1 operators: mm/bmm/addmm/
baddbmm, fused SDPA forward+backward, softmax (+backward, _safe_softmax), layer_norm (+backward), copies
and fills), renames PrivateUse1 to "vk" and installs the `torch.vk` module, so training code written for
the reference `torch_vulkan` package (torch_vulkan/__init__.py:1-270) runs unchanged: tensors move with
`.to("vk")`, every other op falls back to the CPU, and the counters below report which path ran.

The native libraries are built in-tree by `torch-vulkan_amd/build.py`; there is no pure-Python
substitute, so a missing build is an ImportError.
"""

import importlib
import os
import sys
import types

import torch

_THIS_DIR = os.path.dirname(os.path.abspath(__file__))


def _load_extension():
    if _THIS_DIR not in sys.path:
        sys.path.insert(0, _THIS_DIR)
    try:
        return importlib.import_module("torch_vulkan_C")
    except ImportError as e:  # no silent fallback: the device does not exist without its native code
        raise ImportError(
            f"torch_vulkan: the native extension is not built ({e}); run `python torch-vulkan_amd/build.py`"
        ) from e


_C = _load_extension()


def is_available() -> bool:
    return True


def device_count() -> int:
    return 1


def current_device() -> int:
    return 0


def set_device(device) -> None:
    return None


def synchronize(device=None) -> None:
    _C.synchronize()


def device_name() -> str:
    return _C.device_name()


def live_bytes() -> int:
    return _C.live_bytes()


def memory_info() -> dict:
    """Device memory in bytes: budget (what this process can still reach: free + own reservation), usage
    (all processes) and heap (device total)."""
    budget, usage, heap = _C.memory_info()
    return {"budget": budget, "usage": usage, "heap": heap}


def peak_live_bytes() -> int:
    """High-water mark of live device bytes since reset_peak_live_bytes()."""
    return _C.peak_live_bytes()


def reset_peak_live_bytes() -> None:
    _C.reset_peak_live_bytes()


def set_memory_limit(megabytes: int) -> None:
    """Cap the device memory reserved by this process (MiB, 0 = no cap); exceeding it raises an OOM
    RuntimeError.  Also settable with VKT_MEM_LIMIT_MB at import time."""
    _C.set_memory_limit(int(megabytes) << 20)


def set_fused_attention(mode: str) -> None:
    """Policy of the fused F.scaled_dot_product_attention: "auto" (default), "on" or "off".  auto uses it
    for bf16/f16 and, for f32, when the score matrix would be >= 256 MiB.  Env: VKT_FUSED_ATTN=0/1."""
    _C.set_fused_attention({"off": 0, "on": 1, "auto": 2}[mode])


def kernel_counts() -> dict:
    return dict(_C.kernel_counts())


def validation_errors() -> int:
    return _C.validation_errors()


def empty_cache() -> None:
    _C.empty_cache()


def reserved_bytes() -> int:
    return _C.reserved_bytes()


def live_blocks() -> int:
    return _C.live_blocks()


def slab_count() -> int:
    return _C.slab_count()


def workspaces_left_out() -> int:
    """How often an operator ran without a workspace that would have made it faster, for want of device memory; the
    last bits of its result then differ (another order of fp32 sums)."""
    return _C.workspaces_left_out()


def manual_seed(seed: int) -> None:
    # random numbers are drawn on the CPU and copied, as in the reference
    return None


def manual_seed_all(seed: int) -> None:
    return None


def seed() -> None:
    return None


def _is_in_bad_fork() -> bool:
    return False


def get_amp_supported_dtype():
    return [torch.bfloat16, torch.float16]


class device:  # noqa: N801  same name and use as torch.cuda.device
    def __init__(self, device=None):
        self.idx = device

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        return False


def get_rng_state(device="vk") -> torch.Tensor:
    return torch.zeros(1, dtype=torch.uint8)


def set_rng_state(new_state, device="vk") -> None:
    return None


# Names of the runtime counters (include/hrt.h, hrt_stat) as stats() reports them: (key, index, scale).
_RUNTIME_COUNTERS = (
    ("dispatch_s", 0, 1e-9), ("dispatch_n", 1, 1.0), ("transfer_s", 2, 1e-9), ("transfer_n", 3, 1.0),
    ("pipeline_create_s", 4, 1e-9), ("upload_MB", 5, 1.0 / 2**20), ("download_MB", 6, 1.0 / 2**20),
    ("gpu_wait_s", 7, 1e-9),
)


def stats() -> dict:
    """Host-side runtime counters: time spent queueing kernels and in transfers, their counts, kernel-table
    set-up time, bytes moved, time waiting for the GPU, and the time spent in CPU fallbacks."""
    raw = _C.runtime_counters()
    out = {key: raw[i] * scale for key, i, scale in _RUNTIME_COUNTERS}
    out["fallback_s"] = sum(fallback_time_by_op().values())
    return out


def fallback_time_by_op() -> dict:
    return dict(_C.fallback_time_by_op())


def profile() -> str:
    """Per-kernel GPU time ("name\tms\tcount" lines) when HRT_PROFILE=1 was set at start-up."""
    return _C.profile()


def _report_at_exit():
    """VKT_STATS=1 / HRT_PROFILE=1: a summary of where the time went, printed when the process ends."""
    lines = ["runtime " + " ".join(f"{k}={v:.3g}" for k, v in stats().items())]
    slow = sorted(fallback_time_by_op().items(), key=lambda kv: kv[1], reverse=True)
    if slow:
        lines.append("CPU fallbacks by time " + " ".join(f"{k}={v:.3g}s" for k, v in slow[:8]))
    busy = sorted(kernel_counts().items(), key=lambda kv: kv[1], reverse=True)
    lines.append("GPU operators by count " + " ".join(f"{k}={n}" for k, n in busy[:8]))
    prof = [row.split("\t") for row in profile().splitlines() if row]
    if prof:
        total = sum(float(r[1]) for r in prof) or 1.0
        lines.append(f"kernel time {total:.1f} ms")
        lines += [f"  {name:34s} {float(ms):9.1f} ms {100 * float(ms) / total:5.1f}%  x{n}" for name, ms, n in prof[:18]]
    print("\n".join("[torch_vulkan] " + l for l in lines))


if os.environ.get("VKT_STATS") or os.environ.get("HRT_PROFILE"):
    import atexit

    atexit.register(_report_at_exit)


def coop_caps() -> int:
    """Matrix-core kernels available (bit0 = f16, bit1 = bf16): 3 on gfx950."""
    return _C.coop_caps()


def set_coop_enabled(on: bool) -> None:
    """Switch the matrix-core (MFMA) kernels on/off; off routes bf16/f16 to the FMA kernels.
    Env: VKT_NO_COOP=1."""
    _C.set_coop_enabled(bool(on))


def empty_pinned(shape, dtype=torch.float32) -> torch.Tensor:
    """An uninitialised CPU tensor in pinned (page-locked) host memory of the vk runtime.  Copies between it
    and a dense vk tensor of the same dtype and shape with non_blocking=True are asynchronous: uploads run
    on the runtime's copy stream and overlap kernels that do not touch their destination (the kernels that
    do wait for them); downloads are valid after torch_vulkan.synchronize().  The block-swap path:
    frozen weights kept here and streamed into a ring of device buffers each step."""
    return _C.empty_pinned(list(shape), dtype)


def is_pinned(t: torch.Tensor) -> bool:
    """True if CPU tensor t lies in vk pinned host memory (what t.is_pinned(device="vk") answers, without
    PyTorch's deprecation warning for the device argument)."""
    return bool(_C.is_pinned(t))


def pin_memory(t: torch.Tensor) -> torch.Tensor:
    """A copy of CPU tensor t in vk pinned host memory (see empty_pinned); t itself if it already is."""
    if is_pinned(t):
        return t
    out = _C.empty_pinned(list(t.shape), t.dtype)
    out.copy_(t)
    return out


def dequant_int8(q, scale, out_dtype=torch.bfloat16):
    """Weight-only int8 dequant: out[r, c] = float(q[r, c]) * float(scale[r, c // 64]) rounded to out_dtype.

    q: int8 [rows, cols]; scale: bfloat16 [rows, ceil(cols / 64)] (64-column blocks per row).  On vk
    tensors this runs the dq8 kernel; CPU tensors get the same closed form in PyTorch, as the reference's
    function does (torch_vulkan/__init__.py:193-205).
    """
    if q.device.type == "vk":
        return _C.dequant_int8(q.contiguous(), scale.contiguous(), out_dtype)
    # each row padded to whole 64-element blocks, every block times its scale in float32, rounded once
    rows, cols = q.shape
    nb = scale.shape[1]
    blocks = torch.zeros((rows, nb * 64), dtype=torch.float32)
    blocks[:, :cols] = q.float()
    prod = blocks.view(rows, nb, 64) * scale.float().unsqueeze(-1)
    return prod.view(rows, nb * 64)[:, :cols].to(out_dtype)


def dequant_int8_linear(x, q, scale, bias=None):
    """Fused int8 weight-only linear: x @ dequant_int8(q, scale, x.dtype).T (+ bias), x bf16/f16 on vk.

    The dequantized weight never reaches memory; its values are bit-identical to dequant_int8's."""
    if x.device.type != "vk":
        raise RuntimeError("dequant_int8_linear: x must be a vk tensor")
    return _C.dequant_int8_linear(x, q.contiguous(), scale.contiguous(), bias)


_MXFP4_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)  # e2m1 codes 0..7; bit 3 is the sign


def quantize_mxfp4(x):
    """Pack x [..., cols] (float32, bfloat16 or float16) into microscaled 4-bit floating point: (codes, scale), uint8
    [..., ceil(cols / 2)] and [..., ceil(cols / 32)].

    Blocks of 32 consecutive values share a scale byte s, and a value reads back as e2m1 * 2**(s - 127) with e2m1 in
    0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign.  s = floor(log2(largest magnitude)) - 2 + 127, at least 0; each value is
    rounded to the nearest code, ties to the even one, and saturates at 6.  Two codes a byte, the even element in the low
    nibble.  A block with an infinity or NaN gets s = 255 and reads back as NaN.  Not differentiable.
    """
    if x.device.type == "vk":
        return _C.quantize_mxfp4(x)
    if x.dtype not in (torch.float32, torch.bfloat16, torch.float16) or x.dim() < 1:
        raise RuntimeError("quantize_mxfp4: x must be a float32, bfloat16 or float16 tensor of at least one dimension")
    cols = x.shape[-1]
    nb = (cols + 31) // 32
    v = torch.zeros((*x.shape[:-1], nb * 32), dtype=torch.float64)  # exact: quotients by powers of two
    v[..., :cols] = x.detach()
    v = v.view(*x.shape[:-1], nb, 32)
    bits = v.float().abs().view(torch.int32).amax(-1) >> 23  # biased exponents; 255 for infinities and NaN
    scale = torch.where(bits == 255, 255, (bits - 2).clamp(min=0))
    m = v * torch.exp2(127.0 - scale.double()).unsqueeze(-1)
    m = torch.where(scale.unsqueeze(-1) == 255, torch.zeros_like(m), m)
    a = m.abs()
    code = sum(((a > t) if i % 2 == 0 else (a >= t)).to(torch.uint8) for i, t in enumerate((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)))
    code = (code + 8 * torch.signbit(m).to(torch.uint8)).flatten(-2)
    packed = (code[..., 0::2] | (code[..., 1::2] << 4))[..., : (cols + 1) // 2]
    return packed.contiguous(), scale.to(torch.uint8)


def dequant_mxfp4(codes, scale, out_dtype=torch.bfloat16, cols=None):
    """The values that quantize_mxfp4's (codes, scale) stand for, [..., cols] in out_dtype (rounded once: exact in float32
    and bfloat16 up to overflow).  cols: the rows' length, by default twice the bytes of codes (name it where it is odd)."""
    cols = 2 * codes.shape[-1] if cols is None else int(cols)
    if codes.device.type == "vk":
        return _C.dequant_mxfp4(codes, scale, out_dtype, cols)
    if codes.dtype != torch.uint8 or scale.dtype != torch.uint8 or codes.shape[:-1] != scale.shape[:-1] or (
            codes.shape[-1], scale.shape[-1]) != ((cols + 1) // 2, (cols + 31) // 32):
        raise RuntimeError(f"dequant_mxfp4: codes and scale of rows of {cols} values must be uint8 [..., {(cols + 1) // 2}] and "
                           f"[..., {(cols + 31) // 32}], got {tuple(codes.shape)} and {tuple(scale.shape)}")
    code = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)[..., :cols].long()
    v = torch.tensor(_MXFP4_VALUES, dtype=torch.float64)[code & 7] * torch.where(code >= 8, -1.0, 1.0)
    s = torch.where(scale == 255, float("nan"), torch.exp2(scale.double() - 127.0))
    return (v * s.repeat_interleave(32, -1)[..., :cols]).to(out_dtype)


def mxfp4_linear(x, codes, scale, bias=None, quantize_input=False):
    """Linear layer on frozen 4-bit weights: x @ dequant_mxfp4(codes, scale, x.dtype).T (+ bias), x [..., K] bf16/f16 on vk,
    codes [N, ceil(K / 2)], scale [N, ceil(K / 32)].  The dequantized weights never reach memory where K % 32 == 0
    (and N % 8 == 0, for the gradient).

    quantize_input=True rounds x the same way first (quantize_mxfp4 of its rows) and multiplies 4-bit operands, which the
    matrix cores do at four times the 16-bit rate.  Differentiable in x and bias, any number of times (create_graph), in
    reverse mode; the gradient of a quantized x goes straight through (grad @ W, as if x had gone in unrounded).  Autocast casts x
    and bias, as it does for linear."""
    if x.device.type != "vk":
        raise RuntimeError("mxfp4_linear: x must be a vk tensor")
    return _C.mxfp4_linear(x, codes, scale, bias, bool(quantize_input))


def relative_bias_attention(q, k, v, table, key_mask=None, causal=False, scale=None, max_distance=128, query_offset=0):
    """Fused attention with a learned relative position bias: softmax(scale * q @ k.T + table[bucket(j - i - query_offset)]) @ v.

    q [B, H, Sq, D], k, v [B, H, Sk, D] on vk (float32, bfloat16 or float16, D <= 128, any strides), table [buckets, H] of the
    same dtype: one learned bias per bucket and head.  i and j count queries and keys; query_offset is the position of query
    0 among the keys (new tokens after a cache of n: n).  scale defaults to 1 / sqrt(D).

    Buckets of the distance r = j - i - query_offset: with causal=False half of them serve r <= 0 and half r > 0, with causal=True
    (which also hides keys j > i + query_offset) all serve r <= 0.  Of a direction's nb buckets the first nb // 2 hold one
    distance each, the others grow logarithmically up to max_distance, and the last one holds everything beyond.

    key_mask: bool [B, Sk] (or [1, Sk]), True where a key may be seen.  Masked keys and values play no part, whatever they hold,
    nor do those that causal hides from every query (the unwritten end of a cache).  A table entry of -inf, or of bfloat16's or
    float32's lowest value, hides its pairs (finite entries beyond 2e38 * min(1, scale) overflow).  A query without a key to
    see gets zeros and no gradient; one before the first key, by causal, gives none either, whatever it holds.

    Returns [B, H, Sq, D] in token-major memory; differentiable once, in reverse mode, in q, k, v and table.  The backward pass
    reads the output: one changed in place may be refused there.  Autocast casts q, k, v and table, as it does for
    scaled_dot_product_attention.  Nothing of size Sq x Sk is stored."""
    if q.device.type != "vk":
        raise RuntimeError("relative_bias_attention: q must be a vk tensor")
    return _C.relative_bias_attention(q, k, v, table, key_mask, bool(causal), scale, int(max_distance), int(query_offset))


def event_record(slot: int) -> None:
    """Record HIP event `slot` (0..1023) on the runtime's stream (the stream every vk kernel runs on)."""
    _C.event_record(int(slot))


def event_elapsed_ms(start_slot: int, end_slot: int) -> float:
    """Milliseconds between two recorded slots (waits for the later one)."""
    return _C.event_elapsed_ms(int(start_slot), int(end_slot))


def fallback_counts() -> dict:
    return dict(_C.fallback_counts())


def reset_fallback_counts() -> None:
    _C.reset_counts()


def set_inline_backward(on: bool = True) -> None:
    """Run autograd's backward on the calling thread (PyTorch's thread-local
    torch.autograd.set_multithreading_enabled(False)), for the thread that calls this.  PyTorch otherwise
    hands the work of every non-CPU device to a per-device worker thread and waits for it; the vk device
    has one stream, so that thread adds only a cross-thread handoff: on MI355X a backward() call costs
    ~49 us of host time on vk that way against ~24 us inline, which left the GPU idle in short steps.
    Gradients are the same either way.  Opt-in, because it changes the calling thread's autograd state
    (and CUDA or other devices' backward on that thread would run inline too): call it on the thread that
    runs the training loop, or set VKT_INLINE_BACKWARD=1 to apply it to the importing thread at import."""
    torch._C._set_multithreading_enabled(not on)


def _register():
    # Keep nn.Parameter identity when modules move to vk (optimizers built before .to() keep working).
    torch.__future__.set_swap_module_params_on_conversion(True)
    # "vulkan" is taken by PyTorch's own inference backend, hence "vk".
    torch.utils.rename_privateuse1_backend("vk")
    module = types.ModuleType("torch.vk")
    for name in (
        "is_available",
        "device_count",
        "current_device",
        "set_device",
        "synchronize",
        "empty_cache",
        "manual_seed",
        "manual_seed_all",
        "seed",
        "_is_in_bad_fork",
        "get_amp_supported_dtype",
        "device",
        "get_rng_state",
        "set_rng_state",
        "memory_info",
        "set_memory_limit",
        "peak_live_bytes",
        "reset_peak_live_bytes",
        "empty_pinned",
        "pin_memory",
        "is_pinned",
    ):
        setattr(module, name, globals()[name])
    torch._register_device_module("vk", module)


_register()
if os.environ.get("VKT_INLINE_BACKWARD") == "1":
    set_inline_backward(True)


def set_coop_range(lo: int = 0, hi: int = 2**64 - 1, kind: int = 0) -> None:
    """Debug: only matrix-core-eligible GEMM calls numbered [lo, hi) use MFMA (others the FMA kernel);
    kind 0 = all, 1 = bmm only, 2 = mm only.  For bisecting a bad call."""
    _C.set_coop_range(int(lo), int(hi), int(kind))


def reset_coop_calls() -> None:
    _C.reset_coop_calls()


def coop_calls() -> int:
    return _C.coop_calls()


if os.environ.get("VKT_MEM_LIMIT_MB"):
    set_memory_limit(int(os.environ["VKT_MEM_LIMIT_MB"]))
