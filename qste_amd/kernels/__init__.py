"""The operator layer: QSTE's ``qste.kernels`` API on gfx950 HIP kernels.

Same names, arguments, return values and error behaviour as the reference's
dispatch layer (``src/qste/kernels/loader.py:247-368``), for tensors on a
ROCm device.  Every call goes to ``libqste_hip.so`` through its C ABI
(``include/qste_hip.h``) on torch's current stream.  There is no CPU or
pure-torch path: a tensor that is not on the GPU, or a missing library, is an
error (``RuntimeError``), never a silent fallback.

Outputs are allocated through torch's caching allocator, as are the
workspaces the C entry points ask for; the library itself never allocates.
"""

from __future__ import annotations

import contextlib
import ctypes
from typing import NamedTuple

import torch
from torch import Tensor

from . import _lib
from ._lib import KernelError

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}

__all__ = [
    "KernelError",
    "apply_bits",
    "masked_activation",
    "masked_backward",
    "pack_bits",
    "smooth_activation",
    "smooth_backward",
    "unpack_bits",
    "Blocks8",
    "coordinate_update",
    "cuda_available",
    "dequantize_blocks",
    "distill_backward",
    "distill_forward",
    "embedding_backward",
    "packed_embedding",
    "evidence_from_packed",
    "gated_backward",
    "gated_forward",
    "linear_backward",
    "native_available",
    "pack_affine_rows",
    "pack_coordinate",
    "packed_linear_affine",
    "packed_row_inner",
    "packed_transpose",
    "quantize_blocks",
    "status",
    "swiglu_backward",
    "swiglu_backward_blocks",
    "swiglu_forward",
    "swiglu_forward_blocks",
    "token_logprobs_backward",
    "token_logprobs_forward",
    "unpack_rows",
]


# ---------------------------------------------------------------------------
# plumbing
# ---------------------------------------------------------------------------


def _require_gpu(*tensors: Tensor) -> torch.device:
    device = None
    for t in tensors:
        if t is None:
            continue
        own = t.device  # asked for once: a new object each time, a quarter of a microsecond
        if own == device:
            continue
        if own.type != "cuda":
            raise RuntimeError(
                f"qste_amd kernels run on the GPU only; got a tensor on {own} "
                "(move the model to the ROCm device first)"
            )
        if device is not None:
            raise RuntimeError(f"tensors on different devices: {device} and {own}")
        device = own
    if device is None:
        raise RuntimeError("no tensor argument to place the kernel on")
    return device


_RAW_STREAM = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(device: torch.device) -> int:
    """The device's current HIP stream as an address (torch's current-stream
    query without building a Stream object where torch offers it)."""

    if _RAW_STREAM is not None and device.index is not None:
        return _RAW_STREAM(device.index)
    return torch.cuda.current_stream(device).cuda_stream


def _dtype_code(t: Tensor) -> int:
    try:
        return _DTYPES[t.dtype]
    except KeyError:
        raise TypeError(f"unsupported dtype {t.dtype}; expected float32, float16 or bfloat16") from None


def _ptr(t: Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _packed_width(columns: int) -> int:
    return (int(columns) + 7) // 8


def _check_packed(packed: Tensor, columns: int, rows: int | None = None) -> Tensor:
    shape = packed.shape
    if packed.dtype != torch.uint8 or len(shape) != 2:
        raise ValueError("packed signs must be a rank-2 uint8 tensor")
    if shape[1] != _packed_width(columns):
        raise ValueError(
            f"packed sign width {shape[1]} does not match {columns} columns "
            f"(expected {_packed_width(columns)})"
        )
    if rows is not None and shape[0] != rows:
        raise ValueError(f"packed signs have {shape[0]} rows, expected {rows}")
    return packed.contiguous()


def _f32(t: Tensor | None) -> Tensor | None:
    """``t`` as contiguous fp32 (a new tensor unless it already is one).

    Bind the result to a name that lives until the C call returns: a
    temporary passed straight to ``_ptr`` is freed before the launch, and the
    caching allocator hands its block to the next allocation."""

    if t is None:
        return None
    return t.detach().to(torch.float32).contiguous()


def _aligned(t: Tensor) -> Tensor:
    """Contiguous, with the 16-byte start the vector paths need."""

    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _rows2d(t: Tensor, what: str) -> Tensor:
    if t.dim() != 2:
        raise ValueError(f"{what} expects a rank-2 tensor")
    return _aligned(t)


def _workspace(nbytes: int, device: torch.device) -> Tensor:
    return torch.empty(max(int(nbytes), 1), dtype=torch.uint8, device=device)


def native_available() -> bool:
    """Whether the HIP library loads (it does not need a GPU to load)."""

    try:
        _lib.load()
        return True
    except KernelError:
        return False


def cuda_available() -> bool:
    return torch.cuda.is_available() and native_available()


def status() -> dict:
    """Whether the HIP library is built and loadable, and why not if not."""

    ok = native_available()
    return {
        "native": ok,
        "library": str(_lib.LIB_PATH),
        "version": _lib.load().qste_version() if ok else None,
        "failure": _lib.failure(),
        "gpu": torch.cuda.is_available(),
    }


def stream_read(src: Tensor, groups: int | None = None) -> None:
    """A plain streaming read of ``src``'s bytes (measurement probe, no
    counterpart in the reference): the floor for any kernel reading them once."""

    device = _require_gpu(src)
    if not src.is_contiguous() or src.numel() * src.element_size() % 16:
        raise ValueError("stream_read needs a contiguous tensor of a multiple of 16 bytes")
    props = torch.cuda.get_device_properties(device)
    groups = int(groups or 4 * props.multi_processor_count)
    sink = torch.empty(groups * 256, dtype=torch.int32, device=device)
    lib = _lib.load()
    _lib.check(lib.qste_stream_read(_ptr(src), src.numel() * src.element_size(), _ptr(sink), groups,
                                    _stream(device)), "stream_read")


def capture_id(t: Tensor) -> int:
    """The number of the graph capture that ``t``'s device records into now, 0 for none (or a tensor on no GPU)."""

    if not t.is_cuda or not torch.cuda.is_current_stream_capturing():
        return 0
    return _lib.load().qste_capture_id(_stream(t.device))


def device_info(device=None) -> dict:
    """What the runtime reports for ``device``: compute units, maximum shader
    clock and memory clock (MHz), LDS bytes per compute unit."""

    device = torch.device(device or "cuda")
    out = (ctypes.c_int64 * 4)()
    with torch.cuda.device(device):
        _lib.check(_lib.load().qste_device_info(ctypes.cast(out, ctypes.c_void_p)), "device_info")
    return {"cus": int(out[0]), "max_sclk_mhz": out[1] / 1000.0, "mclk_mhz": out[2] / 1000.0,
            "lds_per_cu": int(out[3])}


def measured_sclk_mhz(device=None, spins: int = 1 << 18) -> float:
    """Shader clock one wave sees right now, in MHz: s_memtime cycles over
    s_memrealtime (100 MHz) ticks across a dependent integer loop."""

    device = torch.device(device or "cuda")
    out = torch.zeros(3, dtype=torch.int64, device=device)
    lib = _lib.load()
    _lib.check(lib.qste_clock_probe(_ptr(out), int(spins), _stream(device)), "clock_probe")
    cycles, ticks, _ = (int(v) for v in out.cpu().tolist())
    return cycles / ticks * 100.0 if ticks > 0 else float("nan")


def profile(device=None) -> str:
    """One line: what this build runs on ``device`` (reference
    ``kernels.profile(device).describe()``, src/qste/kernels/device.py:85-91).

    Nothing is autotuned: the kernels are written for gfx950 and take their
    grid sizes from the compute-unit count the runtime reports.  The line
    names the device and architecture, that count, the shader clock (the
    maximum the runtime reports and the one a wave measures now), HBM and LDS
    sizes, the library version, and which kernel each operator takes."""

    device = torch.device(device) if device is not None else torch.device(
        "cuda" if torch.cuda.is_available() else "cpu")
    version = _lib.load().qste_version() if native_available() else None
    if device.type != "cuda":
        return (f"{device} [no QSTE kernels: qste_amd runs on gfx950 GPUs only]  "
                f"library={'libqste_hip v%d' % version if version is not None else 'not built'}")
    props = torch.cuda.get_device_properties(device)
    arch = getattr(props, "gcnArchName", "?").split(":")[0]
    info = device_info(device)
    now_mhz = measured_sclk_mhz(device)
    return (f"{props.name} [{arch}]  cus={info['cus']}  "
            f"sclk={info['max_sclk_mhz']:.0f}MHz max / {now_mhz:.0f}MHz measured  "
            f"hbm={props.total_memory / 2**30:.0f}GiB  lds={info['lds_per_cu'] / 1024:.0f}KiB/CU  "
            f"library=libqste_hip v{version}  "
            "(products: bf16/fp16 MFMA 256x256 tiles, fp32 as three bf16 limbs; up to 64 rows (21 in fp32): weight "
            "bits as sparse-MFMA indexes; coordinate step: one launch for columns % 2048 == 0, else five or six)")


# ---------------------------------------------------------------------------
# operators (reference: src/qste/kernels/loader.py:247-368)
# ---------------------------------------------------------------------------


def pack_coordinate(coordinate: Tensor) -> Tensor:
    """Sign bits of an int8 coordinate matrix, LSB first (fallback.py:91-92)."""

    device = _require_gpu(coordinate)
    if coordinate.dtype != torch.int8 or coordinate.dim() != 2:
        raise ValueError("pack_coordinate expects a rank-2 int8 tensor")
    coordinate = coordinate.contiguous()
    rows, cols = coordinate.shape
    packed = torch.empty(rows, _packed_width(cols), dtype=torch.uint8, device=device)
    code = _lib.load().qste_pack_coordinate(
        _ptr(coordinate), _ptr(packed), rows, cols, _stream(device))
    _lib.check(code, "pack_coordinate")
    return packed


def unpack_rows(packed: Tensor, columns: int, *, dtype: torch.dtype | None = None,
                row_scale: Tensor | None = None) -> Tensor:
    """+-1 matrix of the packed signs (fallback.py:27-29)."""

    dtype = dtype or torch.float32
    device = _require_gpu(packed, row_scale)
    packed = _check_packed(packed, columns)
    out = torch.empty(packed.shape[0], int(columns), dtype=dtype, device=device)
    row_scale_f32 = _f32(row_scale)  # held until the launch is queued
    code = _lib.load().qste_unpack_rows(
        _ptr(packed), _ptr(row_scale_f32), _ptr(out), _dtype_code(out), packed.shape[0],
        int(columns), _stream(device))
    _lib.check(code, "unpack_rows")
    return out


def pack_affine_rows(values: Tensor) -> tuple[Tensor, Tensor, Tensor]:
    """(bits, offset, scale) of each row: x ~ offset + scale * sign(x - offset).

    fallback.py:77-88. Arithmetic in fp32 on the dtype's values.  offset and
    scale are rows 0 and 1 of one fp32 [2, rows] tensor (``stacked_pair``).
    """

    device = _require_gpu(values)
    if values.dim() != 2:
        raise ValueError("pack_affine_rows expects a rank-2 tensor")
    values = values.contiguous()
    rows, cols = values.shape
    if cols == 0:
        raise ValueError("pack_affine_rows needs at least one column")
    packed = torch.empty(rows, _packed_width(cols), dtype=torch.uint8, device=device)
    # rows 0 and 1 of one [2, rows] tensor: the layout a saved encoding keeps
    offset, scale = torch.empty(2, rows, dtype=torch.float32, device=device).unbind(0)
    code = _lib.load().qste_pack_affine_rows(
        _ptr(values), _dtype_code(values), _ptr(packed), _ptr(offset), _ptr(scale), rows, cols,
        _stream(device))
    _lib.check(code, "pack_affine_rows")
    return packed, offset, scale


def stacked_pair(offset: Tensor, scale: Tensor) -> Tensor:
    """``torch.stack((offset, scale))``, without a copy when the two are rows
    0 and 1 of one [2, n] tensor (as ``pack_affine_rows`` returns them)."""

    base = offset._base
    n = offset.numel()
    if (base is not None and scale._base is base and base.dim() == 2 and base.shape[0] == 2
            and base.shape[1] == n and base.is_contiguous() and offset.dtype == scale.dtype == base.dtype
            and offset.data_ptr() == base.data_ptr()
            and scale.data_ptr() == base.data_ptr() + n * base.element_size()):
        return base
    return torch.stack((offset, scale))


def packed_linear_affine(inputs: Tensor, packed: Tensor, scale: Tensor, bias: Tensor | None,
                         columns: int) -> Tensor:
    """``(x @ sign^T) * scale + bias`` in the input dtype (fallback.py:95-108)."""

    device = _require_gpu(inputs, packed, scale, bias)
    if inputs.shape[-1] != columns:
        raise ValueError(f"activation width {inputs.shape[-1]} does not match {columns} columns")
    packed = _check_packed(packed, columns)
    rows = packed.shape[0]
    if scale.numel() != rows:
        raise ValueError("scale must have one entry per output row")
    if bias is not None and bias.numel() != rows:
        raise ValueError("bias must have one entry per output row")
    flat = inputs.reshape(-1, columns).contiguous()
    out = torch.empty(flat.shape[0], rows, dtype=inputs.dtype, device=device)
    scale_f32 = _f32(scale)  # held until the launch is queued
    bias_f32 = _f32(bias)  # held until the launch is queued
    lib = _lib.load()
    # fp32 runs its product through bf16 limbs on the MFMA path, in a
    # workspace; products with few output tiles split K there
    nbytes = lib.qste_packed_linear_affine_workspace_bytes(flat.shape[0], rows, int(columns), _dtype_code(flat))
    if nbytes:
        work = _workspace(nbytes, device)
        code = lib.qste_packed_linear_affine_ws(
            _ptr(flat), _dtype_code(flat), _ptr(packed), _ptr(scale_f32), _ptr(bias_f32),
            _ptr(out), flat.shape[0], rows, int(columns), _ptr(work), work.numel(), _stream(device))
    else:
        code = lib.qste_packed_linear_affine(
            _ptr(flat), _dtype_code(flat), _ptr(packed), _ptr(scale_f32), _ptr(bias_f32),
            _ptr(out), flat.shape[0], rows, int(columns), _stream(device))
    _lib.check(code, "packed_linear_affine")
    return out.view(*inputs.shape[:-1], rows)


def packed_transpose(inputs: Tensor, packed: Tensor, columns: int,
                     row_scale: Tensor | None = None) -> Tensor:
    """``inputs @ (row_scale * sign)`` in the input dtype (fallback.py:111-123)."""

    device = _require_gpu(inputs, packed, row_scale)
    packed = _check_packed(packed, columns)
    rows = packed.shape[0]
    if inputs.shape[-1] != rows:
        raise ValueError(f"transpose width {inputs.shape[-1]} does not match {rows} rows")
    if row_scale is not None and row_scale.numel() != rows:
        raise ValueError("transpose row scale must have one entry per packed row")
    flat = inputs.reshape(-1, rows).contiguous()
    out = torch.empty(flat.shape[0], int(columns), dtype=inputs.dtype, device=device)
    row_scale_f32 = _f32(row_scale)  # held until the launch is queued
    lib = _lib.load()
    nbytes = (lib.qste_packed_transpose_workspace_bytes(flat.shape[0], rows, int(columns), _dtype_code(flat))
              if row_scale_f32 is not None else 0)
    if nbytes:
        work = _workspace(nbytes, device)
        code = lib.qste_packed_transpose_ws(
            _ptr(flat), _dtype_code(flat), _ptr(packed), _ptr(row_scale_f32), _ptr(out),
            flat.shape[0], rows, int(columns), _ptr(work), work.numel(), _stream(device))
    else:
        code = lib.qste_packed_transpose(
            _ptr(flat), _dtype_code(flat), _ptr(packed), _ptr(row_scale_f32), _ptr(out),
            flat.shape[0], rows, int(columns), _stream(device))
    _lib.check(code, "packed_transpose")
    return out.view(*inputs.shape[:-1], int(columns))


def evidence_from_packed(grad: Tensor, packed: Tensor, columns: int,
                         row_scale: Tensor | None = None) -> Tensor:
    """``grad^T @ (row_scale * sign(x))`` as fp32 [rows, columns] (fallback.py:126-138)."""

    device = _require_gpu(grad, packed, row_scale)
    if grad.dim() != 2:
        raise ValueError("evidence grad must be a rank-2 tensor")
    packed = _check_packed(packed, columns)
    samples, rows = grad.shape
    if packed.shape[0] != samples:
        raise ValueError("evidence grad and packed activations disagree on sample count")
    if row_scale is not None and row_scale.numel() != samples:
        raise ValueError("evidence row scale must have one entry per sample")
    grad = grad.contiguous()
    out = torch.empty(rows, int(columns), dtype=torch.float32, device=device)
    row_scale_f32 = _f32(row_scale)  # held until the launch is queued
    lib = _lib.load()
    nbytes = lib.qste_evidence_from_packed_workspace_bytes_dtype(samples, rows, int(columns), _dtype_code(grad))
    work = _workspace(nbytes, device) if nbytes else None
    code = lib.qste_evidence_from_packed(
        _ptr(grad), _dtype_code(grad), _ptr(packed), _ptr(row_scale_f32), _ptr(out), samples,
        rows, int(columns), _ptr(work), 0 if work is None else work.numel(), _stream(device))
    _lib.check(code, "evidence_from_packed")
    return out


def packed_row_inner(matrix: Tensor, packed: Tensor, columns: int) -> Tensor:
    """``sum_c matrix[r, c] * sign[r, c]`` (fallback.py:141-148)."""

    device = _require_gpu(matrix, packed)
    if matrix.dim() != 2 or matrix.shape[1] != columns:
        raise ValueError("row inner shape mismatch")
    packed = _check_packed(packed, columns, matrix.shape[0])
    m = matrix.detach().to(torch.float32).contiguous()
    out = torch.empty(m.shape[0], dtype=torch.float32, device=device)
    code = _lib.load().qste_packed_row_inner(
        _ptr(m), _ptr(packed), _ptr(out), m.shape[0], int(columns), _stream(device))
    _lib.check(code, "packed_row_inner")
    return out.to(matrix.dtype)


def linear_backward(grad: Tensor, packed_x: Tensor, x_offset: Tensor, x_scale: Tensor,
                    packed_w: Tensor, scale: Tensor, columns: int, *, need_bias: bool,
                    need_input: bool = True, offset_dot: Tensor | None = None):
    """All of ``QSTELinearFn.backward``'s products in one call (functional.py:173-194).

    Returns ``(grad_input [samples, columns] in grad's dtype or None,
    evidence fp32 [rows, columns] already multiplied by the row scale,
    grad_scale fp32 [rows], grad_bias fp32 [rows] or None)``.  With
    ``need_input=False`` the input-gradient product is not computed (autograd
    asks for no gradient of the layer's input) and grad_input is None.
    ``offset_dot`` (fp32 [rows], ``sum_t grad[t, r] * x_offset[t]`` summed as
    this call sums it, e.g. by ``swiglu_backward_sums``) spares the call that
    pass over ``grad``; it is ignored when a bias gradient is formed.
    """

    device = _require_gpu(grad, packed_x, x_offset, x_scale, packed_w, scale)
    grad = grad.contiguous()
    samples, rows = grad.shape
    packed_w = _check_packed(packed_w, columns, rows)
    packed_x = _check_packed(packed_x, columns, samples)
    lib = _lib.load()
    dx = torch.empty(samples, int(columns), dtype=grad.dtype, device=device) if need_input else None
    evidence = torch.empty(rows, int(columns), dtype=torch.float32, device=device)
    grad_scale = torch.empty(rows, dtype=torch.float32, device=device)
    grad_bias = torch.empty(rows, dtype=torch.float32, device=device) if need_bias else None
    nbytes = lib.qste_linear_backward_workspace_bytes_dtype(samples, rows, int(columns), _dtype_code(grad))
    work = _workspace(nbytes, device)
    x_offset_f32 = _f32(x_offset)  # held until the launch is queued
    x_scale_f32 = _f32(x_scale)  # held until the launch is queued
    scale_f32 = _f32(scale)  # held until the launch is queued
    if offset_dot is not None:
        if offset_dot.dtype != torch.float32 or offset_dot.numel() != rows or offset_dot.device != device:
            raise ValueError("offset_dot must be fp32 [rows] on the layer's device")
        offset_dot = offset_dot.contiguous()
        code = lib.qste_linear_backward_offset_dot(
            _ptr(grad), _dtype_code(grad), _ptr(packed_x), _ptr(x_offset_f32), _ptr(x_scale_f32),
            _ptr(packed_w), _ptr(scale_f32), _ptr(dx), _ptr(evidence), _ptr(grad_scale),
            _ptr(grad_bias), _ptr(offset_dot), samples, rows, int(columns), _ptr(work), work.numel(),
            _stream(device))
    else:
        code = lib.qste_linear_backward(
            _ptr(grad), _dtype_code(grad), _ptr(packed_x), _ptr(x_offset_f32), _ptr(x_scale_f32),
            _ptr(packed_w), _ptr(scale_f32), _ptr(dx), _ptr(evidence), _ptr(grad_scale),
            _ptr(grad_bias), samples, rows, int(columns), _ptr(work), work.numel(), _stream(device))
    _lib.check(code, "linear_backward")
    return dx, evidence, grad_scale, grad_bias


def coordinate_update(
    gradient: Tensor,
    coordinate: Tensor,
    packed: Tensor,
    moment_q: Tensor,
    moment_scale: Tensor,
    row_v: Tensor,
    col_v: Tensor,
    *,
    beta1: float,
    beta2: float,
    update_clip: float,
    coordinate_lr: float,
    block_size: int,
    seed: int,
    step,
    flips: Tensor | None = None,
    update_enabled: Tensor | None = None,
):
    """One fused coordinate step (fallback.py:158-242; GPU signature cuda.py:1705-1729).

    Returns the flip count as an int, or -- when ``flips`` (a device int64
    tensor) is given -- writes it there without a host synchronization and
    returns that tensor. ``step`` may be a device int64 scalar (read at run
    time, for graph replay). ``update_enabled`` (device uint8) gates every
    state write. ``gradient`` is read, not modified.
    """

    device = _require_gpu(gradient, coordinate, packed, moment_q, moment_scale, row_v, col_v)
    if int(block_size) <= 0:
        raise ValueError("momentum block size must be positive")
    gradient = gradient.detach().to(torch.float32).contiguous()
    rows, cols = gradient.shape
    for name, t, dt in (("coordinate", coordinate, torch.int8), ("packed", packed, torch.uint8),
                        ("moment_q", moment_q, torch.int8), ("moment_scale", moment_scale, torch.float16),
                        ("row_v", row_v, torch.float16), ("col_v", col_v, torch.float16)):
        if t.dtype != dt:
            raise ValueError(f"{name} must be {dt}, got {t.dtype}")
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous (it is updated in place)")
    if coordinate.shape != gradient.shape or moment_q.shape != gradient.shape:
        raise ValueError("coordinate state shape mismatch")
    if packed.shape != (rows, _packed_width(cols)):
        raise ValueError("packed sign shape mismatch")
    blocks = (rows * cols + block_size - 1) // block_size
    if moment_scale.numel() != blocks:
        raise ValueError("momentum scale shape mismatch")
    if row_v.numel() != rows or col_v.numel() != cols:
        raise ValueError("factored statistics shape mismatch")

    step_device = None
    step_value = 0
    if torch.is_tensor(step):
        if step.device != device or step.dtype != torch.int64:
            raise ValueError("a tensor step must be an int64 scalar on the surface's device")
        step_device = step
    else:
        step_value = int(step)
    enabled = None
    if update_enabled is not None:
        enabled = update_enabled.to(device=device, dtype=torch.uint8).contiguous()
    out = flips
    if out is None or out.dtype != torch.int64 or out.device != device:
        out_dev = torch.empty((), dtype=torch.int64, device=device)
    else:
        out_dev = out

    lib = _lib.load()
    nbytes = lib.qste_coordinate_update_workspace_bytes(rows, cols, int(block_size))
    work = _workspace(nbytes, device)
    wrap = lambda v: ((int(v) + (1 << 63)) % (1 << 64)) - (1 << 63)  # noqa: E731
    code = lib.qste_coordinate_update(
        _ptr(gradient), _ptr(coordinate), _ptr(packed), _ptr(moment_q), _ptr(moment_scale),
        _ptr(row_v), _ptr(col_v), rows, cols, float(beta1), float(beta2), float(update_clip),
        float(coordinate_lr), int(block_size), wrap(seed), wrap(step_value), _ptr(step_device),
        _ptr(out_dev), _ptr(enabled), _ptr(work), work.numel(), _stream(device))
    _lib.check(code, "coordinate_update")
    if flips is None:
        return int(out_dev.item())
    if out_dev is not flips:
        flips.copy_(out_dev)
    return flips


# ---------------------------------------------------------------------------
# packed activations (reference: loader.py:256-273, src/qste/nn.py)
# ---------------------------------------------------------------------------

# kinds of masked_activation / smooth_activation (include/qste_hip.h)
MASK_CLAMP, MASK_LEAKY, MASK_INTERVAL = 0, 1, 2
SMOOTH_KINDS = {
    "gelu": 0, "gelu_tanh": 1, "silu": 2, "tanh": 3, "sigmoid": 4, "elu": 5, "celu": 6,
    "selu": 7, "softplus": 8, "mish": 9, "hardswish": 10, "relu_square": 11, "provided": 12,
}


def pack_bits(mask: Tensor) -> Tensor:
    """One bit per element of a rank-2 mask, LSB first (fallback.py:32-47)."""

    device = _require_gpu(mask)
    if mask.dim() != 2:
        raise ValueError("packing expects a rank-2 tensor")
    if mask.dtype == torch.bool:
        mask = mask.contiguous().view(torch.uint8)
    elif mask.dtype != torch.uint8:
        mask = (mask != 0).view(torch.uint8)
    mask = _aligned(mask)
    rows, cols = mask.shape
    packed = torch.empty(rows, _packed_width(cols), dtype=torch.uint8, device=device)
    code = _lib.load().qste_pack_bits(_ptr(mask), _ptr(packed), rows, cols, _stream(device))
    _lib.check(code, "pack_bits")
    return packed


def unpack_bits(packed: Tensor, columns: int, *, dtype: torch.dtype | None = None) -> Tensor:
    """0/1 matrix of packed bits, pad columns dropped (fallback.py:50-54)."""

    dtype = dtype or torch.float32
    device = _require_gpu(packed)
    packed = _check_packed(packed, columns)
    out = torch.empty(packed.shape[0], int(columns), dtype=dtype, device=device)
    code = _lib.load().qste_unpack_bits(
        _ptr(packed), _ptr(out), _dtype_code(out), packed.shape[0], int(columns), _stream(device))
    _lib.check(code, "unpack_bits")
    return out


def apply_bits(values: Tensor, packed: Tensor, columns: int) -> Tensor:
    """``values`` where the bit is set, zero where it is not (fallback.py:57-70)."""

    return masked_backward(values, packed, columns)


def masked_backward(grad: Tensor, packed: Tensor, columns: int, *, inside: float = 1.0,
                    outside: float = 0.0) -> Tensor:
    """Backward of a one-bit activation (src/qste/nn.py:133-136, 168-181, 278-282, 364-368).

    ``kept = bit ? grad : 0``; ``kept * inside`` when ``outside == 0``, else
    ``grad * outside + kept * (inside - outside)``, each product rounded to
    the dtype like the reference's tensor expressions.
    """

    device = _require_gpu(grad, packed)
    grad = _rows2d(grad, "masked_backward")
    rows, cols = grad.shape
    if cols != columns:
        raise ValueError(f"value width {cols} does not match {columns} columns")
    packed = _check_packed(packed, columns, rows)
    out = torch.empty_like(grad)
    code = _lib.load().qste_masked_backward(
        _ptr(grad), _dtype_code(grad), _ptr(packed), _ptr(out), rows, cols, float(inside),
        float(outside), float(inside - outside), _stream(device))
    _lib.check(code, "masked_backward")
    return out


def masked_activation(x: Tensor, kind: int, *, lower: float = 0.0, upper: float | None = None,
                      slope: float = 0.0, want_output: bool = True) -> tuple[Tensor | None, Tensor]:
    """Forward of a one-bit activation and its packed mask, in one pass.

    ``x`` is rank 2; returns ``(output or None, packed)``.
    """

    device = _require_gpu(x)
    x = _rows2d(x, "masked_activation")
    rows, cols = x.shape
    out = torch.empty_like(x) if (want_output and kind != MASK_INTERVAL) else None
    packed = torch.empty(rows, _packed_width(cols), dtype=torch.uint8, device=device)
    code = _lib.load().qste_masked_activation(
        _ptr(x), _dtype_code(x), int(kind), float(lower), float(0.0 if upper is None else upper),
        0 if upper is None else 1, float(slope), _ptr(out), _ptr(packed), rows, cols,
        _stream(device))
    _lib.check(code, "masked_activation")
    return out, packed


def smooth_activation(x: Tensor | None, kind: str, param: float = 0.0, *,
                      output: Tensor | None = None,
                      derivative: Tensor | None = None) -> tuple[Tensor | None, Tensor, Tensor]:
    """Smooth activation with its row-quantized derivative (src/qste/nn.py:487-502).

    ``x`` rank 2.  When ``output`` is given it holds f(x) already and is read;
    otherwise f(x) is computed and returned.  ``kind == "provided"`` quantizes
    ``derivative`` (fp32) instead.  Returns ``(output, payload, scale)``:
    payload int8 (uint8 for ``relu_square``) ``[rows, cols]``, scale fp32 ``[rows]``.
    """

    code_kind = SMOOTH_KINDS[kind]
    if kind == "provided":
        device = _require_gpu(derivative)
        derivative = _rows2d(derivative.float(), "smooth_activation")
        rows, cols = derivative.shape
        dtype_code, x_ptr, y_ptr, y_given = 0, None, None, 0
        out = None
    else:
        device = _require_gpu(x, output)
        x = _rows2d(x, "smooth_activation")
        rows, cols = x.shape
        dtype_code = _dtype_code(x)
        if output is not None:
            output = _rows2d(output, "smooth_activation")
            if output.shape != x.shape or output.dtype != x.dtype:
                raise ValueError("output must match the input's shape and dtype")
            out, y_given = output, 1
        else:
            out, y_given = torch.empty_like(x), 0
        x_ptr, y_ptr = _ptr(x), _ptr(out)
    payload = torch.empty(rows, cols, dtype=torch.uint8 if kind == "relu_square" else torch.int8,
                          device=device)
    scale = torch.empty(rows, dtype=torch.float32, device=device)
    code = _lib.load().qste_smooth_activation(
        x_ptr, dtype_code, code_kind, float(param), y_ptr, y_given, _ptr(derivative),
        _ptr(payload), _ptr(scale), rows, cols, _stream(device))
    _lib.check(code, "smooth_activation")
    return out, payload, scale


def smooth_backward(grad: Tensor, payload: Tensor, scale: Tensor) -> Tensor:
    """``grad * (payload * scale)`` per row (src/qste/nn.py:504-507, 325-330)."""

    device = _require_gpu(grad, payload, scale)
    grad = _rows2d(grad, "smooth_backward")
    rows, cols = grad.shape
    if payload.shape != grad.shape or scale.shape != (rows,):
        raise ValueError("payload/scale do not match the gradient's shape")
    payload = _aligned(payload)
    out = torch.empty_like(grad)
    scale_f32 = _f32(scale)  # held until the launch is queued
    code = _lib.load().qste_smooth_backward(
        _ptr(grad), _dtype_code(grad), _ptr(payload), 1 if payload.dtype == torch.uint8 else 0,
        _ptr(scale_f32), _ptr(out), rows, cols, _stream(device))
    _lib.check(code, "smooth_backward")
    return out


# ---------------------------------------------------------------------------
# the SwiGLU gate (no counterpart in the reference)
# ---------------------------------------------------------------------------


def swiglu_forward(gate: Tensor, up: Tensor, *, encode: bool = False):
    """``silu(gate) * up`` with torch's roundings, in one pass.

    Returns ``(out, encoding)``; with ``encode`` the encoding is
    ``(packed, offset, scale)`` of ``out``'s rows as ``pack_affine_rows``
    gives them (last dimension = row), else None.
    """

    device = _require_gpu(gate, up)
    if gate.shape != up.shape or gate.dtype != up.dtype:
        raise ValueError("gate and up must have the same shape and dtype")
    g, u = _aligned(gate), _aligned(up)
    cols = int(g.shape[-1]) if g.dim() else 1
    rows = g.numel() // cols if cols else 0
    out = torch.empty_like(g)
    packed = offset = scale = None
    if encode:
        packed = torch.empty(rows, _packed_width(cols), dtype=torch.uint8, device=device)
        offset, scale = torch.empty(2, rows, dtype=torch.float32, device=device).unbind(0)
    code = _lib.load().qste_swiglu_forward(
        _ptr(g), _ptr(u), _dtype_code(g), _ptr(out), _ptr(packed), _ptr(offset), _ptr(scale), rows, cols,
        _stream(device))
    _lib.check(code, "swiglu_forward")
    return out, ((packed, offset, scale) if encode else None)


def swiglu_backward(grad: Tensor, gate: Tensor, up: Tensor) -> tuple[Tensor, Tensor]:
    """``(grad_gate, grad_up)`` of ``silu(gate) * up`` with torch's roundings."""

    device = _require_gpu(grad, gate, up)
    if not (grad.shape == gate.shape == up.shape) or not (grad.dtype == gate.dtype == up.dtype):
        raise ValueError("grad, gate and up must have the same shape and dtype")
    dh, g, u = _aligned(grad), _aligned(gate), _aligned(up)
    dg, du = torch.empty_like(g), torch.empty_like(g)
    code = _lib.load().qste_swiglu_backward(
        _ptr(dh), _ptr(g), _ptr(u), _dtype_code(g), _ptr(dg), _ptr(du), g.numel(), _stream(device))
    _lib.check(code, "swiglu_backward")
    return dg, du


def swiglu_backward_sums(grad: Tensor, gate: Tensor, up: Tensor, offset_gate: Tensor,
                         offset_up: Tensor, *, side_by_side: bool = False):
    """``swiglu_backward`` of [rows, cols] operands plus ``sums`` fp32 [2, cols]:
    ``sum_t grad_gate[t] * offset_gate[t]`` and ``sum_t grad_up[t] * offset_up[t]``,
    each what ``linear_backward`` would sum from that gradient and offset
    (its ``offset_dot``).  Returns ``(grad_gate, grad_up, sums)``.

    With ``side_by_side`` (16-bit dtypes, cols a multiple of 8) both
    gradients go into one [rows, 2 cols] tensor, grad_gate in its first
    cols columns and grad_up in the rest, and the call returns ``(grads,
    sums)``: two layers that read one input then run their backward as one
    ``linear_backward`` over ``grads`` and their concatenated signs
    (``qste_swiglu_backward_sums_into``)."""

    device = _require_gpu(grad, gate, up, offset_gate, offset_up)
    if not (grad.shape == gate.shape == up.shape) or not (grad.dtype == gate.dtype == up.dtype):
        raise ValueError("grad, gate and up must have the same shape and dtype")
    if grad.dim() != 2:
        raise ValueError("swiglu_backward_sums expects rank-2 operands")
    rows, cols = grad.shape
    offs = []
    for name, o in (("offset_gate", offset_gate), ("offset_up", offset_up)):
        if o.dtype != torch.float32 or o.numel() != rows:
            raise ValueError(f"{name} must be fp32 [rows]")
        offs.append(o.contiguous())
    dh, g, u = _aligned(grad), _aligned(gate), _aligned(up)
    sums = torch.empty(2, cols, dtype=torch.float32, device=device)
    lib = _lib.load()
    work = _workspace(lib.qste_swiglu_backward_sums_workspace_bytes(rows, cols), device)
    if side_by_side:
        both = torch.empty(rows, 2 * cols, dtype=g.dtype, device=device)
        code = lib.qste_swiglu_backward_sums_into(
            _ptr(dh), _ptr(g), _ptr(u), _dtype_code(g), _ptr(both), _ptr(offs[0]), _ptr(offs[1]), _ptr(sums),
            rows, cols, _ptr(work), work.numel(), _stream(device))
        _lib.check(code, "swiglu_backward_sums")
        return both, sums
    dg, du = torch.empty_like(g), torch.empty_like(g)
    code = lib.qste_swiglu_backward_sums(
        _ptr(dh), _ptr(g), _ptr(u), _dtype_code(g), _ptr(dg), _ptr(du), _ptr(offs[0]), _ptr(offs[1]),
        _ptr(sums), rows, cols, _ptr(work), work.numel(), _stream(device))
    _lib.check(code, "swiglu_backward_sums")
    return dg, du, sums


# ---------------------------------------------------------------------------
# 8-bit blocks, and the gated feed-forward block (no counterparts in the reference)
# ---------------------------------------------------------------------------

BLOCK = 32  # columns that share a power of two, as in csrc/blocks.hpp


class Blocks8(NamedTuple):
    """A tensor in 8-bit blocks: ``payload * 2 ** (codes - 133)``, a code for every
    32 columns of a row (the last may have fewer)."""

    payload: Tensor  # int8, the tensor's shape
    codes: Tensor  # uint8 [..., ceil(columns / 32)]
    dtype: torch.dtype  # the tensor's


_HERE = contextlib.nullcontext()


def _device_of(device: torch.device):
    """A context in which the library's launches go to ``device``: nothing where that is the current one."""

    return _HERE if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _blocks_like(t: Tensor) -> Blocks8:
    """Room for t's blocks."""

    codes = torch.empty(*t.shape[:-1], -(-t.shape[-1] // BLOCK), dtype=torch.uint8, device=t.device)
    return Blocks8(torch.empty(t.shape, dtype=torch.int8, device=t.device), codes, t.dtype)


def _check_blocks(b: Blocks8, what: str) -> Blocks8:
    payload, codes, dtype = b
    if payload.dtype != torch.int8 or codes.dtype != torch.uint8:
        raise TypeError(f"{what} need an int8 payload and uint8 codes, got {payload.dtype} and {codes.dtype}")
    if dtype not in _DTYPES:
        raise TypeError(f"unsupported dtype {dtype}; expected float32, float16 or bfloat16")
    if payload.dim() == 0 or codes.shape != (*payload.shape[:-1], -(-payload.shape[-1] // BLOCK)):
        raise ValueError(f"{what} with a payload of shape {tuple(payload.shape)} have codes of shape "
                         f"{tuple(codes.shape)}")
    return Blocks8(payload.contiguous(), codes.contiguous(), dtype)


def _rows_of(t: Tensor) -> tuple[int, int]:
    """(rows, columns) of a tensor over its last dimension."""

    cols = int(t.shape[-1])
    return (t.numel() // cols if cols else 0), cols


def quantize_blocks(values: Tensor) -> Blocks8:
    """``values`` (fp32, fp16 or bf16, any shape but a scalar's) in 8-bit blocks along the last dimension;
    without a gradient, as every call here."""

    device = _require_gpu(values)
    code = _dtype_code(values)
    if values.dim() == 0:
        raise ValueError("quantize_blocks needs at least one dimension")
    x = values.detach().contiguous()
    out = _blocks_like(x)
    with _device_of(device):
        _lib.check(_lib.load().qste_quantize_blocks(_ptr(x), code, _ptr(out.payload), _ptr(out.codes), *_rows_of(x),
                                                    _stream(device)), "quantize_blocks")
    return out


def dequantize_blocks(blocks: Blocks8, dtype: torch.dtype | None = None) -> Tensor:
    """What ``blocks`` stand for, in their own dtype (exactly) or in ``dtype`` (rounded once)."""

    payload, codes, own = _check_blocks(blocks, "blocks")
    device = _require_gpu(payload, codes)
    out = torch.empty(payload.shape, dtype=own if dtype is None else dtype, device=device)
    code = _dtype_code(out)
    with _device_of(device):
        _lib.check(_lib.load().qste_dequantize_blocks(_ptr(payload), _ptr(codes), _ptr(out), code, *_rows_of(out),
                                                      _stream(device)), "dequantize_blocks")
    return out


def swiglu_forward_blocks(gate: Tensor, up: Tensor, *, encode: bool = False):
    """``swiglu_forward`` that also keeps gate and up in 8-bit blocks, from the
    same pass.  Returns ``(out, encoding, gate blocks, up blocks)``."""

    device = _require_gpu(gate, up)
    if gate.shape != up.shape or gate.dtype != up.dtype:
        raise ValueError("gate and up must have the same shape and dtype")
    code = _dtype_code(gate)
    if gate.dim() == 0:
        raise ValueError("swiglu with a checkpoint needs at least one dimension")
    g, u = _aligned(gate), _aligned(up)
    rows, cols = _rows_of(g)
    out, kept_g, kept_u = torch.empty_like(g), _blocks_like(g), _blocks_like(g)
    packed = offset = scale = None
    if encode:
        packed = torch.empty(rows, _packed_width(cols), dtype=torch.uint8, device=device)
        offset, scale = torch.empty(2, rows, dtype=torch.float32, device=device).unbind(0)
    with _device_of(device):
        _lib.check(_lib.load().qste_swiglu_forward_blocks(
            _ptr(g), _ptr(u), code, _ptr(out), _ptr(packed), _ptr(offset), _ptr(scale), _ptr(kept_g.payload),
            _ptr(kept_g.codes), _ptr(kept_u.payload), _ptr(kept_u.codes), rows, cols, _stream(device)),
            "swiglu_forward_blocks")
    return out, ((packed, offset, scale) if encode else None), kept_g, kept_u


def swiglu_backward_blocks(grad: Tensor, gate: Blocks8, up: Blocks8, offset_gate: Tensor | None = None,
                           offset_up: Tensor | None = None, *, side_by_side: bool = False):
    """The gradients of ``silu(gate) * up`` at the gate and up that 8-bit blocks stand
    for, ``(grad_gate, grad_up)``, rounded once; with offsets fp32 [rows] also their
    sums, laid out as ``swiglu_backward_sums`` does (``side_by_side`` as there, for
    callers of these functions: the autograd nodes that run two layers as one take
    ``gated_backward``'s pass)."""

    gate, up = _check_blocks(gate, "gate blocks"), _check_blocks(up, "up blocks")
    device = _require_gpu(grad, gate.payload, gate.codes, up.payload, up.codes, offset_gate, offset_up)
    if not (grad.shape == gate.payload.shape == up.payload.shape) or not (grad.dtype == gate.dtype == up.dtype):
        raise ValueError("grad and the blocks of gate and up must have the same shape and dtype")
    code = _dtype_code(grad)
    dh = _aligned(grad)
    rows, cols = _rows_of(dh)
    kept = (_ptr(gate.payload), _ptr(gate.codes), _ptr(up.payload), _ptr(up.codes))
    lib = _lib.load()
    if offset_gate is None and offset_up is None:
        if side_by_side:
            raise ValueError("side_by_side needs the offsets")
        dg, du = torch.empty_like(dh), torch.empty_like(dh)
        with _device_of(device):
            _lib.check(lib.qste_swiglu_backward_blocks(_ptr(dh), code, *kept, _ptr(dg), _ptr(du), rows, cols,
                                                       _stream(device)), "swiglu_backward_blocks")
        return dg, du
    offs = []
    for name, o in (("offset_gate", offset_gate), ("offset_up", offset_up)):
        if o is None or o.dtype != torch.float32 or o.numel() != rows:
            raise ValueError(f"{name} must be fp32 [rows]")
        offs.append(o.contiguous())
    if side_by_side and (dh.dtype == torch.float32 or cols % 8):
        raise ValueError("side_by_side needs a 16-bit dtype and columns in whole eights")
    sums = torch.empty(2, cols, dtype=torch.float32, device=device)
    work = _workspace(lib.qste_swiglu_backward_blocks_sums_workspace_bytes(rows, cols), device)
    if side_by_side:
        both = torch.empty(rows, 2 * cols, dtype=dh.dtype, device=device)
        at, ld = (_ptr(both), _ptr(both) + cols * dh.element_size()), 2 * cols
    else:
        dg, du = torch.empty_like(dh), torch.empty_like(dh)
        at, ld = (_ptr(dg), _ptr(du)), cols
    with _device_of(device):
        _lib.check(lib.qste_swiglu_backward_blocks_sums(_ptr(dh), code, *kept, *at, ld, _ptr(offs[0]), _ptr(offs[1]),
                                                        _ptr(sums), rows, cols, _ptr(work), work.numel(),
                                                        _stream(device)), "swiglu_backward_blocks_sums")
    return (both, sums) if side_by_side else (dg, du, sums)


def _layer_vector(t: Tensor | None, rows: int, what: str) -> Tensor | None:
    """A layer's scale or bias, an entry per row in any shape, as contiguous fp32 [rows]."""

    if t is None:
        return None
    if t.shape != (rows,):
        if t.numel() != rows:
            raise ValueError(f"{what} has shape {tuple(t.shape)}, expected ({rows},)")
        t = t.reshape(rows)
    return t if t.dtype is torch.float32 and t.is_contiguous() else _f32(t)


def gated_forward(inputs: Tensor, gate: Tensor, gate_scale: Tensor, gate_bias: Tensor | None, up: Tensor,
                  up_scale: Tensor, up_bias: Tensor | None, columns: int, *, keep: str = ""):
    """``silu(g) * u`` of two packed layers of one input, g and u being
    ``packed_linear_affine`` of ``gate`` and ``up`` (packed signs [rows, ...]).

    ``keep`` says what a backward is to find: "" nothing, "values" g and u, "blocks"
    them in 8-bit blocks.  Returns ``(out, g, u)``, g and u tensors, ``Blocks8``
    or None.
    """

    device = _require_gpu(inputs, gate, gate_scale, gate_bias, up, up_scale, up_bias)
    code = _dtype_code(inputs)
    columns = int(columns)
    if inputs.dim() == 0 or inputs.shape[-1] != columns:
        raise ValueError(f"inputs of shape {tuple(inputs.shape)} do not match {columns} columns")
    if keep not in ("", "values", "blocks"):
        raise ValueError(f"keep must be '', 'values' or 'blocks', got {keep!r}")
    gate, up = _check_packed(gate, columns), _check_packed(up, columns)
    rows = gate.shape[0]
    if up.shape[0] != rows:
        raise ValueError(f"gate has {rows} rows and up {up.shape[0]}")
    gs, us = _layer_vector(gate_scale, rows, "gate_scale"), _layer_vector(up_scale, rows, "up_scale")
    gb = None if gate_bias is None else _layer_vector(gate_bias, rows, "gate_bias")
    ub = None if up_bias is None else _layer_vector(up_bias, rows, "up_bias")
    x = _aligned(inputs)
    # the signs are contiguous already: in place of a second look by _aligned, 0.3 us
    if gate.data_ptr() % 16:
        gate = gate.clone()
    if up.data_ptr() % 16:
        up = up.clone()
    m = x.numel() // columns if columns else _leading(inputs)
    out = torch.empty((*x.shape[:-1], rows), dtype=x.dtype, device=device)
    g = u = None
    values, blocks = (None, None), (None, None, None, None)
    if keep == "values":
        g, u = torch.empty_like(out), torch.empty_like(out)
        values = (_ptr(g), _ptr(u))
    elif keep == "blocks":
        g, u = _blocks_like(out), _blocks_like(out)
        blocks = (_ptr(g.payload), _ptr(g.codes), _ptr(u.payload), _ptr(u.codes))
    lib = _lib.load()
    nbytes = lib.qste_gated_workspace_bytes(m, rows, columns, code, {"": 0, "values": 1, "blocks": 2}[keep])
    work = _workspace(nbytes, device) if nbytes else None
    with _device_of(device):
        _lib.check(lib.qste_gated(x.data_ptr(), code, gate.data_ptr(), gs.data_ptr(), _ptr(gb), up.data_ptr(),
                                  us.data_ptr(), _ptr(ub), out.data_ptr(), *values, *blocks, m, rows, columns,
                                  _ptr(work), nbytes, _stream(device)), "gated_forward")
    return out, g, u


def gated_backward(grad: Tensor, gate, up, packed_x: Tensor, x_offset: Tensor, x_scale: Tensor, packed_w: Tensor,
                   scale: Tensor, columns: int, *, need_input: bool = True, need_bias: bool = False):
    """The backward of ``gated_forward`` from out's gradient [samples, rows] (bf16 or
    fp16, rows a multiple of 8): ``(dx, evidence, grad_scale, grad_bias)`` of the two
    layers as one of 2 rows, dx None without ``need_input`` and grad_bias without ``need_bias``.

    ``gate`` and ``up`` are what the forward kept, tensors or ``Blocks8``; ``packed_x``,
    ``x_offset`` and ``x_scale`` the encoding of its input (``pack_affine_rows``), ``packed_w``
    [2 rows, ...] and ``scale`` [2 rows] both layers' signs and scales, gate's first.
    """

    grads = _gated_grads(grad, gate, up, x_offset, x_scale)
    return _gated_products(*grads, packed_x, x_scale, packed_w, scale, columns, need_input, need_bias)


# In two halves for the autograd nodes: out's gradient is free once the first is queued.


def _gated_grads(grad: Tensor, gate, up, x_offset: Tensor, x_scale: Tensor) -> tuple[Tensor, Tensor, Tensor]:
    """gate's and up's gradients side by side [samples, 2 rows], the same as the
    evidence takes them, and the sums over the samples (``qste_gated_backward``)."""

    kept = isinstance(gate, Blocks8)
    if kept != isinstance(up, Blocks8):
        raise TypeError("gate and up are both tensors or both Blocks8")
    if kept:
        gate, up = _check_blocks(gate, "gate blocks"), _check_blocks(up, "up blocks")
        parts, shapes = (*gate[:2], *up[:2]), (gate.payload.shape, up.payload.shape)
    else:
        parts, shapes = (gate, up), (gate.shape, up.shape)
    device = _require_gpu(grad, *parts, x_offset, x_scale)
    if grad.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"gated_backward takes bfloat16 or float16, got {grad.dtype}")
    if grad.dim() != 2 or grad.shape[1] % 8 or not grad.numel():
        raise ValueError("gated_backward expects a rank-2 gradient with rows and whole eights of columns")
    if not (grad.shape == shapes[0] == shapes[1]) or not (grad.dtype == gate.dtype == up.dtype):
        raise ValueError("grad, gate and up must have the same shape and dtype")
    samples, rows = (int(s) for s in grad.shape)
    offset, xs = _layer_vector(x_offset, samples, "x_offset"), _layer_vector(x_scale, samples, "x_scale")
    dh = _aligned(grad)
    parts = tuple(_aligned(t) for t in parts)  # held until the launch is queued
    sources = (None, None, *map(_ptr, parts)) if kept else (*map(_ptr, parts), None, None, None, None)
    both, ev = torch.empty(2, samples, 2 * rows, dtype=grad.dtype, device=device).unbind(0)
    sums = torch.empty(4 * rows, dtype=torch.float32, device=device)
    lib = _lib.load()
    work = _workspace(lib.qste_gated_backward_workspace_bytes(samples, rows), device)
    with _device_of(device):
        _lib.check(lib.qste_gated_backward(_ptr(dh), _DTYPES[grad.dtype], *sources, _ptr(both), _ptr(ev), _ptr(offset),
                                           _ptr(xs), _ptr(sums), samples, rows, _ptr(work), work.numel(),
                                           _stream(device)), "gated_backward")
    return both, ev, sums


def _gated_products(both: Tensor, ev: Tensor, sums: Tensor, packed_x: Tensor, x_scale: Tensor, packed_w: Tensor,
                    scale: Tensor, columns: int, need_input: bool, need_bias: bool):
    """What ``gated_backward`` returns, from what ``_gated_grads`` does."""

    device = _require_gpu(both, packed_x, x_scale, packed_w, scale)
    samples, rows = both.shape
    columns = int(columns)
    packed_x, packed_w = _check_packed(packed_x, columns, samples), _check_packed(packed_w, columns, rows)
    xs, scale = _layer_vector(x_scale, samples, "x_scale"), _layer_vector(scale, rows, "scale")
    dx = torch.empty(samples, columns, dtype=both.dtype, device=device) if need_input else None
    evidence = torch.empty(rows, columns, dtype=torch.float32, device=device)
    grad_scale = torch.empty(rows, dtype=torch.float32, device=device)
    lib, code = _lib.load(), _DTYPES[both.dtype]
    nbytes = lib.qste_linear_backward_operands_workspace_bytes(samples, rows, columns, code)
    work = _workspace(nbytes, device)
    with _device_of(device):
        _lib.check(lib.qste_linear_backward_operands(
            _ptr(both), _ptr(ev), code, _ptr(packed_x), _ptr(xs), _ptr(packed_w), _ptr(scale), _ptr(dx), _ptr(evidence),
            _ptr(grad_scale), _ptr(sums), samples, rows, columns, _ptr(work), nbytes, _stream(device)),
            "linear_backward_operands")
    return dx, evidence, grad_scale, (sums[rows:] if need_bias else None)


def _leading(t: Tensor) -> int:
    count = 1
    for size in t.shape[:-1]:
        count *= int(size)
    return count


def row_scale(log_scale: Tensor, lo: float, hi: float) -> tuple[Tensor, Tensor]:
    """``(clamp(exp(log_scale), lo, hi), exp(log_scale))`` in log_scale's
    dtype (fp32, fp16 or bf16), one launch (surface.py:84-85), rounded as
    torch's ``exp().clamp()`` on that dtype."""

    device = _require_gpu(log_scale)
    ls = log_scale.detach().contiguous()
    scale, e = torch.empty_like(ls), torch.empty_like(ls)
    code = _lib.load().qste_row_scale(_ptr(ls), _dtype_code(ls), _ptr(scale), _ptr(e), ls.numel(), float(lo),
                                      float(hi), _stream(device))
    _lib.check(code, "row_scale")
    return scale, e


def row_scale_backward(exp_value: Tensor, grad: Tensor, lo: float, hi: float) -> Tensor:
    """Gradient of ``row_scale`` at log_scale: ``(lo <= e <= hi ? grad : 0) * e``,
    in e's dtype (grad is taken in that dtype)."""

    device = _require_gpu(exp_value, grad)
    if grad.shape != exp_value.shape:
        raise ValueError("row_scale_backward takes operands of one shape")
    e, g = exp_value.contiguous(), grad.to(exp_value.dtype).contiguous()
    out = torch.empty_like(e)
    code = _lib.load().qste_row_scale_backward(_ptr(e), _ptr(g), _dtype_code(e), _ptr(out), e.numel(), float(lo),
                                               float(hi), _stream(device))
    _lib.check(code, "row_scale_backward")
    return out


def pair_scale(log_gate: Tensor, gate_bounds: tuple[float, float], log_up: Tensor, up_bounds: tuple[float, float],
               padded: int) -> tuple[Tensor, Tensor]:
    """``row_scale`` of two layers that run as one: ``(scale, exp)``, fp32 [2 padded]
    of values in the log-scales' own dtypes, zeros behind each layer's rows."""

    device = _require_gpu(log_gate, log_up)
    rows, padded = log_gate.numel(), int(padded)
    if log_up.numel() != rows or padded < rows:
        raise ValueError(f"log-scales of {rows} and {log_up.numel()} rows in {padded}")
    lg, lu = log_gate.detach().contiguous(), log_up.detach().contiguous()
    out = torch.empty(2, 2 * padded, dtype=torch.float32, device=device)
    scale, e = out.unbind(0)
    with _device_of(device):
        _lib.check(_lib.load().qste_pair_scale(_ptr(lg), _dtype_code(lg), *gate_bounds, _ptr(lu), _dtype_code(lu),
                                               *up_bounds, _ptr(scale), _ptr(e), rows, padded, _stream(device)),
                   "pair_scale")
    return scale, e


def pair_scale_backward(exp_value: Tensor, grad: Tensor, gate_dtype: torch.dtype, gate_bounds: tuple[float, float],
                        up_dtype: torch.dtype, up_bounds: tuple[float, float], rows: int) -> tuple[Tensor, Tensor]:
    """The log-scales' gradients [rows] for the gradient fp32 [2 padded] of
    ``pair_scale``'s scales: in fp32, rounded once to their dtypes."""

    device = _require_gpu(exp_value, grad)
    if exp_value.shape != grad.shape or not exp_value.dtype == grad.dtype == torch.float32 or exp_value.dim() != 1:
        raise ValueError("pair_scale_backward takes fp32 vectors of one shape")
    e, g = exp_value.contiguous(), grad.contiguous()
    log_g = torch.empty(rows, dtype=gate_dtype, device=device)
    log_u = torch.empty(rows, dtype=up_dtype, device=device)
    with _device_of(device):
        _lib.check(_lib.load().qste_pair_scale_backward(
            _ptr(e), _ptr(g), _ptr(log_g), _dtype_code(log_g), *gate_bounds, _ptr(log_u), _dtype_code(log_u), *up_bounds,
            rows, e.numel() // 2, _stream(device)), "pair_scale_backward")
    return log_g, log_u


def step_finish(log_scales: list[Tensor], lo: float, hi: float, flips: list[Tensor]) -> Tensor | None:
    """``clamp_(lo, hi)`` of every log-scale and the sum of the flip counters
    (device int64 scalars), one launch; None, with nothing done, unless all
    are plain tensors of one GPU (log-scales fp32 and contiguous)."""

    device = log_scales[0].device
    if device.type != "cuda" or len(flips) > len(log_scales):
        return None
    for t in log_scales:
        if type(t) is not Tensor or t.dtype != torch.float32 or t.device != device or not t.is_contiguous():
            return None
    for t in flips:
        if type(t) is not Tensor or t.dtype != torch.int64 or t.device != device or t.numel() != 1:
            return None
    count = len(log_scales)
    total = torch.empty((), dtype=torch.int64, device=device)
    pointers, lengths = ctypes.c_void_p * count, ctypes.c_int64 * count
    code = _lib.load().qste_step_finish(
        pointers(*[t.data_ptr() for t in log_scales]), lengths(*[t.numel() for t in log_scales]), count,
        pointers(*[t.data_ptr() for t in flips]), len(flips), float(lo), float(hi), _ptr(total), _stream(device))
    _lib.check(code, "step_finish")
    return total


# ---------------------------------------------------------------------------
# binary embedding (reference: cuda.py:1691-1702, functional.py:260-287)
# ---------------------------------------------------------------------------


def _check_ids(ids: Tensor, rows: int) -> Tensor:
    flat = ids.reshape(-1).to(torch.int64).contiguous()
    if flat.numel():
        lo, hi = torch.stack(torch.aminmax(flat)).tolist()  # one reduction, one copy to the host
    if flat.numel() and (lo < 0 or hi >= rows):
        raise IndexError(f"embedding id out of range for {rows} rows")
    return flat


def packed_embedding(ids: Tensor, packed: Tensor, scale: Tensor, columns: int) -> Tensor:
    """``sign(packed[ids]) * scale[ids]``, shape ``ids.shape + (columns,)``, in scale's dtype.

    fallback.py:151-155.
    """

    device = _require_gpu(ids, packed, scale)
    packed = _check_packed(packed, columns)
    rows = packed.shape[0]
    if scale.shape != (rows,):
        raise ValueError(f"scale has shape {tuple(scale.shape)}, expected ({rows},)")
    flat = _check_ids(ids, rows)
    out_dtype = scale.dtype if scale.dtype in _DTYPES else torch.float32
    out = torch.empty(flat.numel(), int(columns), dtype=out_dtype, device=device)
    scale_f32 = _f32(scale)  # held until the launch is queued
    code = _lib.load().qste_packed_embedding(
        _ptr(flat), flat.numel(), _ptr(packed), _ptr(scale_f32), _ptr(out), _dtype_code(out), rows,
        int(columns), _stream(device))
    _lib.check(code, "packed_embedding")
    return out.view(*ids.shape, int(columns)).to(scale.dtype)


def embedding_backward(ids: Tensor, grad: Tensor, packed: Tensor, scale: Tensor,
                       columns: int) -> tuple[Tensor, Tensor]:
    """``(evidence, grad_scale)`` of an embedding (functional.py:274-286).

    ``evidence = zeros(R, C).index_add_(0, ids, grad) * scale[r]`` (fp32,
    token-order sums) and ``grad_scale = row_inner(index_add_, signs)``.
    """

    device = _require_gpu(ids, grad, packed, scale)
    packed = _check_packed(packed, columns)
    rows = packed.shape[0]
    flat = _check_ids(ids, rows)
    g = grad.reshape(-1, int(columns)).contiguous()
    if g.shape[0] != flat.numel():
        raise ValueError("gradient rows do not match the number of ids")
    evidence = torch.empty(rows, int(columns), dtype=torch.float32, device=device)
    grad_scale = torch.empty(rows, dtype=torch.float32, device=device)
    lib = _lib.load()
    ws = _workspace(lib.qste_embedding_backward_workspace_bytes(flat.numel(), rows), device)
    scale_f32 = _f32(scale)  # held until the launch is queued
    code = lib.qste_embedding_backward(
        _ptr(flat), flat.numel(), _ptr(g), _dtype_code(g), _ptr(packed), _ptr(scale_f32),
        _ptr(evidence), _ptr(grad_scale), rows, int(columns), _ptr(ws), ws.numel(), _stream(device))
    _lib.check(code, "embedding_backward")
    return evidence, grad_scale


# ---------------------------------------------------------------------------
# scores of tokens, distillation from a teacher's top tokens (no counterparts
# in the reference)
# ---------------------------------------------------------------------------

MAX_TOP, MAX_ENTRIES, MAX_VOCAB, DISTILL_STATS = 128, 1024, 1 << 30, 6  # as in include/qste_hip.h


def _logit_rows(logits: Tensor) -> tuple[Tensor, tuple[int, int, int, int, int]]:
    """``logits`` and its rows as (outer, inner, outer_stride, inner_stride, vocab):
    itself where the leading dimensions come down to two strides (any view
    whose columns are adjacent, such as ``logits[:, :-1]``), else a copy."""

    if logits.dim() == 0 or not 0 < logits.shape[-1] <= MAX_VOCAB:
        raise ValueError(f"logits need a last dimension of 1 to {MAX_VOCAB} columns")
    vocab = int(logits.shape[-1])
    if logits.is_contiguous():
        rows = logits.numel() // vocab
        return logits, (1, rows, 0, vocab, vocab) if rows else (0, 0, 0, 0, vocab)
    groups = _merged_rows(logits)
    if len(groups) > 2 or (vocab > 1 and logits.stride(-1) != 1):
        return _logit_rows(logits.detach().contiguous())
    (outer, outer_stride), (inner, inner_stride) = [(1, 0)] * (2 - len(groups)) + groups
    return logits, (outer, inner, outer_stride, inner_stride, vocab)


def _merged_rows(t: Tensor) -> list[tuple[int, int]]:
    """(size, stride) of the leading dimensions, those that step alike as one."""

    groups: list[tuple[int, int]] = []
    for size, stride in zip(t.shape[:-1], t.stride()[:-1]):
        if size == 1:
            continue
        if groups and groups[-1][1] == size * stride:
            size *= groups.pop()[0]
        groups.append((size, stride))
    return groups


def _temperature(value: float) -> float:
    value = float(value)
    if not 1e-30 <= value < 1e30:
        raise ValueError(f"temperature must be positive and finite, got {value}")
    return value


def _row_tokens(tokens: Tensor, shape, what: str) -> Tensor:
    """Token numbers of the given shape as contiguous int64."""

    if tokens.shape != shape:
        raise ValueError(f"{what} have shape {tuple(tokens.shape)}, expected {tuple(shape)}")
    if tokens.dtype != torch.int64:
        if tokens.dtype not in (torch.int32, torch.int16, torch.int8, torch.uint8):
            raise TypeError(f"{what} must be integers, got {tokens.dtype}")
        tokens = tokens.to(torch.int64)
    return tokens.contiguous()


def _row_weights(weights: Tensor | None, shape, what: str) -> Tensor | None:
    if weights is None:
        return None
    if weights.shape != shape:
        raise ValueError(f"{what} has shape {tuple(weights.shape)}, expected {tuple(shape)}")
    if weights.dtype == torch.float32 and weights.is_contiguous():
        return weights
    return _f32(weights)


# The forwards below come in two layers: the checks, which also say how the rows
# lie and bring tokens and weights to the types the library takes, and the call.
# An autograd node keeps what the checks made and makes its backward's call
# without them (they are half of a small call's time on the host).


def _check_scores(logits: Tensor, tokens: Tensor | None, top: int, temperature: float):
    """(rows, layout, tokens int64 or None, top, temperature)"""

    _require_gpu(logits, tokens)
    _dtype_code(logits)
    rows, layout = _logit_rows(logits)
    top, most = int(top), min(MAX_TOP, layout[4])
    if not 0 <= top <= most:
        raise ValueError(f"top must lie in 0 .. {most}, got {top}")
    tokens_i64 = None if tokens is None else _row_tokens(tokens, logits.shape[:-1], "tokens")
    return rows, layout, tokens_i64, top, _temperature(temperature)


def _call_scores(rows: Tensor, layout, tokens: Tensor | None, top: int, temperature: float, want_stats: bool):
    shape, device, code = rows.shape[:-1], rows.device, _DTYPES[rows.dtype]
    entropy = torch.empty(shape, dtype=torch.float32, device=device)
    logprobs = None if tokens is None else torch.empty_like(entropy)
    top_logprobs = torch.empty(*shape, top, dtype=torch.float32, device=device) if top else None
    top_tokens = torch.empty(*shape, top, dtype=torch.int64, device=device) if top else None
    stats = torch.empty(*shape, 2, dtype=torch.float32, device=device) if want_stats else None
    lib = _lib.load()
    nbytes = lib.qste_token_logprobs_workspace_bytes(entropy.numel(), layout[4], code, top)
    work = _workspace(nbytes, device) if nbytes else None
    _lib.check(lib.qste_token_logprobs(
        rows.data_ptr(), code, *layout, _ptr(tokens), temperature, top, _ptr(logprobs), entropy.data_ptr(),
        _ptr(top_logprobs), _ptr(top_tokens), _ptr(stats), _ptr(work), nbytes, _stream(device)), "token_logprobs")
    return logprobs, entropy, top_logprobs, top_tokens, stats


def _call_scores_backward(rows: Tensor, layout, tokens: Tensor | None, temperature: float, logprob_grad: Tensor | None,
                          entropy_grad: Tensor | None, entropy: Tensor, stats: Tensor) -> Tensor:
    grad = torch.empty(rows.shape, dtype=rows.dtype, device=rows.device)
    _lib.check(_lib.load().qste_token_logprobs_backward(
        rows.data_ptr(), _DTYPES[rows.dtype], *layout, _ptr(tokens), temperature, _ptr(logprob_grad),
        _ptr(entropy_grad), entropy.data_ptr(), stats.data_ptr(), grad.data_ptr(), _stream(rows.device)),
        "token_logprobs_backward")
    return grad


def token_logprobs_forward(logits: Tensor, tokens: Tensor | None, *, top: int = 0, temperature: float = 1.0,
                           want_stats: bool = False):
    """``(logprobs, entropy, top_logprobs, top_tokens, stats)`` of the rows of logits.

    ``logits`` [..., vocab], ``tokens`` [...] or None (logprobs is None then); a
    negative token marks a row that is not scored.  ``top_logprobs`` and
    ``top_tokens`` [..., top] are None for ``top = 0``; ``stats`` fp32 [..., 2], what
    ``token_logprobs_backward`` reads, is None unless asked for.  All but
    ``top_tokens`` (int64) are fp32.
    """

    return _call_scores(*_check_scores(logits, tokens, top, temperature), want_stats)


def token_logprobs_backward(logits: Tensor, tokens: Tensor | None, logprob_grad: Tensor | None,
                            entropy_grad: Tensor | None, entropy: Tensor, stats: Tensor, *,
                            temperature: float = 1.0) -> Tensor:
    """The logits' gradient, contiguous in their dtype, for gradients [...] of the
    log probabilities and the entropies (None: zeros)."""

    _require_gpu(logits, tokens, logprob_grad, entropy_grad, entropy, stats)
    rows, layout, tokens_i64, _, temperature = _check_scores(logits, tokens, 0, temperature)
    shape = logits.shape[:-1]
    return _call_scores_backward(
        rows, layout, tokens_i64, temperature, _row_weights(logprob_grad, shape, "logprob_grad"),
        _row_weights(entropy_grad, shape, "entropy_grad"), _row_weights(entropy, shape, "entropy"),
        _row_weights(stats, (*shape, 2), "stats"))


def _check_distill(logits: Tensor, top_tokens: Tensor, top_logprobs: Tensor, temperature: float, tail: bool):
    """(rows, layout, tokens int64, log probabilities fp32, temperature, tail)"""

    _require_gpu(logits, top_tokens, top_logprobs)
    _dtype_code(logits)
    rows, layout = _logit_rows(logits)
    if top_tokens.dim() != logits.dim() or not 1 <= top_tokens.shape[-1] <= MAX_ENTRIES:
        raise ValueError(f"top_tokens need the logits' leading dimensions and 1 to {MAX_ENTRIES} entries, "
                         f"got {tuple(top_tokens.shape)}")
    if not top_logprobs.dtype.is_floating_point:
        raise TypeError(f"top_logprobs must be floating point, got {top_logprobs.dtype}")
    shape = (*logits.shape[:-1], top_tokens.shape[-1])
    return (rows, layout, _row_tokens(top_tokens, shape, "top_tokens"),
            _row_weights(top_logprobs, shape, "top_logprobs"), _temperature(temperature), int(tail))


def _call_distill(rows: Tensor, layout, tokens: Tensor, values: Tensor, temperature: float, tail: int,
                  weights: Tensor | None, want_stats: bool):
    shape, device, code = rows.shape[:-1], rows.device, _DTYPES[rows.dtype]
    losses = torch.empty(shape, dtype=torch.float32, device=device)
    stats = torch.empty(*shape, DISTILL_STATS, dtype=torch.float32, device=device) if want_stats else None
    grad = torch.empty(rows.shape, dtype=rows.dtype, device=device) if weights is not None else None
    lib = _lib.load()
    nbytes = lib.qste_distill_workspace_bytes(losses.numel(), layout[4], code, int(grad is not None))
    work = _workspace(nbytes, device) if nbytes else None
    _lib.check(lib.qste_distill(
        rows.data_ptr(), code, *layout, tokens.data_ptr(), values.data_ptr(), tokens.shape[-1], temperature, tail,
        losses.data_ptr(), _ptr(stats), _ptr(weights), _ptr(grad), _ptr(work), nbytes, _stream(device)), "distill")
    return losses, stats, grad


def _call_distill_backward(rows: Tensor, layout, tokens: Tensor, values: Tensor, temperature: float, tail: int,
                           weights: Tensor, stats: Tensor) -> Tensor:
    grad = torch.empty(rows.shape, dtype=rows.dtype, device=rows.device)
    _lib.check(_lib.load().qste_distill_backward(
        rows.data_ptr(), _DTYPES[rows.dtype], *layout, tokens.data_ptr(), values.data_ptr(), tokens.shape[-1],
        temperature, tail, stats.data_ptr(), weights.data_ptr(), grad.data_ptr(), _stream(rows.device)),
        "distill_backward")
    return grad


def distill_forward(logits: Tensor, top_tokens: Tensor, top_logprobs: Tensor, *, temperature: float = 1.0,
                    tail: bool = False, loss_grad: Tensor | None = None, want_stats: bool = False):
    """``(losses, stats, grad)``: the losses fp32 [...] of logits [..., vocab] against
    a teacher's ``top_tokens`` and ``top_logprobs`` [..., k]; ``stats`` fp32 [..., 6], what
    ``distill_backward`` reads, if asked for; and with ``loss_grad`` [...] the
    logits' gradient for these weights, from the same pass, else None."""

    checked = _check_distill(logits, top_tokens, top_logprobs, temperature, tail)
    if loss_grad is not None:
        _require_gpu(logits, loss_grad)
    return _call_distill(*checked, _row_weights(loss_grad, logits.shape[:-1], "loss_grad"), want_stats)


def distill_backward(logits: Tensor, top_tokens: Tensor, top_logprobs: Tensor, loss_grad: Tensor, stats: Tensor, *,
                     temperature: float = 1.0, tail: bool = False) -> Tensor:
    """The logits' gradient, contiguous in their dtype, for the weights ``loss_grad`` [...]."""

    checked = _check_distill(logits, top_tokens, top_logprobs, temperature, tail)
    _require_gpu(logits, loss_grad, stats)
    shape = logits.shape[:-1]
    return _call_distill_backward(*checked, _row_weights(loss_grad, shape, "loss_grad"),
                                  _row_weights(stats, (*shape, DISTILL_STATS), "stats"))
