"""MXFP4 projections: 4-bit siblings of the INT8 ops in quant.py.

* ``mxfp4_quant(x)``                 -> (codes uint8 [..., K / 2], scale uint8)
* ``mxfp4_quant_into(q, scale, x)``  the same into caller storage
* ``mxfp4_dequant(q, scale)``        the bf16 values they stand for
* ``mxfp4_scaled_mm(a, b, scale_a, scale_b, out_dtype=torch.bfloat16, bias=None)`` and
  ``mxfp4_scaled_mm_out(out, a, b, scale_a, scale_b, bias=None)``, in the argument order of
  ``cutlass_scaled_mm`` / ``cutlass_scaled_mm_out``: ``b`` is ``weight.t()`` of the row-major codes
* ``mxfp4_linear(inputs, weight, weight_scale, bias=None)``  a projection of bf16 rows
* ``mxfp4_scale_from_rows`` / ``mxfp4_scale_to_rows``  to and from scale bytes kept as ``[rows, K / 32]``

A matrix ``[rows, K]`` (K a multiple of 32) is held as two e2m1 codes a byte
(the even column in the low half) and a scale byte 2^(byte - 127) for every 32
columns of a row (OCP microscaling: the exponent of the block's largest
magnitude less 2; a block that holds an infinity or NaN gets 255, NaN, and all
of its values become NaN).  Scale bytes are kept in the order the product reads
them, ``[ceil(K / 512), 4, R, 4]`` with R = rows rounded up to a multiple of 4:
byte ``b`` of entry ``(s, g, row)`` is that of columns ``512 s + 128 b + 32 g``
and on, zero where there is no such column or row.  The product adds in fp32
and rounds once, to bf16.  Every op runs a gfx950 HIP kernel from libtmhd.so.
"""

from __future__ import annotations

from typing import Any

from . import _native

MXFP4_BLOCK = 32


def _torch():
    import torch

    return torch


def scale_shape(rows: int, cols: int) -> tuple[int, int, int, int]:
    """Shape of the scale bytes of a ``[rows, cols]`` matrix."""
    return (-(-int(cols) // 512), 4, -(-int(rows) // 4) * 4, 4)


def mxfp4_scale_from_rows(scale: Any) -> Any:
    """Scale bytes kept as ``[rows, K / 32]`` (uint8) in the product's order."""
    torch = _torch()
    if not torch.is_tensor(scale) or scale.dtype != torch.uint8 or scale.ndim != 2 or int(scale.shape[1]) == 0:
        raise ValueError("scale must be a [rows, K / 32] uint8 tensor")
    rows, nb = int(scale.shape[0]), int(scale.shape[1])
    blocks, _, r4, _ = scale_shape(rows, nb * MXFP4_BLOCK)
    padded = torch.zeros((r4, blocks * 16), dtype=torch.uint8, device=scale.device)
    padded[:rows, :nb] = scale
    return padded.view(r4, blocks, 4, 4).permute(1, 3, 0, 2).contiguous()


def mxfp4_scale_to_rows(scale: Any, rows: int, cols: int) -> Any:
    """The ``[rows, cols / 32]`` bytes of a scale in the product's order."""
    _check_scale(_torch(), scale, int(rows), int(cols), "scale")
    return scale.permute(2, 0, 3, 1).flatten(1)[: int(rows), : int(cols) // MXFP4_BLOCK].contiguous()


def _check_scale(torch: Any, scale: Any, rows: int, cols: int, name: str) -> None:
    shape = scale_shape(rows, cols)
    if not torch.is_tensor(scale) or scale.dtype != torch.uint8 or scale.shape != shape or not scale.is_contiguous():
        raise ValueError(f"{name} must be a contiguous uint8 tensor of shape {list(shape)} (mxfp4_scale_from_rows)")


def _check_cols(cols: int, name: str) -> None:
    if cols <= 0 or cols % MXFP4_BLOCK:
        raise ValueError(f"{name} needs a multiple of {MXFP4_BLOCK} columns, got {cols}")


def _bf16_rows(torch: Any, x: Any, name: str) -> tuple[Any, int, int, int]:
    """``x`` as 2-D bf16 rows that the kernels read in place (copied if they cannot), their count, width and stride."""
    _native.require_device_tensor(torch, x, name)
    if x.dtype != torch.bfloat16 or x.ndim < 1:
        raise ValueError(f"{name} must be a bf16 tensor with at least one dimension")
    k = x.shape[-1]
    _check_cols(k, name)
    rows = x if x.ndim == 2 else x.reshape(-1, k)
    m = rows.shape[0]
    stride, step = rows.stride()
    if m <= 1:
        stride = k  # a single row's stride says nothing
    if step != 1 or stride % 8 or stride < k or rows.data_ptr() % 16:
        rows = rows.clone(memory_format=torch.contiguous_format)
        stride = k
    return rows, m, k, stride


def _launch_quant(torch: Any, q: Any, scale: Any, rows: Any, m: int, k: int, stride: int) -> None:
    with _native.device_of(torch, rows):
        status = _native.load().tmhd_mxfp4_quant(
            q.data_ptr(), scale.data_ptr(), rows.data_ptr(), m, k, stride, _native.stream_ptr(torch, rows.device),
        )
    _native.check(status, "tmhd_mxfp4_quant")


def mxfp4_quant_into(q: Any, scale: Any, x: Any) -> None:
    """``mxfp4_quant`` writing into caller storage: ``q`` a contiguous uint8
    ``[rows, K / 2]`` tensor, ``scale`` uint8 of ``scale_shape(rows, K)``."""
    torch = _torch()
    rows, m, k, stride = _bf16_rows(torch, x, "x")
    _native.require_same_gpu(torch, rows.device, q=q, scale=scale)
    if q.dtype != torch.uint8 or tuple(q.shape) != (m, k // 2) or not q.is_contiguous():
        raise ValueError("q must be a contiguous uint8 [rows, K / 2] tensor")
    _check_scale(torch, scale, m, k, "scale")
    _launch_quant(torch, q, scale, rows, m, k, stride)


def mxfp4_quant(x: Any) -> tuple[Any, Any]:
    """Rows of bf16 to MXFP4: ``(codes [..., K / 2], scale)`` (activations and weights alike)."""
    torch = _torch()
    rows, m, k, stride = _bf16_rows(torch, x, "x")
    q = torch.empty((*x.shape[:-1], k // 2), dtype=torch.uint8, device=x.device)
    scale = torch.empty(scale_shape(m, k), dtype=torch.uint8, device=x.device)
    _launch_quant(torch, q, scale, rows, m, k, stride)
    return q, scale


def mxfp4_dequant(q: Any, scale: Any) -> Any:
    """The bf16 ``[..., K]`` values that codes ``[..., K / 2]`` and their scale stand for (exact)."""
    torch = _torch()
    _native.require_device_tensor(torch, q, "q")
    if q.dtype != torch.uint8 or q.ndim < 1:
        raise ValueError("q must be a uint8 tensor with at least one dimension")
    k = 2 * int(q.shape[-1])
    _check_cols(k, "q")
    codes = q.reshape(-1, k // 2).contiguous()
    if codes.data_ptr() % 16:
        codes = codes.clone()
    m = codes.shape[0]
    _native.require_same_gpu(torch, codes.device, scale=scale)
    _check_scale(torch, scale, m, k, "scale")
    out = torch.empty((*q.shape[:-1], k), dtype=torch.bfloat16, device=codes.device)
    with _native.device_of(torch, codes):
        status = _native.load().tmhd_mxfp4_dequant(
            out.data_ptr(), codes.data_ptr(), scale.data_ptr(), m, k, _native.stream_ptr(torch, codes.device),
        )
    _native.check(status, "tmhd_mxfp4_dequant")
    return out


def _bias_ptr(torch: Any, bias: Any | None, n: int) -> tuple[int | None, Any]:
    if bias is None:
        return None, None
    if bias.dtype != torch.bfloat16 or bias.numel() != n:
        raise ValueError("bias must be a bf16 vector of N values")
    bias = bias.reshape(-1).contiguous()
    return _native.ptr(bias), bias


def _check_codes(torch: Any, a: Any, b: Any, scale_a: Any, scale_b: Any, bias: Any) -> tuple[int, int, int, int, int]:
    _native.require_device_tensor(torch, a, "a")
    _native.require_same_gpu(torch, a.device, b=b, scale_a=scale_a, scale_b=scale_b, bias=bias)
    if a.dtype != torch.uint8 or b.dtype != torch.uint8:
        raise ValueError("a and b must hold MXFP4 codes in uint8")
    if a.ndim != 2 or b.ndim != 2 or a.stride(1) != 1:
        raise ValueError("a must be a row-major [M, K / 2] matrix of codes")
    m, kb = a.shape
    kb_b, n = b.shape
    step, ldb = b.stride()
    if step != 1:
        raise ValueError("b must be the [K / 2, N] column-major view (weight.t()) of row-major [N, K / 2] codes")
    if kb_b != kb:
        raise ValueError(f"inner dimensions differ: a {tuple(a.shape)}, b {tuple(b.shape)}")
    _check_cols(2 * kb, "a")
    _check_scale(torch, scale_a, m, 2 * kb, "scale_a")
    _check_scale(torch, scale_b, n, 2 * kb, "scale_b")
    # a single row's stride says nothing
    return m, n, 2 * kb, a.stride(0) if m > 1 else kb, ldb if n > 1 else kb


def _launch_mm(torch: Any, out: Any, ldo: int, a: Any, b: Any, scale_a: Any, scale_b: Any, bias: Any,
               sizes: tuple[int, int, int, int, int]) -> None:
    m, n, k, lda, ldb = sizes
    bias_at, bias = _bias_ptr(torch, bias, n)
    with _native.device_of(torch, a):
        status = _native.load().tmhd_gemm_mxfp4(
            out.data_ptr(), a.data_ptr(), b.data_ptr(), scale_a.data_ptr(), scale_b.data_ptr(), bias_at, m, n, k, lda, ldb,
            ldo, _native.stream_ptr(torch, a.device),
        )
    _native.check(status, "tmhd_gemm_mxfp4")


def mxfp4_scaled_mm_out(out: Any, a: Any, b: Any, scale_a: Any, scale_b: Any, bias: Any | None = None) -> None:
    """out = bf16(sum_k a[m, k] b[k, n] (+ bias[n])) of MXFP4 operands, fp32 sums.

    ``a``: codes ``[M, K / 2]``; ``b``: the ``[K / 2, N]`` view (``weight.t()``) of a weight's row-major codes
    ``[N, K / 2]``; the scales as ``mxfp4_quant`` gives them (``scale_b`` for the weight's N rows)."""
    torch = _torch()
    sizes = _check_codes(torch, a, b, scale_a, scale_b, bias)
    m, n = sizes[:2]
    _native.require_same_gpu(torch, a.device, out=out)
    if out.dtype != torch.bfloat16:
        raise NotImplementedError("only bf16 output is implemented")
    if tuple(out.shape) != (m, n) or (n > 1 and out.stride(1) != 1):
        raise ValueError("out must be a row-major [M, N] bf16 tensor")
    _launch_mm(torch, out, out.stride(0) if m > 1 else n, a, b, scale_a, scale_b, bias, sizes)


def mxfp4_scaled_mm(a: Any, b: Any, scale_a: Any, scale_b: Any, out_dtype: Any = None, bias: Any | None = None) -> Any:
    """Allocating form of ``mxfp4_scaled_mm_out``."""
    torch = _torch()
    if out_dtype is not None and out_dtype != torch.bfloat16:
        raise NotImplementedError("only bf16 output is implemented")
    sizes = _check_codes(torch, a, b, scale_a, scale_b, bias)
    out = torch.empty(sizes[:2], dtype=torch.bfloat16, device=a.device)
    _launch_mm(torch, out, sizes[1], a, b, scale_a, scale_b, bias, sizes)
    return out


def mxfp4_linear(inputs: Any, weight: Any, weight_scale: Any, bias: Any | None = None) -> Any:
    """A projection of bf16 rows ``[..., K]`` on an MXFP4 weight (``mxfp4_quant`` of ``[N, K]``): ``[..., N]`` bf16,
    the bits of ``mxfp4_scaled_mm`` of the quantised rows (few rows are quantised inside the product)."""
    torch = _torch()
    rows, m, k, stride = _bf16_rows(torch, inputs, "inputs")
    device = rows.device
    _native.require_same_gpu(torch, device, weight=weight, weight_scale=weight_scale, bias=bias)
    if weight.dtype != torch.uint8 or weight.ndim != 2 or weight.stride(1) != 1 or weight.shape[1] * 2 != k:
        raise ValueError(f"weight must hold row-major MXFP4 codes [N, {k // 2}] in uint8")
    n = weight.shape[0]
    _check_scale(torch, weight_scale, n, k, "weight_scale")
    bias_at, bias = _bias_ptr(torch, bias, n)
    out = torch.empty((*inputs.shape[:-1], n), dtype=torch.bfloat16, device=device)
    with _native.device_of(torch, rows):
        lib = _native.load()
        need = lib.tmhd_linear_mxfp4_workspace_bytes(m, n, k)
        # from the caching allocator each time: ordered with its stream, and a captured graph's own
        ws = torch.empty(need, dtype=torch.uint8, device=device) if need else None
        status = lib.tmhd_linear_mxfp4(
            out.data_ptr(), rows.data_ptr(), weight.data_ptr(), weight_scale.data_ptr(), bias_at, m, n, k, stride,
            weight.stride(0) if n > 1 else k // 2, n, ws.data_ptr() if need else None, need,
            _native.stream_ptr(torch, device),
        )
    _native.check(status, "tmhd_linear_mxfp4")
    return out
