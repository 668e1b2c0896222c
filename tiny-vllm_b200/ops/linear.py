"""x . W^T for the parts, by storage dtype.

float32: the package's own kernels, true 32-bit: up to F32_CORE_ROWS rows and narrow products on the float32 cores, the others
on the tensor cores with every operand as three bfloat16.  Each of the two gives a row the same bits whatever else is in the
batch, but not each other's: a row's last bits change between 32 and 33 rows and wherever else the kernel does.
bfloat16: the tensor-core kernels of this package where they take the shape,
else cuBLAS through ``torch.nn.functional.linear``, which is what the
reference's engine calls for every projection (tinyvllm/layers.py:84-85).
"""

from __future__ import annotations

import functools
import os

import torch

from . import kernels


def linear(x: torch.Tensor, weight: torch.Tensor, *, out_dtype: torch.dtype | None = None,
           out: torch.Tensor | None = None, weight_constant: bool = False) -> torch.Tensor:
    """x [m, k] times weight [n, k] transposed; the result has ``out_dtype``
    (default: the dtype of x).  ``weight_constant``: nothing in flight on the stream writes the weight (a model's, loaded
    long ago), so that float32 products may read it while the kernel before them still runs.  (bfloat16 products of few
    rows always do.)"""
    if not x.is_cuda:
        raise kernels.KernelError("linear runs on CUDA tensors only; there is no CPU path")
    out_dtype = out_dtype or x.dtype
    if x.dtype == torch.float32:
        if out_dtype != torch.float32:
            raise kernels.KernelError("a float32 product has a float32 result")
        return _linear_f32(x, weight, out, weight_constant)
    from . import gemm

    return gemm.linear_bf16(x, weight, out_dtype=out_dtype, out=out)


# Rows up to which a float32 product stays on the float32 cores: the tensor-core kernel takes 25 to 28 us for a layer's
# products at any number of rows up to 128 (a CTA walks 1,024 k in 16 steps of 1.2 us), the float32 cores 16 to 24 us
# for 32 rows, 29 to 42 us for 48.
F32_CORE_ROWS = 32
# Smallest k of the tensor cores.  Their error against 64 bits is larger below (operands of either sign, k = 4 / 8 / 16: 4.9e-8,
# 4.9e-8, 5.0e-8; float32 cores 4.1e-8, 4.8e-8, 6.0e-8).
F32_TENSOR_K = 16


@functools.lru_cache(maxsize=4096)
def _tensor_cores_are_quicker(rows: int, columns: int, k: int) -> bool:
    """Whether the tensor cores take a float32 product of more than F32_CORE_ROWS rows, by the two kernels' estimates.  The
    float32 cores are quicker where one round of their tiles holds all of a narrow or short product: splitting x, a launch
    more, and columns up to 128 are then not paid back.  Measured (us, float32 cores / tensor cores): 301 x 512 x 64 5.3 /
    6.3, 8,192 x 128 x 64 7.6 / 15.2, 2,048 x 64 x 2,048 29 / 34, 8,192 x 64 x 4,096 127 / 176; but 301 x 64 x 512 27 /
    15, 677 x 128 x 1,024 28.7 / 27.0, 2,048 x 256 x 2,048 76 / 35."""
    return k >= F32_TENSOR_K and kernels.gemm_f32_tc_us(rows, columns, k) < kernels.gemm_f32_us(rows, columns, k)


def _linear_f32(x: torch.Tensor, weight: torch.Tensor, out: torch.Tensor | None, weight_constant: bool) -> torch.Tensor:
    # (an ``out`` that is larger than the result, or of another type, is written by the float32 cores' kernels alone)
    if (x.dim() == 2 and x.shape[0] > F32_CORE_ROWS and kernels.gemm_f32_tc_takes(x, weight)
            and (out is None or (out.dtype == torch.float32 and out.shape == (x.shape[0], weight.shape[0])))
            and _tensor_cores_are_quicker(x.shape[0], weight.shape[0], x.shape[1])):
        return kernels.gemm_f32_tc(x, weight, out=out, weight_constant=weight_constant)
    return kernels.gemm_nt_simt(x, weight, out=out, weight_constant=weight_constant)


def _projection_f32(x: torch.Tensor, weight: torch.Tensor, out: torch.Tensor | None, weight_constant: bool) -> torch.Tensor:
    """:func:`linear` of bfloat16 operands with a float32 result that has not passed through bfloat16.  More than 256 rows of a k that is
    no multiple of 8, or of a weight whose rows are not contiguous, do so there (and fewer of the latter are refused): here k is filled
    up with zeros, which add nothing, for the library's product with a float32 result (1,025 x 3,537 x 1,096: 54 us and 4e-6 off on the whole, 96 us and 0.0023 there; the float32
    cores 437 us)."""
    k = x.shape[1]
    if x.stride(1) == 1 and weight.stride(1) == 1 and (x.shape[0] <= 256 or k % 8 == 0):
        return linear(x, weight, out_dtype=torch.float32, out=out, weight_constant=weight_constant)
    if k % 8:
        x, weight = (torch.nn.functional.pad(t, (0, -k % 8)) for t in (x, weight))
    result = torch.mm(x, weight.t(), out_dtype=torch.float32)
    return result if out is None else out.copy_(result)


def linear_adapted(x: torch.Tensor, weight: torch.Tensor, down: torch.Tensor, up: torch.Tensor, ids: torch.Tensor,
                   scales: torch.Tensor | None = None, *, out_dtype: torch.dtype | None = None,
                   out: torch.Tensor | None = None, weight_constant: bool = False) -> torch.Tensor:
    """:func:`linear` with a low-rank adapter of each row's own: row t of the result is x[t] W^T + s (x[t] A^T) B^T with
    A = ``down[ids[t]]`` ([adapters, rank, k]), B = ``up[ids[t]]`` ([adapters, n, rank]), s = ``scales[ids[t]]`` (float32
    [adapters]; None: 1).  ``ids`` (int32 [m]) may come in any order; a row whose number names no adapter (-1) has the
    projection alone.  Adapters of lower rank are filled up with zeros; ranks up to 256.

    x A^T is summed in float32 and kept to 2^-16 of itself (two bfloat16; float32 operands: float32).  The adapter's part is added to
    the projection as :func:`linear` gives it, rounded to bfloat16 where the result is (a row without an adapter is then bit for bit
    what :func:`linear` makes of it), and the sum is rounded to the result's type: two roundings of a bfloat16 result.  The projection
    stays float32 in between where the result is, and where n is no multiple of 8; ``out_dtype=torch.float32`` is the way to one
    rounding of one's own.

    Rows whose adapters lie together go fastest; up to 512 they may as well come in any order."""
    x_shape, weight_shape, down_shape, dtype = x.shape, weight.shape, down.shape, x.dtype
    if len(x_shape) != 2 or len(weight_shape) != 2 or x_shape[1] != weight_shape[1] or weight.dtype != dtype or x_shape[1] < 1:
        raise kernels.KernelError("linear_adapted wants x [m, k] and a weight [n, k] of its type")
    (m, k), n = x_shape, weight_shape[0]
    kernels.dtype_tag(dtype)
    adapters, rank = (down_shape[0], down_shape[1]) if len(down_shape) == 3 else (0, 0)
    if not kernels._is(down, dtype, adapters, rank, k) or not kernels._is(up, dtype, adapters, n, rank) or adapters < 1 \
            or not 1 <= rank <= kernels.ADAPTERS_MAX_RANK:
        raise kernels.KernelError(f"linear_adapted: down and up must be contiguous [adapters, rank, {k}] and [adapters, {n}, rank] "
                                  f"of the type of x, at least one adapter, ranks from 1 to {kernels.ADAPTERS_MAX_RANK}")
    if not kernels._is(ids, torch.int32, m):
        raise kernels.KernelError(f"linear_adapted: ids must be contiguous int32 [{m}]")
    if scales is not None and not kernels._is(scales, torch.float32, adapters):
        raise kernels.KernelError(f"linear_adapted: scales must be contiguous float32 [{adapters}]")
    if x.stride()[1] != 1 and k > 1:
        raise kernels.KernelError("linear_adapted: the rows of x must be contiguous")
    if m > kernels.ADAPTERS_MAX_ROWS:
        raise kernels.KernelError(f"linear_adapted takes up to {kernels.ADAPTERS_MAX_ROWS} rows")
    out_dtype = out_dtype or (dtype if out is None else out.dtype)
    if out_dtype != dtype and out_dtype != torch.float32:
        raise kernels.KernelError("linear_adapted: the result has the type of x, or float32")
    if out is not None and (out.shape != (m, n) or out.dtype != out_dtype or out.stride(1) != 1 and n > 1
                            or m > 1 and out.stride(0) < n or kernels._overlaps(out, x, weight, down, up, ids, scales)):
        raise kernels.KernelError(f"linear_adapted: out must be {out_dtype} [{m}, {n}] with contiguous rows, in memory of its own")
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or down.requires_grad or up.requires_grad
                                    or scales is not None and scales.requires_grad or out is not None and out.requires_grad):
        raise kernels.KernelError("linear_adapted has no backward pass: call it under torch.no_grad() or torch.inference_mode()")
    stream = kernels._here("linear_adapted", x, weight, down, up, ids, scales, out)
    if m == 0 or n == 0:
        return torch.empty((m, n), dtype=out_dtype, device=x.device) if out is None else out
    if out_dtype == torch.bfloat16 and n % 8:
        # The library sums such products in pieces that it rounds to bfloat16 (262 x 3,536 x 1,097: 0.0029 off on the whole, one
        # rounding is 0.0017 off), and takes no longer for a float32 result (80 us either way, 2,471 x 1,920 x 2,524 105 and 108).
        y = _projection_f32(x, weight, None, weight_constant)
        out = torch.empty((m, n), dtype=out_dtype, device=x.device) if out is None else out
    elif out_dtype != dtype:                    # float32 of bfloat16 operands
        y = out = _projection_f32(x, weight, out, weight_constant)
    else:
        # As `linear` rounds it: rows without an adapter keep their bits, and y passes half the bytes.  With y in float32 the result is
        # 0.0017 off 64 bits on the whole, one rounding, else 0.0021 to 0.0023; us with it / as here: 48 rows 4096 -> 6144 22.8 / 22.0,
        # 4,099 rows 4096 -> 4096 of rank 64 216 / 122.
        y = out = linear(x, weight, out_dtype=out_dtype, out=out, weight_constant=weight_constant)
    kernels.add_adapters(y, x, down, up, ids, scales, out, stream)
    return out


def linear_silu(x: torch.Tensor, gate_up_weight: torch.Tensor, *, weight_constant: bool = False) -> torch.Tensor:
    """round(round(silu(x . gate^T)) * (x . up^T)) for a packed [gate | up] weight, [m, inter].  ``weight_constant``: as in
    :func:`linear`."""
    if not x.is_cuda:
        raise kernels.KernelError("linear_silu runs on CUDA tensors only; there is no CPU path")
    if x.dtype == torch.float32:
        return kernels.silu_mul(_linear_f32(x, gate_up_weight, None, weight_constant))
    from . import gemm

    return gemm.linear_silu_bf16(x, gate_up_weight)


# Every CTA of the fused kernel reads all rows of the input to normalise them for itself; beyond
# a few rows those reads cost more (in L2 bandwidth) than the separate norm kernel they replace.
FUSED_NORM_MAX_ROWS = int(os.environ.get("TINYVLLM_B200_FUSED_NORM_ROWS", "2"))


# TINYVLLM_B200_STREAM_ADD=0: output projections never add to the stream themselves (the norm kernel
# runs between every two products), for comparison
STREAM_ADD = os.environ.get("TINYVLLM_B200_STREAM_ADD", "1") != "0"


def linear_into_stream(x: torch.Tensor, weight: torch.Tensor, stream: torch.Tensor, *, weight_constant: bool = False):
    """A part's output projection, added to the residual stream where that saves a kernel.  ``weight_constant``: as in
    :func:`linear`.

    Returns (None, stream + linear(x, weight)) when the product's kernel does the addition on its
    way out (small bfloat16 batches): the new stream then carries ``row_squares``, the sums of
    squares of its rows tile by tile, with which :func:`linear_norm` applies the next pre-norm
    inside the next product, so that no norm kernel runs between the two (there the norm weight
    multiplies the stream before the product and the inverse RMS the sums after it: one rounding
    where the norm kernel has two).  Otherwise
    (linear(x, weight), stream), and the next norm adds the two as usual."""
    from . import gemm

    if (STREAM_ADD and x.dtype == torch.bfloat16 and weight.dtype == torch.bfloat16 and stream is not None
            and stream.dtype == torch.bfloat16 and stream.is_contiguous() and gemm.small(x, weight)
            and stream.shape == (x.shape[0], weight.shape[0])):
        summed, squares = kernels.gemm_small_m(x, weight, kernels.GEMM_BF16, add_stream=stream,
                                               prefetch=gemm.next_weight(weight))
        summed.row_squares = squares
        return None, summed
    return linear(x, weight, weight_constant=weight_constant), stream


def linear_norm(hidden: torch.Tensor | None, residual: torch.Tensor | None, norm, weight: torch.Tensor, *,
                silu: bool = False, weight_constant: bool = False):
    """(linear(norm(hidden + residual), weight), hidden + residual): a pre-norm and the
    projection behind it as one operation.  ``norm`` is a norm part (``weight``, ``eps``,
    ``forward``, ``add``).  Without a residual the stream is ``hidden`` itself; without
    ``hidden`` (None) the residual holds the sum already (:func:`linear_into_stream`).  ``silu``
    applies SiLU(gate) * up to a packed [gate | up] weight.  Small bfloat16 batches run as
    one kernel; everything else as the norm kernel and the product.  ``weight_constant``: as in
    :func:`linear`."""
    from . import gemm

    if hidden is None:
        squares = getattr(residual, "row_squares", None)
        if (squares is not None and weight.dtype == torch.bfloat16 and getattr(norm, "folds_into_product", False)
                and gemm.small(residual, weight) and residual.is_contiguous()
                and norm.weight.data_ptr() % 16 == 0):
            mode = kernels.GEMM_SILU if silu else kernels.GEMM_BF16
            out = kernels.gemm_small_m(residual, weight, mode, norm_weight=norm.weight, eps=norm.eps,
                                       row_squares=squares, prefetch=gemm.next_weight(weight))
            return out, residual
        x = norm.forward(residual)
        return (linear_silu if silu else linear)(x, weight, weight_constant=weight_constant), residual
    if (hidden.dtype == torch.bfloat16 and weight.dtype == torch.bfloat16 and hidden.is_contiguous()
            and getattr(norm, "folds_into_product", False) and gemm.small(hidden, weight)
            and hidden.shape[0] <= FUSED_NORM_MAX_ROWS and (residual is None or residual.data_ptr() % 16 == 0)
            and kernels.gemm_small_m_takes_norm(hidden.shape[0], hidden.shape[1])):
        mode = kernels.GEMM_SILU if silu else kernels.GEMM_BF16
        out, stream = kernels.gemm_small_m(hidden, weight, mode, norm_weight=norm.weight,
                                           residual=residual, eps=norm.eps,
                                           prefetch=gemm.next_weight(weight))
        return out, (hidden if residual is None else stream)
    if residual is None:
        x, stream = norm.forward(hidden), hidden
    else:
        x, stream = norm.add(hidden, residual)
    return (linear_silu if silu else linear)(x, weight, weight_constant=weight_constant), stream
