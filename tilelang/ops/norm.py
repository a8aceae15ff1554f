"""Fused RMSNorm (reference counterpart: examples/norm/rms_norm.py and the model's ``RMSNorm``), and
its form in front of the block-scaled fp8 GEMMs: residual addition, norm and e4m3 quantisation in one pass."""
from __future__ import annotations

import functools
from typing import NamedTuple, Optional

import torch

import tilelang
import tilelang.language as T
from tilelang import _native


@functools.lru_cache(maxsize=None)
def _rms_kernel_padded(M, N, dtype, eps, target, threads=128):
    """Widths that do not tile over the block (e.g. 3200): one row per workgroup, the row padded
    to a multiple of 4 * threads in registers, masked loads and stores."""
    Np = -(-N // (4 * threads)) * (4 * threads)

    @T.prim_func
    def main(X: T.Tensor((M, N), dtype), Wt: T.Tensor((N, ), dtype), Y: T.Tensor((M, N), dtype)):
        with T.Kernel(M, threads=threads) as bx:
            x = T.alloc_fragment((Np, ), "float32")
            sq = T.alloc_fragment((Np, ), "float32")
            ss = T.alloc_fragment((1, ), "float32")
            for j in T.Parallel(Np):
                x[j] = T.if_then_else(j < N, T.Cast("float32", X[bx, T.min(j, N - 1)]), 0.0)
                sq[j] = x[j] * x[j]
            T.reduce_sum(sq, ss, dim=0)
            for j in T.Parallel(Np):
                if j < N:
                    Y[bx, j] = T.Cast(dtype, x[j] * T.rsqrt(ss[0] / N + eps) * T.Cast("float32", Wt[j]))

    return tilelang.compile(main, out_idx=[-1], target=target)


@functools.lru_cache(maxsize=None)
def _rms_kernel(M, N, dtype, eps, target):
    if N % 1024:
        return _rms_kernel_padded(M, N, dtype, eps, target)
    blk_m = 4 if N <= 8192 else 1
    threads = 256

    @T.prim_func
    def main(X: T.Tensor((M, N), dtype), Wt: T.Tensor((N, ), dtype), Y: T.Tensor((M, N), dtype)):
        with T.Kernel(T.ceildiv(M, blk_m), threads=threads) as bx:
            x = T.alloc_fragment((blk_m, N), "float32")
            sq = T.alloc_fragment((blk_m, N), "float32")
            ss = T.alloc_fragment((blk_m, ), "float32")
            y = T.alloc_fragment((blk_m, N), dtype)
            T.copy(X[bx * blk_m, 0], x)
            for i, j in T.Parallel(blk_m, N):
                sq[i, j] = x[i, j] * x[i, j]
            T.reduce_sum(sq, ss, dim=1)
            for i in T.Parallel(blk_m):
                ss[i] = T.rsqrt(ss[i] / N + eps)
            for i, j in T.Parallel(blk_m, N):
                y[i, j] = x[i, j] * ss[i] * Wt[j]
            T.copy(y, Y[bx * blk_m, 0])

    return tilelang.compile(main, out_idx=[-1], target=target)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    shp = x.shape
    x2 = x.reshape(-1, shp[-1]).contiguous()
    M, N = x2.shape
    dt = {torch.float16: "float16", torch.bfloat16: "bfloat16", torch.float32: "float32"}[x2.dtype]
    k = _rms_kernel(M, N, dt, float(eps), "cpu" if x2.device.type == "cpu" else "hip")
    return k(x2, weight.to(x2.dtype).contiguous()).reshape(shp)


class NormQuant(NamedTuple):
    """What ``add_rms_norm_quant`` returns; ``h`` and ``y`` are None where they were not asked for."""
    q: torch.Tensor  # float8_e4m3fn, as x
    scale: torch.Tensor  # float32 [..., N / group]
    h: Optional[torch.Tensor]  # x + residual, in x's type
    y: Optional[torch.Tensor]  # the normalised row, in x's type


def add_rms_norm_quant(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None,
                       eps: float = 1e-6, group: int = 128, pow2_scale: bool = False,
                       return_norm: bool = False) -> NormQuant:
    """h = x + residual, y = rms_norm(h) * weight, and y in e4m3 with one scale for every ``group`` values:

        scale = max(max |y|, 1e-4) / 448, or the next power of two (``pow2_scale``);  q = e4m3(y / scale)

    the operand format of ``fp8_gemm`` for ``group=128``. ``group=0``: one scale for each row; otherwise a power of
    two from 16 to 512 that divides the row. x [..., N] in bf16, fp16 or fp32 (N up to 65536) with weight [N] and
    residual of its type. Sums and norms are float32 throughout: the codes come from the y that was not rounded to
    x's type (``rms_norm`` followed by ``act_quant`` rounds it in between). ``h`` is returned if a residual is
    given, ``y`` with ``return_norm``. A row with a not-a-number has not-a-number codes; one whose squares sum to
    more than float32 holds (an infinite element, say) has zeros, and not-a-number at an infinite element. No
    derivative: inputs that require a gradient or carry a tangent are refused while gradients are on.
    """
    return NormQuant(*_native.ops().add_rms_norm_quant(x, weight, residual, eps, group, pow2_scale, return_norm))
