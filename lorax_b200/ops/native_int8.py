"""Bindings of the operators of layers in 8-bit integers: `csrc/kernels/norm_block.cu`, `int8_rows.cu` and `gemm_int8.cu`.  Imported into
:mod:`lorax_b200.ops.native`; `reference` states what they compute.

Arguments that do not fit raise ValueError in front of any launch.  Outputs are allocated by the call, on the current stream of the tensors' device, whichever
device is the current one; there is no scratch, so that calls on several streams, and captured graphs, share nothing."""

from __future__ import annotations

from ctypes import c_float, c_int, c_longlong, c_void_p
from typing import Optional, Union

import torch

from . import native as nv
from .native_steps import _on_its_device, _stream_of
from .reference import (INT8_MAX_K, NORM_BLOCK_MAX_WIDTH, Int8Rows, check_act_mul_int8, check_gemm_int8, check_norm_block, check_quant_rows_int8,
                        empty_int8_rows)

P, I, L, F = c_void_p, c_int, c_longlong, c_float

SIGNATURES = {
    "lx_norm_block_max_width": ([], I),
    "lx_norm_block": ([P, L, P, L, P, L, P, P, P, P, P, L, I, P, L, P, L, P, I, I, F, F, F, I, P, I, I, P], I),
    "lx_rows_int8": ([P, L, P, L, P, P, L, I, I, I, I, I, P], I),
    "lx_gemm_int8_max_k": ([], I),
    "lx_gemm_int8_plan": ([I, I, I, I, P, P], I),
    "lx_gemm_int8_clusters": ([I], I),
    "lx_gemm_int8": ([P, L, P, P, L, P, P, P, L, I, I, I, I, P, I, I, P], I),
}


def check_limits(lib):
    for name, here in (("lx_norm_block_max_width", NORM_BLOCK_MAX_WIDTH), ("lx_gemm_int8_max_k", INT8_MAX_K)):
        said = getattr(lib, name, None)           # (a subset of the library may lack these operators)
        if said is not None and said() != here:
            raise nv.NativeError(f"{name}: C++ says {said()}, Python says {here}")


def _bf16(op: str, t: torch.Tensor):
    if t.dtype != torch.bfloat16:
        raise ValueError(f"{op}: the kernels are bf16; got {t.dtype}")


_devices = {}


def _device(at: int):
    """(SMs, status words' address) of a device, which live as long as its workspace."""
    known = _devices.get(at)
    if known is None:
        ws = nv.workspace(torch.device("cuda", at))
        known = _devices[at] = (ws.num_sms, ws.status.data_ptr())
    return known


def _pitch(t: Optional[torch.Tensor]) -> int:
    """Elements between two rows (one row's own stride says nothing)."""
    return 0 if t is None else t.stride(0) if t.shape[0] > 1 else (t.shape[1] + 15) // 16 * 16


def _rows(x: torch.Tensor, T: int, n: int, act: int, gated: bool, out: Optional[torch.Tensor]) -> Int8Rows:
    stream = _stream_of(x)
    r = empty_int8_rows(T, n, x.device)
    if T:
        rc = nv.load().lx_rows_int8(x.data_ptr(), _pitch(x), r.q.data_ptr(), _pitch(r.q), r.scale.data_ptr(), nv._ptr(out), _pitch(out), T, n, act,
                                    int(gated), _device(x.get_device())[0], stream)
        nv._check(rc, "lx_rows_int8")
    return r


@_on_its_device
def quant_rows_int8(x: torch.Tensor) -> Int8Rows:
    """Rows x [T, K] in 8-bit integers, with a scale for each row (`reference.quant_rows_int8` states the numbers)."""
    T, K = check_quant_rows_int8(x)
    _bf16("quant_rows_int8", x)
    return _rows(x, T, K, -1, False, None)


@_on_its_device
def act_mul_int8(x: torch.Tensor, inter: int, act: str = "silu", gated: bool = True, out: Optional[torch.Tensor] = None) -> Int8Rows:
    """act(gate) * up of rows [gate | up], or act(gate), in 8-bit integers with a scale for each row; `out` takes the values in bf16 too
    (`reference.act_mul_int8`)."""
    T = check_act_mul_int8(x, inter, act, gated, out)
    _bf16("act_mul_int8", x)
    return _rows(x, T, inter, nv._ACTS[act], gated, out)


def norm_block(y: Optional[torch.Tensor], residual: torch.Tensor, weight: torch.Tensor, eps: float, post_weight: Optional[torch.Tensor] = None,
               gate: Optional[torch.Tensor] = None, scale: float = 1.0, bias: Optional[torch.Tensor] = None, post_bias: Optional[torch.Tensor] = None,
               weight_offset: float = 0.0, layernorm: bool = False, residual_out: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
               int8: bool = False) -> Union[torch.Tensor, Int8Rows]:
    """Norms on both sides of a block with its gate and scale, the residual stream between them, in one pass (`reference.norm_block` states them)."""
    T, H, gate, to = check_norm_block(y, residual, weight, post_weight, gate, scale, bias, post_bias, residual_out, out, int8)
    _bf16("norm_block", residual)
    return _norm_block(residual, y, weight, eps, post_weight, gate, scale, bias, post_bias, weight_offset, layernorm, to, out, int8)


@_on_its_device
def _norm_block(residual, y, weight, eps, post_weight, gate, scale, bias, post_bias, weight_offset, layernorm, to, out, int8, ring=-1):
    T, H = residual.shape
    stream = _stream_of(residual)
    if out is None and not int8:
        out = torch.empty(T, H, dtype=residual.dtype, device=residual.device)
    r = empty_int8_rows(T, H, residual.device) if int8 else None
    if T:
        q, q_scale = r if int8 else (None, None)
        sms, status = _device(residual.get_device())
        rc = nv.load().lx_norm_block(nv._ptr(y), _pitch(y), residual.data_ptr(), _pitch(residual), nv._ptr(to), _pitch(to), nv._ptr(post_weight),
                                     nv._ptr(post_bias), weight.data_ptr(), nv._ptr(bias), nv._ptr(gate), 0 if gate is None or T == 1 else gate.stride(0),
                                     0 if gate is None or H == 1 else gate.stride(1), nv._ptr(out), _pitch(out), nv._ptr(q), _pitch(q), nv._ptr(q_scale),
                                     T, H, eps, weight_offset, scale, int(layernorm), status, sms, ring, stream)
        nv._check(rc, "lx_norm_block")
    return r if int8 else out


def gemm_int8(x: Int8Rows, w: torch.Tensor, w_scale: torch.Tensor, bias: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
              dtype: torch.dtype = torch.bfloat16, w_const: bool = False) -> torch.Tensor:
    """out[T, N] = (x.q @ w^T) * w_scale[n] * x.scale[t] + bias[n], the sums whole numbers, rounded to bf16 once (`reference.gemm_int8`).  `w_const` as for `gemm`: the
    kernel in front on the stream does not write `w`."""
    check_gemm_int8(x, w, w_scale, bias, out, dtype)
    if dtype != torch.bfloat16:
        raise ValueError(f"gemm_int8: the kernels are bf16; got {dtype}")
    return _gemm_int8(x.q, x.scale, w, w_scale, bias, out, w_const)


@_on_its_device
def _gemm_int8(q, scale, w, w_scale, bias, out, w_const, plan=None):
    """`plan`: (by pairs of CTAs, token tile, parts of K) in place of the library's choice, to measure and test each."""
    (T, K), N = q.shape, w.shape[0]
    stream = _stream_of(q)
    if out is None:
        out = torch.empty(T, N, dtype=torch.bfloat16, device=q.device)
    if T and N:
        sms, status = _device(q.get_device())
        force = 0 if plan is None else 1 + int(plan[0]) + 2 * (plan[2] | plan[1] << 8)
        rc = nv.load().lx_gemm_int8(q.data_ptr(), _pitch(q), scale.data_ptr(), w.data_ptr(), _pitch(w), w_scale.data_ptr(), nv._ptr(bias), out.data_ptr(),
                                    out.stride(0) if T > 1 else N, T, N, K, int(w_const), status, sms, force, stream)
        nv._check(rc, "lx_gemm_int8")
    return out
