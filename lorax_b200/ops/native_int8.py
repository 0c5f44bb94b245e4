"""Bindings of the operators of layers in 8-bit integers: `csrc/kernels/norm_block.cu`, `int8_rows.cu` and `gemm_int8.cu`.  Imported into
:mod:`lorax_b200.ops.native`; `reference` states what they compute.

Arguments that do not fit raise ValueError in front of any launch.  Outputs are allocated by the call, on the current stream of the tensors' device, whichever
device is the current one; there is no scratch, so that calls on several streams, and captured graphs, share nothing."""

from __future__ import annotations

import struct
from ctypes import c_char_p, c_int, c_void_p
from typing import Optional, Union

import torch

from . import native as nv
from .reference import (INT8_MAX_K, NORM_BLOCK_MAX_WIDTH, Int8Rows, check_act_mul_int8, check_gemm_int8, check_norm_block, check_quant_rows_int8,
                        empty_int8_rows)

P, I, B = c_void_p, c_int, c_char_p

SIGNATURES = {
    "lx_norm_block_max_width": ([], I),
    "lx_norm_block_bytes": ([], I),
    "lx_norm_block": ([B], I),
    "lx_rows_int8_bytes": ([], I),
    "lx_rows_int8": ([B], I),
    "lx_gemm_int8_max_k": ([], I),
    "lx_gemm_int8_plan": ([I, I, I, I, P, P], I),
    "lx_gemm_int8_clusters": ([I], I),
    "lx_gemm_int8_bytes": ([], I),
    "lx_gemm_int8": ([B], I),
}

# The launchers' arguments, in the order of the structs of the same names (LxNormBlockArgs ... in csrc/kernels): whole numbers and addresses, then the norm's numbers.
_NORM = struct.Struct("25q3d")
_ROWS = struct.Struct("15q")
_GEMM = struct.Struct("17q")


def check_limits(lib):
    for name, here in (("lx_norm_block_max_width", NORM_BLOCK_MAX_WIDTH), ("lx_gemm_int8_max_k", INT8_MAX_K), ("lx_norm_block_bytes", _NORM.size),
                       ("lx_rows_int8_bytes", _ROWS.size), ("lx_gemm_int8_bytes", _GEMM.size)):
        said = getattr(lib, name, None)           # (a subset of the library may lack these operators)
        if said is not None and said() != here:
            raise nv.NativeError(f"{name}: C++ says {said()}, Python says {here}")


_devices = {}


def _device(at: int):
    """(SMs, status words' address) of a device, which live as long as its workspace."""
    known = _devices.get(at)
    if known is None:
        ws = nv.workspace(torch.device("cuda", at))
        known = _devices[at] = (ws.num_sms, ws.status.data_ptr())
    return known


def _on(t: torch.Tensor, call, *args):
    """`call` with `t`'s device as the current one: launches go to the current device."""
    at = t.get_device()
    if at < 0:
        raise ValueError(f"tensors on {t.device}: the kernels take those of a CUDA device")
    if at == torch._C._cuda_getDevice():
        return call(at, torch._C._cuda_getCurrentRawStream(at), *args)
    with torch.cuda.device(at):
        return call(at, torch._C._cuda_getCurrentRawStream(at), *args)


def _rows(at: int, stream: int, x: torch.Tensor, ldx: int, T: int, n: int, act: int, gated: bool, out: Optional[torch.Tensor], ring: int = -1) -> Int8Rows:
    """`ring` as for `_norm_block`."""
    r = empty_int8_rows(T, n, x)
    if T:
        sms, status = _device(at)
        q, scale = r
        rc = nv.load().lx_rows_int8(_ROWS.pack(x.data_ptr(), ldx, q.data_ptr(), (n + 15) // 16 * 16, scale.data_ptr(), 0 if out is None else out.data_ptr(),
                                               0 if out is None else out.stride(0), T, n, act, gated, status, sms, ring, stream))
        nv._check(rc, "lx_rows_int8")
    return r


def quant_rows_int8(x: torch.Tensor) -> Int8Rows:
    """Rows x [T, K] in 8-bit integers, with a scale for each row (`reference.quant_rows_int8` states the numbers)."""
    T, K, ldx = check_quant_rows_int8(x)
    if x.dtype != torch.bfloat16:
        raise ValueError(f"quant_rows_int8: the kernels are bf16; got {x.dtype}")
    return _on(x, _rows, x, ldx, T, K, -1, False, None)


def act_mul_int8(x: torch.Tensor, inter: int, act: str = "silu", gated: bool = True, out: Optional[torch.Tensor] = None) -> Int8Rows:
    """act(gate) * up of rows [gate | up], or act(gate), in 8-bit integers with a scale for each row; `out` takes the values in bf16 too
    (`reference.act_mul_int8`)."""
    T, ldx = check_act_mul_int8(x, inter, act, gated, out)
    if x.dtype != torch.bfloat16:
        raise ValueError(f"act_mul_int8: the kernels are bf16; got {x.dtype}")
    return _on(x, _rows, x, ldx, T, inter, nv._ACTS[act], bool(gated), out)


def norm_block(y: Optional[torch.Tensor], residual: torch.Tensor, weight: torch.Tensor, eps: float, post_weight: Optional[torch.Tensor] = None,
               gate: Optional[torch.Tensor] = None, scale: float = 1.0, bias: Optional[torch.Tensor] = None, post_bias: Optional[torch.Tensor] = None,
               weight_offset: float = 0.0, layernorm: bool = False, residual_out: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
               int8: bool = False) -> Union[torch.Tensor, Int8Rows]:
    """Norms on both sides of a block with its gate and scale, the residual stream between them, in one pass (`reference.norm_block` states them)."""
    checked = check_norm_block(y, residual, weight, post_weight, gate, scale, bias, post_bias, residual_out, out, int8)
    if residual.dtype != torch.bfloat16:
        raise ValueError(f"norm_block: the kernels are bf16; got {residual.dtype}")
    return _on(residual, _norm_block, checked, eps, scale, weight_offset, layernorm, out, int8)


_NONE = (0, 0, None, 0)


def _norm_block(at: int, stream: int, checked, eps: float, scale: float, weight_offset: float, layernorm: bool, out, int8: bool, ring: int = -1):
    """`ring`: 0 or 1 in place of the library's choice between a block per row and blocks that stay, to measure and test each."""
    T, H, gate, to, spans = checked              # (gate: its strides)
    get = spans.get
    residual = spans["residual"]
    q = q_scale = 0
    if int8:
        r = empty_int8_rows(T, H, residual[2])
        q, q_scale = r.q.data_ptr(), r.scale.data_ptr()
        o, _, _, ldo = get("out", _NONE)
    elif out is None:
        r = residual[2].new_empty_strided((T, H), (H, 1))
        o, ldo = r.data_ptr(), H
    else:
        r = out
        o, _, _, ldo = spans["out"]
    if T:
        y = get("y", _NONE)
        h = _NONE if to is None else get("residual_out", residual)
        sms, status = _device(at)
        rc = nv.load().lx_norm_block(_NORM.pack(y[0], y[3], residual[0], residual[3], h[0], h[3], get("post_weight", _NONE)[0], get("post_bias", _NONE)[0],
                                                spans["weight"][0], get("bias", _NONE)[0], get("gate", _NONE)[0], gate[0],
                                                gate[1], o, ldo, q, (H + 15) // 16 * 16, q_scale, T, H, bool(layernorm),
                                                status, sms, ring, stream, eps, weight_offset, scale))
        nv._check(rc, "lx_norm_block")
    return r


def gemm_int8(x: Int8Rows, w: torch.Tensor, w_scale: torch.Tensor, bias: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
              dtype: torch.dtype = torch.bfloat16, w_const: bool = False) -> torch.Tensor:
    """out[T, N] = (x.q @ w^T) * w_scale[n] * x.scale[t] + bias[n], the sums whole numbers, rounded to bf16 once (`reference.gemm_int8`).  `w_const` as for `gemm`: the
    kernel in front on the stream does not write `w`.  Rows of a result that the call allocates lie a multiple of 16 bytes apart."""
    sizes = check_gemm_int8(x, w, w_scale, bias, out, dtype)
    if dtype != torch.bfloat16:
        raise ValueError(f"gemm_int8: the kernels are bf16; got {dtype}")
    return _on(w, _gemm_int8, x, w, w_scale, bias, out, sizes, w_const)


def _gemm_int8(at: int, stream: int, x: Int8Rows, w, w_scale, bias, out, sizes, w_const: bool, plan=None):
    """`plan`: (by pairs of CTAs, token tile, parts of K) in place of the library's choice, to measure and test each."""
    T, N, K, ldq, ldw = sizes
    if out is None:
        # (rows of a multiple of 8: written 16 bytes at a time, over thousands of rows up to twice as quick as rows that begin anywhere)
        ldo = (N + 7) // 8 * 8
        out = w.new_empty_strided((T, N), (ldo, 1), dtype=torch.bfloat16)
    else:
        ldo = out.stride(0) if T > 1 else N
    if T and N:
        sms, status = _device(at)
        q, scale = x
        rc = nv.load().lx_gemm_int8(_GEMM.pack(q.data_ptr(), ldq, scale.data_ptr(), w.data_ptr(), ldw, w_scale.data_ptr(), 0 if bias is None else bias.data_ptr(),
                                               out.data_ptr(), ldo, T, N, K, bool(w_const), status, sms,
                                               0 if plan is None else 1 + int(plan[0]) + 2 * (plan[2] | plan[1] << 8), stream))
        nv._check(rc, "lx_gemm_int8")
    return out
