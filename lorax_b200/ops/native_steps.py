"""Bindings of the operators of short ragged steps: `csrc/kernels/step_tables.cu`, `moe_few.cu` and `token_scores.cu`.  Imported into
:mod:`lorax_b200.ops.native`; `reference` states what they compute.

Arguments that do not fit raise ValueError in front of any launch.  Outputs and scratch are allocated by the call, on the current stream of the tensors' device,
whichever device is the current one (calls on several streams, and captured graphs, share nothing)."""

from __future__ import annotations

import functools
from ctypes import c_float, c_int, c_longlong, c_void_p
from typing import Optional, Sequence, Tuple

import torch

from . import native as nv
from .reference import MOE_FEW_TOKENS, STEP_SEQS_MAX, TOP_MAX, StepTables, TokenScores, check_moe_few, check_step_tables, check_token_scores

P, I, L, F = c_void_p, c_int, c_longlong, c_float

SIGNATURES = {
    "lx_step_tables_max_seqs": ([], I),
    "lx_step_tables": ([P, L, P, I, I, I, I, I, I, I, P, P, I, P, I, I, I, P, P], I),
    "lx_moe_few_max_tokens": ([], I),
    "lx_moe_few_down_stages": ([I, I, I, I, I], I),
    "lx_moe_few": ([P, L, P, L, P, P, P, P, P, L, I, I, I, I, I, I, I, I, I, F, P, I, P], I),
    "lx_token_scores_max_top": ([], I),
    "lx_token_scores": ([P, L, I, I, I, P, I, I, F, P, P, P, P, P], I),
}


def check_limits(lib):
    for name, here in (("lx_step_tables_max_seqs", STEP_SEQS_MAX), ("lx_moe_few_max_tokens", MOE_FEW_TOKENS), ("lx_token_scores_max_top", TOP_MAX)):
        if getattr(lib, name)() != here:
            raise nv.NativeError(f"{name}: C++ says {getattr(lib, name)()}, Python says {here}")


def _on_its_device(op):
    """`op` with its first tensor's device as the current one: launches go to the current device.  (That the others are on the same one is among its checks.)"""
    name = op.__code__.co_varnames[0]

    @functools.wraps(op)
    def call(*args, **kw):
        t = args[0] if args else kw.get(name)
        at = t.get_device() if isinstance(t, torch.Tensor) else -1
        if at < 0 or at == torch._C._cuda_getDevice():
            return op(*args, **kw)
        with torch.cuda.device(at):
            return op(*args, **kw)
    return call


def _stream_of(t: torch.Tensor) -> int:
    at = t.get_device()
    if at < 0:
        raise ValueError(f"tensors on {t.device}: the kernels take those of a CUDA device")
    return torch._C._cuda_getCurrentRawStream(at)


@_on_its_device
def step_tables(seqs: torch.Tensor, pages: torch.Tensor, tokens: int, max_blocks: int, page: int, window: int = 0,
                tiles: Sequence[Tuple[int, int]] = (), lora_tiles: int = 0, lora_rows: int = 32, row_offset: int = 0,
                lead: Optional[torch.Tensor] = None) -> StepTables:
    """Tables of a ragged step from its sequences' lengths (`reference.step_tables` states them), in one launch."""
    B = check_step_tables(seqs, pages, tokens, max_blocks, page, window, tiles, lora_tiles, lora_rows, row_offset, lead)
    stream = _stream_of(seqs)
    M, n_lead, n_lists = max_blocks, 0 if lead is None else lead.shape[0], len(tiles)
    sizes = [4 * (n_lead + lora_tiles), B + 1, tokens, tokens, tokens, B * M]
    for _, n in tiles:
        sizes += (n, n)
    out = torch.empty(sum(sizes), dtype=torch.int32, device=seqs.device)
    heights, counts = (I * n_lists)(*[h for h, _ in tiles]), (I * n_lists)(*[n for _, n in tiles])
    rc = nv.load().lx_step_tables(seqs.data_ptr(), seqs.stride(0), pages.data_ptr(), pages.shape[0], B, tokens, M, page, window, row_offset, heights, counts,
                                  n_lists, None if lead is None else lead.data_ptr(), n_lead, lora_rows, lora_tiles, out.data_ptr(), stream)
    nv._check(rc, "lx_step_tables")
    lora, cu, pos, slots, tok, bt, *lists = out.split_with_sizes(sizes)
    return StepTables(cu, pos, slots, tok, bt.view(B, M), tuple(zip(lists[::2], lists[1::2])), lora.view(-1, 4))


@_on_its_device
def moe_few(x: torch.Tensor, router_w: torch.Tensor, w13: torch.Tensor, w2: torch.Tensor, k: int, e0: int = 0, act: str = "silu", renorm: bool = True,
            scale: float = 1.0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The mixture-of-experts feed-forward of up to `MOE_FEW_TOKENS` tokens (`reference.moe_few` states it; `moe_ffn` takes any number)."""
    T, E, H, inter = check_moe_few(x, router_w, w13, w2, k, e0, act, scale, out)
    if x.dtype != torch.bfloat16:
        raise ValueError(f"moe_few: the kernels are bf16; got {x.dtype}")
    stream = _stream_of(x)
    if out is None:
        out = torch.empty(T, H, dtype=x.dtype, device=x.device)
    if T == 0:
        return out
    # scratch: h (two planes), then the logits
    h_bytes = (4 * T * k * inter + 15) // 16 * 16
    scratch = torch.empty(h_bytes + 4 * T * E, dtype=torch.uint8, device=x.device)
    at, ws = scratch.data_ptr(), nv.workspace(x.device)
    rc = nv.load().lx_moe_few(x.data_ptr(), x.stride(0) if T > 1 else H, router_w.data_ptr(), router_w.stride(0) if E > 1 else H, w13.data_ptr(), w2.data_ptr(),
                              at + h_bytes, at, out.data_ptr(), out.stride(0), T, E, k, e0, w13.shape[0], H, inter, nv._ACTS[act], int(renorm), scale, ws.status.data_ptr(), ws.num_sms, stream)
    nv._check(min(rc, 0), "lx_moe_few")
    nv.launch_count += rc - 1            # (two or three)
    return out


@_on_its_device
def token_scores(logits: torch.Tensor, targets: Optional[torch.Tensor] = None, k: int = 0, softcap: float = 0.0,
                 entropy: bool = True) -> TokenScores:
    """Log-probability of a given token of every row, entropy of the row, and its `k` best tokens with their log-probabilities
    (`reference.token_scores` states them): one pass over the logits, one launch.  (`entropy` saves the kernel nothing.)"""
    T, V = check_token_scores(logits, targets, k, softcap)
    if logits.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"token_scores: the kernels take bf16 and fp32 logits; got {logits.dtype}")
    stream = _stream_of(logits)
    t_ptr = wide = 0
    if targets is not None:
        targets = targets.contiguous()
        t_ptr, wide = targets.data_ptr(), int(targets.dtype == torch.int64)
    lp, ent, best = torch.empty(T * (2 + k), dtype=torch.float32, device=logits.device).split_with_sizes([T, T, T * k])
    ids = torch.empty(T, k, dtype=torch.int32, device=logits.device)
    rc = nv.load().lx_token_scores(logits.data_ptr(), logits.stride(0), int(logits.dtype == torch.float32), T, V, t_ptr, wide, k, softcap,
                                   lp.data_ptr() if t_ptr else 0, ent.data_ptr(), ids.data_ptr(), best.data_ptr(), stream)
    nv._check(rc, "lx_token_scores")
    return TokenScores(lp if targets is not None else None, ent if entropy else None, ids, best.view(T, k))
