"""Bindings of the operators of short ragged steps: `csrc/kernels/step_tables.cu`, `moe_few.cu` and `token_scores.cu`.  Imported into
:mod:`lorax_b200.ops.native`; `reference` states what they compute.

Arguments that do not fit raise ValueError in front of any launch.  Outputs and scratch are allocated by the call, on the stream that is current
(calls on several streams, and captured graphs, share nothing)."""

from __future__ import annotations

import ctypes
from ctypes import c_float, c_int, c_longlong, c_void_p
from typing import Optional, Sequence, Tuple

import torch

from . import native as nv
from .reference import MOE_FEW_TOKENS, TOP_MAX, StepTables, TokenScores, check_moe_few, check_step_tables, check_token_scores

P, I, L, F = c_void_p, c_int, c_longlong, c_float

SIGNATURES = {
    "lx_step_tables_max_seqs": ([], I),
    "lx_step_tables": ([P, L, P, I, I, I, I, I, I, I, P, P, I, P, I, I, I, P, P], I),
    "lx_moe_few_max_tokens": ([], I),
    "lx_moe_few": ([P, L, P, P, P, P, P, P, L, I, I, I, I, I, I, I, I, I, F, I, P], I),
    "lx_token_scores_max_top": ([], I),
    "lx_token_scores": ([P, L, I, I, I, P, I, I, F, P, P, P, P, P], I),
}


def check_limits(lib):
    for name, here in (("lx_moe_few_max_tokens", MOE_FEW_TOKENS), ("lx_token_scores_max_top", TOP_MAX)):
        if getattr(lib, name)() != here:
            raise nv.NativeError(f"{name}: C++ says {getattr(lib, name)()}, Python says {here}")


def _on_current_device(*tensors: Optional[torch.Tensor]):
    here = torch.cuda.current_device()
    for t in tensors:
        if t is not None and t.device.index != here:
            raise ValueError(f"a tensor on {t.device} while cuda:{here} is the current device")


def step_tables(seqs: torch.Tensor, pages: torch.Tensor, tokens: int, max_blocks: int, page: int, window: int = 0,
                tiles: Sequence[Tuple[int, int]] = (), lora_tiles: int = 0, lora_rows: int = 32, row_offset: int = 0,
                lead: Optional[torch.Tensor] = None) -> StepTables:
    """Tables of a ragged step from its sequences' lengths (`reference.step_tables` states them), in one launch."""
    B = check_step_tables(seqs, pages, tokens, max_blocks, page, window, tiles, lora_tiles, lora_rows, lead)
    _on_current_device(seqs, pages, lead)
    M, n_lead, n_lists = max_blocks, 0 if lead is None else lead.shape[0], len(tiles)
    sizes = [4 * (n_lead + lora_tiles), B + 1, tokens, tokens, tokens, B * M]
    for _, n in tiles:
        sizes += (n, n)
    out = torch.empty(sum(sizes), dtype=torch.int32, device=seqs.device)
    heights, counts = (I * n_lists)(*[h for h, _ in tiles]), (I * n_lists)(*[n for _, n in tiles])
    rc = nv.load().lx_step_tables(seqs.data_ptr(), seqs.stride(0), pages.data_ptr(), pages.shape[0], B, tokens, M, page, window, row_offset, heights, counts,
                                  n_lists, None if lead is None else lead.data_ptr(), n_lead, lora_rows, lora_tiles, out.data_ptr(), nv._stream())
    nv._check(rc, "lx_step_tables")
    lora, cu, pos, slots, tok, bt, *lists = out.split(sizes)
    return StepTables(cu, pos, slots, tok, bt.view(B, M), tuple(zip(lists[::2], lists[1::2])), lora.view(-1, 4))


def moe_few(x: torch.Tensor, router_w: torch.Tensor, w13: torch.Tensor, w2: torch.Tensor, k: int, e0: int = 0, act: str = "silu", renorm: bool = True,
            scale: float = 1.0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The mixture-of-experts feed-forward of up to `MOE_FEW_TOKENS` tokens (`reference.moe_few` states it; `moe_ffn` takes any number)."""
    T, E, H, inter = check_moe_few(x, router_w, w13, w2, k, e0, act, scale, out)
    if x.dtype != torch.bfloat16:
        raise ValueError(f"moe_few: the kernels are bf16; got {x.dtype}")
    _on_current_device(x, router_w, w13, w2, out)
    if out is None:
        out = torch.empty(T, H, dtype=x.dtype, device=x.device)
    if T == 0:
        return out
    lib, stream = nv.load(), nv._stream()
    logits = torch.empty(T, E, dtype=torch.float32, device=x.device)
    nv._check(lib.lx_moe_router_logits(x.data_ptr(), x.stride(0), router_w.data_ptr(), router_w.stride(0), logits.data_ptr(), T, E, H, None, 0, stream),
              "lx_moe_router_logits")
    ids = torch.empty(T * k, dtype=torch.int32, device=x.device)
    h = torch.empty(2 * T * k * inter, dtype=torch.bfloat16, device=x.device)
    rc = lib.lx_moe_few(x.data_ptr(), x.stride(0), logits.data_ptr(), w13.data_ptr(), w2.data_ptr(), ids.data_ptr(), h.data_ptr(), out.data_ptr(), out.stride(0),
                        T, E, k, e0, w13.shape[0], H, inter, nv._ACTS[act], int(renorm), scale, nv.workspace(x.device).num_sms, stream)
    nv._check(rc, "lx_moe_few")
    nv.launch_count += 1                 # (two kernels)
    return out


def token_scores(logits: torch.Tensor, targets: Optional[torch.Tensor] = None, k: int = 0, softcap: float = 0.0) -> TokenScores:
    """Log-probability of a given token of every row, entropy of the row, and its `k` best tokens with their log-probabilities
    (`reference.token_scores` states them): one pass over the logits, one launch."""
    T, V = check_token_scores(logits, targets, k, softcap)
    if logits.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"token_scores: the kernels take bf16 and fp32 logits; got {logits.dtype}")
    _on_current_device(logits, targets)
    if targets is not None and not targets.is_contiguous():
        targets = targets.contiguous()
    out = torch.empty(T * (2 + 2 * k), dtype=torch.float32, device=logits.device)
    lp, ent, top, ids = out.split([T, T, T * k, T * k])
    rc = nv.load().lx_token_scores(logits.data_ptr(), logits.stride(0), int(logits.dtype == torch.float32), T, V, None if targets is None else targets.data_ptr(),
                                   int(targets is not None and targets.dtype == torch.int64), k, softcap, None if targets is None else lp.data_ptr(), ent.data_ptr(),
                                   ids.data_ptr(), top.data_ptr(), nv._stream())
    nv._check(rc, "lx_token_scores")
    return TokenScores(None if targets is None else lp, ent, ids.view(torch.int32).view(T, k), top.view(T, k))
