"""Causal attention of whole prompts over their own keys and values.

``prompt_attention`` serves the prompts of a step whose keys and values are in hand: packed
sequences of different lengths, grouped heads, query ``i`` of a sequence sees its keys up to
``i`` at full precision. Nothing is read from the cache (``kernels.prefill`` attends over
cached, quantized keys). Keys before the prompt join through ``prefix``: attention of the
same query rows over them (``kernels.shared.prefix_attention``) and its log-sum-exp. The
reference has no counterpart: its prefill reads the chunk back from the cache
(``echokv_vllm/kernels/prefill.py:170-207``).

Kernels: ``echokv_amd/csrc/attend_any.hip``, through ``echokv_prompt``.
"""

from __future__ import annotations

from typing import NamedTuple

import numpy as np
import torch

from echokv_amd import _lib
from echokv_amd._util import to_device
from echokv_amd.kernels.prefill import _out_view

MAX_HEAD_SIZE = 256


class PromptPlan(NamedTuple):
    """Query tiles of a step's prompts, built once for every layer."""

    tiles: torch.Tensor  # [n, 4] int32: (sequence's first row, its tokens, tile's first token, its tokens)
    tile_m: int  # query tokens per tile
    rows: int  # rows that query, key, value and output hold at least
    entries: tuple  # ((q_start, q_end), ...)
    gqa: int
    head_size: int


def _entries(prefill) -> tuple:
    """The non-empty row ranges, checked: inside the tensors and apart from one another."""
    out = []
    for e in prefill:
        qs, qe = int(e[0]), int(e[1])
        if qs < 0 or qe < qs:
            raise ValueError(f"bad prompt rows [{qs}, {qe})")
        if qe > qs:
            out.append((qs, qe))
    ordered = sorted(out)
    for (_, a), (b, _) in zip(ordered, ordered[1:]):
        if b < a:
            raise ValueError("prompts overlap: every row belongs to one sequence")
    return tuple(out)


def build_prompt_plan(prefill, gqa: int, head_size: int, device) -> PromptPlan:
    """The tiles of the prompts ``prefill``: ``(q_start, q_end, ...)`` row ranges of the packed
    tensors (as ``kernels.prefill.build_tiles`` takes them), one per sequence. Tiles with the
    most keys first, so that the longest workgroups start earliest."""
    tile_m = _lib.size("echokv_prompt_tile_m", gqa, 1, head_size)
    entries = _entries(prefill)
    rows = [(qs, qe - qs, t, min(tile_m, qe - qs - t)) for qs, qe in entries for t in range(0, qe - qs, tile_m)]
    rows.sort(key=lambda r: -(r[2] + r[3]))
    tiles = torch.from_numpy(np.array(rows, np.int32).reshape(-1, 4))
    return PromptPlan(to_device(tiles, device), tile_m, max((qe for _, qe in entries), default=0), entries, gqa,
                      head_size)


def _row_state(lse: torch.Tensor, rows: int, hq: int, name: str) -> torch.Tensor:
    if lse.dtype != torch.float32 or not lse.is_contiguous() or lse.dim() != 2 or lse.shape[0] < rows or lse.shape[1] != hq:
        raise ValueError(f"{name} must be contiguous float32 [T, {hq}]")
    return lse


def prompt_attention(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, output: torch.Tensor, prefill,
                     softmax_scale: float, plan: PromptPlan | None = None, lse: torch.Tensor | None = None,
                     prefix: tuple | None = None) -> None:
    """Write causal attention of every prompt into ``output [T, Hq, D]`` (or ``[T, Hq * D]``).

    ``query [T, Hq, D]``, ``key`` and ``value`` ``[T, H, D]`` (one dtype: float32, float16 or
    bfloat16; Hq a multiple of H; D a multiple of 4 up to 256) hold the step's tokens;
    ``prefill`` lists the row range of each prompt (``build_prompt_plan``), and rows outside
    them are left as they are. ``plan`` may be built once per step and shared by every layer.
    ``lse`` (float32 ``[T, Hq]``) receives each row's log-sum-exp of the scaled scores, in log2
    units. ``prefix = (part, part_lse)``: attention of the same rows over keys before their
    prompt, float32 ``[T, Hq, D]`` with its log-sum-exp ``[T, Hq]``
    (``kernels.shared.prefix_attention``), joined with the result."""
    if plan is None and not prefill:
        return
    if query.dim() != 3 or key.dim() != 3 or value.shape != key.shape:
        raise ValueError("query must be [T, Hq, D], key and value [T, H, D]")
    hq, h, d = query.shape[1], key.shape[1], query.shape[2]
    if h == 0 or hq % h or key.shape[2] != d:
        raise ValueError(f"{hq} query heads of {d} channels do not fit {h} KV heads of {key.shape[2]}")
    if key.dtype != query.dtype or value.dtype != query.dtype:
        raise ValueError(f"query, key and value must share a dtype, got {query.dtype}, {key.dtype}, {value.dtype}")
    out = _out_view(output, hq)
    if out.shape[1:] != query.shape[1:]:
        raise ValueError(f"output rows of shape {tuple(out.shape[1:])}, the query's are {tuple(query.shape[1:])}")
    _lib.require_current(query, key, value, output, lse)
    if plan is None:
        plan = build_prompt_plan(prefill, hq // h, d, query.device)
    if plan.gqa != hq // h or plan.head_size != d:
        raise ValueError("the plan was built for other heads")
    if plan.rows > min(t.shape[0] for t in (query, key, value, out)):
        raise ValueError(f"the prompts reach row {plan.rows}, the tensors hold fewer")
    if plan.tiles.shape[0] == 0:
        return
    _lib.require_current(plan.tiles)
    query, key, value = (t if t.stride(2) == 1 else t.contiguous() for t in (query, key, value))
    if lse is not None:
        _row_state(lse, plan.rows, hq, "lse")
    part, p_lse, p_s = None, None, (0, 0)
    if prefix is not None:
        part, p_lse = prefix
        _lib.require_current(part, p_lse)
        if part.dtype != torch.float32 or part.shape[1:] != query.shape[1:] or part.shape[0] < plan.rows or part.stride(2) != 1:
            raise ValueError("prefix rows must be float32 [T, Hq, D] with contiguous channels")
        _row_state(p_lse, plan.rows, hq, "the prefix's log-sum-exp")
        p_s = part.stride(0), part.stride(1)
    _lib.call(
        "echokv_prompt", _lib.ptr(query), query.stride(0), query.stride(1), _lib.ptr(key), key.stride(0), key.stride(1),
        _lib.ptr(value), value.stride(0), value.stride(1), _lib.dtype_code(query), hq, h, d, _lib.ptr(plan.tiles),
        plan.tiles.shape[0], plan.tile_m, float(softmax_scale), _lib.ptr(part), *p_s, _lib.ptr(p_lse), _lib.ptr(out),
        out.stride(0), out.stride(1), _lib.dtype_code(out), _lib.ptr(lse), _lib.stream(),
    )
