"""Causal attention of whole prompts over their own keys and values.

``prompt_attention`` serves the prompts of a step whose keys and values are in hand: packed
sequences of different lengths, grouped heads, query ``i`` of a sequence sees its keys up to
``i`` at full precision. Nothing is read from the cache (``kernels.prefill`` attends over
cached, quantized keys). Keys before the prompt join through ``prefix``: attention of the
same query rows over them (``kernels.shared.prefix_attention``) and its log-sum-exp. The
reference has no counterpart: its prefill reads the chunk back from the cache
(``echokv_vllm/kernels/prefill.py:170-207``).

Kernels: ``echokv_amd/csrc/prompt.hip`` (float16 and bfloat16 of head size 64, 128 or 256) and
``echokv_amd/csrc/attend_any.hip`` (32-bit arithmetic, every other case), through ``echokv_prompt``.
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
    reach = max((qe for _, qe in entries), default=0)
    if reach > np.iinfo(np.int32).max:
        raise ValueError(f"the prompts reach row {reach}: rows are 32 bits")
    start, end = np.array(entries, np.int64).reshape(-1, 2).T
    n = -(-(end - start) // tile_m)  # tiles of each prompt
    seq = np.repeat(np.arange(len(entries)), n)
    first = (np.arange(seq.size) - np.repeat(np.cumsum(n) - n, n)) * tile_m
    last = np.minimum(first + tile_m, (end - start)[seq])
    rows = np.stack([start[seq], (end - start)[seq], first, last - first], 1)[np.argsort(-last, kind="stable")]
    tiles = torch.from_numpy(rows.astype(np.int32))
    return PromptPlan(to_device(tiles, device), tile_m, reach, entries, gqa, head_size)


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
    (``kernels.shared.prefix_attention``), joined with the result; a row whose ``part_lse`` is -inf
    has none. 16-bit rows of head size 64, 128 or 256, 16-byte aligned, have the same bits whatever
    else the step holds, and each of their softmax weights is rounded to the inputs' type once (of
    weight x |value| bfloat16 2^-8, float16 2^-11), whatever the output's type; in the 32-bit kernels
    (every other case) nothing is held in fewer than 32 bits, and the bits depend on the step's size
    through float rounding."""
    if plan is None and not prefill:
        return
    qs, ks = query.shape, key.shape
    if len(qs) != 3 or len(ks) != 3 or value.shape != ks:
        raise ValueError("query must be [T, Hq, D], key and value [T, H, D]")
    t, hq, d = qs
    h = ks[1]
    if h == 0 or hq % h or ks[2] != d:
        raise ValueError(f"{hq} query heads of {d} channels do not fit {h} KV heads of {ks[2]}")
    dtype = query.dtype
    if key.dtype != dtype or value.dtype != dtype:
        raise ValueError(f"query, key and value must share a dtype, got {dtype}, {key.dtype}, {value.dtype}")
    out = output if output.dim() == 3 else _out_view(output, hq)
    out_rows, out_hq, out_d = out.shape
    if out_hq != hq or out_d != d:
        raise ValueError(f"output rows of shape {(out_hq, out_d)}, the query's are {(hq, d)}")
    if plan is None:
        _lib.require_current(query)
        plan = build_prompt_plan(prefill, hq // h, d, query.device)
    part, p_lse = prefix if prefix is not None else (None, None)
    if (part is None) != (p_lse is None):
        raise ValueError("a prefix is rows and their log-sum-exp, both")
    _lib.require_current(query, key, value, output, lse, part, p_lse, plan.tiles)
    if plan.gqa != hq // h or plan.head_size != d:
        raise ValueError("the plan was built for other heads")
    if plan.rows > min(t, ks[0], out_rows):
        raise ValueError(f"the prompts reach row {plan.rows}, the tensors hold fewer")
    n_tiles = plan.tiles.shape[0]
    if n_tiles == 0:
        return
    (q, q0, q1), (k, k0, k1), (v, v0, v1) = _rows(query), _rows(key), _rows(value)
    o0, o1, o2 = out.stride()
    if o2 != 1:
        raise ValueError("output rows must be contiguous along head_dim")
    p0 = p1 = 0
    if lse is not None:
        _row_state(lse, plan.rows, hq, "lse")
    if part is not None:
        if part.dtype != torch.float32 or part.shape[1:] != qs[1:] or part.shape[0] < plan.rows or part.stride(2) != 1:
            raise ValueError("prefix rows must be float32 [T, Hq, D] with contiguous channels")
        _row_state(p_lse, plan.rows, hq, "the prefix's log-sum-exp")
        p0, p1, _ = part.stride()
    code = _lib.dtype_code(query)
    _lib.call(
        "echokv_prompt", q.data_ptr(), q0, q1, k.data_ptr(), k0, k1, v.data_ptr(), v0, v1, code, hq, h, d,
        plan.tiles.data_ptr(), n_tiles, plan.tile_m, float(softmax_scale), _lib.ptr(part), p0, p1, _lib.ptr(p_lse),
        out.data_ptr(), o0, o1, code if out.dtype == dtype else _lib.dtype_code(out), _lib.ptr(lse), _lib.stream(),
    )


def _rows(t: torch.Tensor) -> tuple:
    """``t`` with contiguous channels, and its row and head strides."""
    s0, s1, s2 = t.stride()
    if s2 != 1:
        t = t.contiguous()
        s0, s1, _ = t.stride()
    return t, s0, s1
