"""Attention of a batch over a cached prefix that all of it shares, computed once.

Sequences that begin with the same cached blocks (a system prompt, a document, the samples of
one request) have the same keys there. ``prefix_attention`` reads and dequantizes those keys
once for every query row of the batch; ``shared_prefix_decode`` is paged decode
(``kernels.decode.decode_attention``) of such a batch: the shared blocks once, each sequence's
own blocks as before, joined by log-sum-exp. The reference has no counterpart: its builder
takes vLLM's ``common_prefix_len`` and does not use it (``echokv_vllm/backend.py:337-496``).

The prefix is cut into ranges by the number of query rows, so a sequence's result depends on
its batch through float rounding (``decode_attention`` alone is batch-invariant).

Precision: scores, maxima, sums and outputs are float32. Into float16 and float32 outputs
``shared_prefix_decode`` holds keys, values and weights as exact float16 parts, as
``decode_attention`` does. Into bfloat16 outputs, for speed, the prefix's values and (bfloat16
queries) weights are rounded to float16 once each: together at most 2^-10 of the sum of weight x
|value|, where the output's own rounding is 2^-8. ``prefix_attention`` rounds the values to float16
once (2^-11, as the chunked prefill's kernels), and for bfloat16 queries the weights too. The
32-bit kernels hold everything in 32 bits.

Kernels: ``echokv_amd/csrc/shared.hip`` (head sizes 64, 128 and 256; queries and keys there are
float16 parts, so both are to stay within float16's range, as in ``decode_attention``), and
``echokv_amd/csrc/attend_any.hip`` (32-bit arithmetic for every other layout, and the join), through
``echokv_prefix`` and ``echokv_shared_decode``.
"""

from __future__ import annotations

import math

import torch

from echokv_amd import _lib
from echokv_amd.kernels import decode as dec


def _query(store, query: torch.Tensor) -> torch.Tensor:
    L, shape = store.layout, query.shape
    if len(shape) != 3 or shape[2] != L.head_size or shape[1] == 0 or shape[1] % L.num_kv_heads:
        raise ValueError(f"query of shape {tuple(shape)} does not fit {L.num_kv_heads} KV heads of {L.head_size}")
    return query if query.stride(2) == 1 else query.contiguous()


def _blocks(store, blocks: torch.Tensor, prefix_len: int) -> torch.Tensor:
    need = -(-prefix_len // store.layout.block_size)
    if blocks.dim() != 1 or blocks.numel() < need:
        raise ValueError(f"blocks must list the {need} blocks of a prefix of {prefix_len} tokens")
    blocks = blocks[:need]
    return blocks if blocks.dtype == torch.int32 and blocks.stride(0) == 1 else blocks.to(torch.int32).contiguous()


def _workspace(workspace: torch.Tensor | None, need: int, device) -> torch.Tensor | None:
    if workspace is None:
        return torch.empty(need, dtype=torch.uint8, device=device) if need else None
    if workspace.dtype != torch.uint8 or not workspace.is_contiguous() or workspace.numel() < need:
        raise ValueError(f"the workspace must be {need} contiguous uint8 bytes")
    if workspace.data_ptr() % 16:
        raise ValueError("the workspace must be aligned to 16 bytes")
    return workspace


def prefix_attention(store, query: torch.Tensor, blocks: torch.Tensor, prefix_len: int, softmax_scale: float,
                     part: torch.Tensor | None = None, lse: torch.Tensor | None = None,
                     workspace: torch.Tensor | None = None,
                     q_rows: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Attention of every row of ``query [T, Hq, D]`` over the first ``prefix_len`` cached tokens
    of the block list ``blocks`` (int32 ``[>= ceil(prefix_len / block_size)]``), each read once
    (the tokens of a block outside the cache count as zeros). ``q_rows`` (int64 indices into
    ``query``): of these rows alone; the others are left as they are, with a log-sum-exp of -inf where
    the call allocates ``lse``.

    Returns ``(part, lse)``: normalized float32 rows ``[T, Hq, D]`` and their log-sum-exp
    ``[T, Hq]`` in log2 units (zeros and -inf for an empty prefix), what
    ``kernels.prompt.prompt_attention`` takes as ``prefix``. ``workspace``: uint8,
    ``prefix_workspace_bytes(...)``; by default the call allocates it."""
    query = _query(store, query)
    t, hq, d = query.shape
    prefix_len = int(prefix_len)
    if q_rows is not None and q_rows.dim() != 1:
        raise ValueError("q_rows must be one row index after another")
    n = t if q_rows is None else q_rows.shape[0]
    if n and not t:
        raise ValueError(f"{n} row indices, no query rows")
    need = prefix_workspace_bytes(store, hq, n, prefix_len)
    _lib.require_current(query, blocks, part, lse, workspace, q_rows, store.pages)
    blocks = _blocks(store, blocks, prefix_len)
    q_rows = dec._i64(q_rows, query.device)
    if part is None:
        part = torch.empty(t, hq, d, device=query.device, dtype=torch.float32)
    if part.dtype != torch.float32 or part.shape != query.shape or part.stride(2) != 1:
        raise ValueError(f"part must be float32 {tuple(query.shape)} with contiguous channels")
    if lse is None:
        lse = torch.empty(t, hq, device=query.device, dtype=torch.float32)
        if q_rows is not None:
            lse.fill_(-math.inf)
    if lse.dtype != torch.float32 or lse.shape != (t, hq) or not lse.is_contiguous():
        raise ValueError(f"lse must be contiguous float32 {(t, hq)}")
    ws = _workspace(workspace, need, query.device)
    res = _lib.residual(store.res_k)
    q0, q1, _ = query.stride()
    p0, p1, _ = part.stride()
    _lib.call(
        "echokv_prefix", _lib.byref(store.abi), store.pages.data_ptr(), store.block_res.data_ptr(),
        store.res_group.data_ptr(), _lib.byref(res), query.data_ptr(), q0, q1, _lib.dtype_code(query), hq,
        _lib.ptr(q_rows), n, blocks.data_ptr(), prefix_len, float(softmax_scale), _lib.ptr(ws),
        0 if ws is None else ws.numel(), part.data_ptr(), p0, p1, lse.data_ptr(), _lib.stream(),
    )
    return part, lse


def prefix_workspace_bytes(store, num_q_heads: int, num_rows: int, prefix_len: int) -> int:
    """Workspace of a ``prefix_attention`` call, of any query type: partial rows by the number of rows,
    and at most 128 MiB for keys dequantized once for many rows, however long the prefix is."""
    return _lib.size("echokv_prefix_workspace", _lib.byref(store.abi), num_q_heads, num_rows, prefix_len)


def shared_workspace_bytes(store, num_q_heads: int, num_seqs: int, prefix_len: int, num_splits: int) -> int:
    """Workspace of a ``shared_prefix_decode`` call."""
    return _lib.size("echokv_shared_decode_workspace", _lib.byref(store.abi), num_q_heads, num_seqs, prefix_len,
                     num_splits)


def suffix_blocks(store, num_seqs: int) -> int:
    """Blocks per split of the tokens behind the prefix when the caller names none: 128 tokens
    for few sequences (up to 64 groups of four KV heads), else 256. A split is a serial chain of
    tiles, and these results depend on the batch anyway. us a call at 128 / 256 / 1024 tokens:
    4 sequences of 500-2000 behind 2048 tokens 32 / 40 / 84, 16 of them 40 / 45 / 90, 64
    73 / 68 / 115, 128 of 100-2000 104 / 100 / 141."""
    L = store.layout
    tokens = 128 if num_seqs * -(-L.num_kv_heads // 4) <= 64 else 256
    return max(1, tokens // L.block_size)


def suffix_splits(max_blocks: int, block_size: int, prefix_len: int, blocks_per_split: int,
                  max_len: int | None) -> int:
    """Splits of the tokens behind the prefix for sequences of at most ``max_blocks`` blocks (and
    ``max_len`` tokens)."""
    cols = max(0, max_blocks - prefix_len // block_size)
    longest = cols if max_len is None else min(cols, -(-max(0, max_len - prefix_len) // block_size))
    return max(dec.SHORT_SPLITS, min(-(-longest // blocks_per_split), dec.MAX_SPLITS))


def shared_prefix_decode(store, query: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                         prefix_len: int, softmax_scale: float, blocks_per_split: int | None = None,
                         q_rows: torch.Tensor | None = None, bt_rows: torch.Tensor | None = None,
                         blocks: torch.Tensor | None = None, out: torch.Tensor | None = None,
                         max_len: int | None = None, num_splits: int | None = None,
                         workspace: torch.Tensor | None = None, tier: int | None = None,
                         tier_mask: torch.Tensor | str | None = None) -> torch.Tensor:
    """``decode_attention`` of sequences whose first ``prefix_len`` tokens (a multiple of the
    block size) are the same cached blocks, which are read once for the batch.

    Arguments as ``decode_attention``'s; ``seq_lens[i]`` counts the prefix, and row
    ``bt_rows[i]`` of the block table begins with the shared blocks. ``blocks``: their list (int32), by
    default the first row of the table (name it where that row is padding). A sequence shorter than
    ``prefix_len`` (length 0: graph padding) leaves its row untouched. ``num_splits`` and
    ``blocks_per_split`` (default ``suffix_blocks``) cut the tokens behind the prefix.
    ``workspace``: uint8, ``shared_workspace_bytes(...)``; by default the call allocates it. A prefix
    of 0 tokens is plain decode. Short prefixes (below about 1024 tokens) take no less time here than
    in ``decode_attention``: two launches more, and little to share. Outputs in bfloat16 round the
    prefix's weights and values once more than ``decode_attention`` (see the module)."""
    prefix_len = int(prefix_len)
    if prefix_len == 0:
        return dec.decode_attention(store, query, block_table, seq_lens, softmax_scale,
                                    blocks_per_split or dec.BLOCKS_PER_SPLIT, q_rows, bt_rows, out, max_len, num_splits,
                                    None, tier, True, tier_mask)
    L = store.layout
    if prefix_len < 0 or prefix_len % L.block_size:
        raise ValueError(f"prefix_len must be a multiple of the block size {L.block_size}, got {prefix_len}")
    query = _query(store, query)
    hq, d = query.shape[1:]
    s = seq_lens.shape[0]
    if q_rows is not None and q_rows.shape[0] < s or bt_rows is not None and bt_rows.shape[0] < s:
        raise ValueError(f"{s} sequences, fewer row indices")
    if bt_rows is None and block_table.shape[0] < s:
        raise ValueError(f"{s} sequences, {block_table.shape[0]} block-table rows")
    if out is not None and out.shape[0] < (s if q_rows is None else 1):
        raise ValueError(f"{s} sequences, {out.shape[0]} output rows")
    _lib.require_current(query, block_table, seq_lens, q_rows, bt_rows, blocks, out, workspace, store.pages)
    if q_rows is None and query.shape[0] < s:
        raise ValueError(f"{s} sequences, {query.shape[0]} query rows")
    if block_table.dim() != 2 or block_table.shape[1] * L.block_size < prefix_len:
        raise ValueError(f"the block table holds fewer than {prefix_len} tokens a row")
    if block_table.dtype != torch.int32 or block_table.stride(1) != 1:
        block_table = block_table.to(torch.int32).contiguous()
    if s and blocks is None and block_table.shape[0] == 0:
        raise ValueError("the block table has no row to take the shared blocks from")
    if blocks_per_split is None:
        blocks_per_split = suffix_blocks(store, s)
    if num_splits is None:
        num_splits = suffix_splits(block_table.shape[1], L.block_size, prefix_len, blocks_per_split, max_len)
    need = shared_workspace_bytes(store, hq, s, prefix_len, int(num_splits))
    dev = query.device
    lens, q_rows, bt_rows = dec._i64(seq_lens, dev), dec._i64(q_rows, dev), dec._i64(bt_rows, dev)
    if out is None:
        out = torch.empty(s if q_rows is None else query.shape[0], hq, d, device=dev, dtype=torch.float32)
    if out.dim() != 3 or out.shape[1:] != query.shape[1:] or out.stride(2) != 1:
        raise ValueError("out must be [rows, Hq, D] with contiguous channels")
    if s == 0:
        return out
    blocks = _blocks(store, block_table[0] if blocks is None else blocks, prefix_len)
    tier_mask = dec.tier_mask_of(store, tier_mask, dev)
    if tier is None:
        tier = store.pool.majority_tier()
    ws = _workspace(workspace, need, dev)
    res = _lib.residual(store.res_k)
    q0, q1, _ = query.stride()
    o0, o1, _ = out.stride()
    _lib.call(
        "echokv_shared_decode", _lib.byref(store.abi), store.pages.data_ptr(), store.block_res.data_ptr(),
        store.res_group.data_ptr(), _lib.byref(res), query.data_ptr(), q0, q1, _lib.dtype_code(query), hq,
        _lib.ptr(q_rows), block_table.data_ptr(), block_table.stride(0), _lib.ptr(bt_rows), lens.data_ptr(), s,
        blocks.data_ptr(), prefix_len, float(softmax_scale), int(num_splits), int(blocks_per_split), int(tier),
        _lib.ptr(tier_mask), ws.data_ptr(), ws.numel(), out.data_ptr(), o0, o1, _lib.dtype_code(out), _lib.stream(),
    )
    return out
