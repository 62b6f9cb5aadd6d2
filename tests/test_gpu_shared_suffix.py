"""GPU: decode behind a shared prefix with suffixes of 0 to some thousand tokens, cut into few and many
splits, against float64. Each query is the sum of two cached keys, one of them at an end of a block, split
or range: the two share the weight, so that a key lost there or counted twice moves the row by a large
part of its value."""

import numpy as np
import pytest
import torch

from attend64 import Rows, check
from test_gpu_shared_prefix import BF16, BOUND, F16, Cache

from echokv_amd.kernels.shared import shared_prefix_decode

pytestmark = pytest.mark.gpu

TAILS = [1, 2113, 0, 130, 1500, 16, 643, 1024]


def ends(c, n):
    """Positions below ``n`` around the ends of what the keys may be cut into: the prefix, and steps
    of 64 to 1024 tokens on either side of it."""
    cuts = {0, c.prefix, n}
    for step in (64, 128, 256, 1024):
        cuts.update(range(step, min(c.prefix, 4 * step), step))
        cuts.update(range(c.prefix + step, n, step))
    at = sorted({p for x in cuts for p in (x - 1, x) if 0 <= p < n})
    return at


def probes(c, gqa, dtype, step):
    """A query for each sequence and head: its key at one of ``ends`` plus one anywhere."""
    rng = np.random.default_rng(step)
    q = torch.zeros(len(c.lens), c.h * gqa, c.d, device=c.device)
    for i, n in enumerate(c.lens):
        if n == 0:
            continue
        k, _ = c.tokens(i, n)
        at = ends(c, n)
        for j in range(c.h * gqa):
            a, b = at[(step * c.h * gqa + 7 * i + j) % len(at)], int(rng.integers(n))
            q[i, j] = (k[a, j // gqa].float() + k[b, j // gqa].float()) * (12 * c.d ** -0.5)
    return q.to(dtype)


def run(c, gqa, dtype, calls, rows=None, **kw):
    lens = torch.tensor(c.lens, device=c.device)
    for step in range(calls):
        q = probes(c, gqa, dtype, step)
        out = torch.full(q.shape, 9.0, device=c.device)
        shared_prefix_decode(c.store, q, c.table, lens, c.prefix, c.d ** -0.5, out=out, **kw)
        torch.cuda.synchronize()
        for i in rows if rows is not None else range(len(c.lens)):
            check(out[i : i + 1], Rows(q[i : i + 1], *c.tokens(i, c.lens[i]), [c.lens[i]], c.d ** -0.5), **BOUND)


@pytest.mark.parametrize("kw", [dict(), dict(d=64), dict(d=256), dict(d=96, vg=24), dict(bs=64, kg=32),
                                dict(bs=128, kg=64, vg=64)], ids=str)
@pytest.mark.parametrize("max_len", [False, True])
def test_mixed_suffixes(device, kw, max_len):
    print(f"[suffix] {kw} {max_len}", flush=True)
    c = Cache(device, 256, TAILS, seed=11, **kw)
    run(c, 8, F16, 4, max_len=max(c.lens) if max_len else None)


@pytest.mark.parametrize("d", [128, 96])
@pytest.mark.parametrize("num_splits,blocks_per_split", [(1, 1), (1, 16), (2, 3), (5, 2), (33, 1), (64, 2), (100, 1)])
def test_few_and_many_splits(device, d, num_splits, blocks_per_split):
    """Sequences of more blocks than the splits were named for, and of fewer."""
    print(f"[suffix] {num_splits} x {blocks_per_split} D{d}", flush=True)
    c = Cache(device, 128, TAILS, d=d, vg=32 if d == 128 else 24, seed=12)
    run(c, 4, BF16, 4, num_splits=num_splits, blocks_per_split=blocks_per_split)


@pytest.mark.parametrize("prefix,tail,num_splits", [(8192, 900, 64), (7936, 2000, 20), (8192, 5, 4)])
def test_more_pieces_than_lanes(device, prefix, tail, num_splits):
    """64 or 62 ranges of the prefix and up to 57 splits: the join takes them 64 at a time."""
    print(f"[suffix] {prefix} + {tail}", flush=True)
    c = Cache(device, prefix, [tail], h=2, seed=13)
    run(c, 8, F16, 6, num_splits=num_splits, blocks_per_split=1)


@pytest.mark.parametrize("seqs", [3, 200])
def test_suffixes_of_two_tiers(device, seqs):
    """Each tier's blocks by its own kernel into the same pieces."""
    print(f"[suffix] tiers {seqs}", flush=True)
    tails = [(1, 700, 33, 300)[i % 4] for i in range(seqs)]
    c = Cache(device, 512, tails, tiers=(4, 8), seed=14)
    run(c, 4, F16, 2, rows=(0, 1, 2) if seqs == 3 else (0, 1, 101, 199), tier_mask="auto")


def test_suffixes_behind_a_packed_prefix(device):
    """Enough rows that the prefix is dequantized first."""
    print("[suffix] packed", flush=True)
    tails = [(1, 1300, 0, 300, 130, 17)[i % 6] for i in range(160)]
    c = Cache(device, 3200, tails, h=4, bs=64, kg=32, seed=15)
    run(c, 8, BF16, 2, rows=(0, 1, 2, 81, 159))
