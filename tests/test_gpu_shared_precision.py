"""GPU: how many bits the prefix kernels hold, on inputs where nothing else is rounded.

A few keys of the prefix take all of the weight, their scores are single products of numbers that two
float16 parts hold exactly (channel 0 alone of the query, keys from 0 to their group's maximum), and
all other keys' scores are 30 below: the 8192 of them add less than 2^-29 to any sum. What is left of
the error is a few roundings of float32, against which one of 2^-11 shows."""

import numpy as np
import pytest
import torch

from attend64 import Rows, check, unit

from echokv_amd.kernels.shared import prefix_attention, shared_prefix_decode
from echokv_amd.tiered_cache import TieredKVCache, TieredLayout

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TARGETS = 5
TWO_PARTS = 2.0 ** -21  # a float16 hi + lo pair: 2^-22, the product of two low parts left out as much


class Probe:
    def __init__(self, device, d, gqa, seqs, prefix, whole_values, h=2, bs=16, vg=32, seed=0, tier=4, largest=0.0):
        g = torch.Generator(device=device)
        g.manual_seed(seed)
        rng = np.random.default_rng(seed)
        self.d, self.prefix, self.bs, self.device, tail = d, prefix, bs, device, 5
        shared = prefix // bs
        nb = shared + seqs
        perm = rng.permutation(nb)
        table = np.zeros((seqs, shared + 1), np.int64)
        table[:, :shared], table[:, shared] = perm[:shared], perm[shared:]
        layout = TieredLayout(h, d, bs, 8, bs, vg)
        pages = torch.zeros(nb, bs * TieredLayout.per_token_bytes(h, d, 8, bs, vg), dtype=torch.uint8, device=device)
        self.store = TieredKVCache(layout, pages, residual_slots=seqs + 4, residual_dtype=F16)
        n = prefix + tail * seqs
        k, v = (torch.randn(n, h, d, device=device, generator=g) for _ in range(2))
        k[:, :, 0] = 0.0
        # One target a K group at most: its value is 15 steps of the group, the others' 0. All in 128 aligned
        # keys, so in one range: alone in its range a target's weight is 1, which every type holds.
        groups = rng.integers(prefix // 128) * (128 // bs) + rng.choice(128 // bs, TARGETS, replace=False)
        self.targets = np.sort(groups) * bs + rng.integers(0, bs, TARGETS)
        k[torch.from_numpy(self.targets).to(device), :, 0] = 30 + torch.rand(TARGETS, h, device=device, generator=g)
        if whole_values:  # 0 to 15, both in every V group: exact in INT4 and in float16
            v = torch.randint(0, 16, v.shape, device=device, generator=g).float()
            v[:, :, ::vg], v[:, :, 1::vg] = 0.0, 15.0
        if largest:  # both signs in every V group
            v = largest * (2 * torch.rand(v.shape, device=device, generator=g) - 1)
            v[:, :, ::vg], v[:, :, 1::vg] = -largest, largest
        slots = np.concatenate([table[0][np.arange(prefix) // bs] * bs + np.arange(prefix) % bs,
                                (table[:, -1:] * bs + np.arange(tail)).reshape(-1)])
        self.store.write(k.half(), v.half(), torch.from_numpy(slots), tier)
        self.table_np, self.table = table, torch.from_numpy(table).to(device, torch.int32)
        self.lens = torch.full((seqs,), prefix + tail, device=device)
        self.q = torch.zeros(seqs, h * gqa, d, device=device)
        self.q[:, :, 0] = 1 + torch.arange(seqs, device=device)[:, None] % 4 / 4

    def rows(self, i, n):
        p = np.arange(n)
        blk = torch.from_numpy(self.table_np[i][p // self.bs]).to(self.device)
        k, v = self.store.gather(blk, torch.from_numpy(p % self.bs).to(self.device))
        return k, v


def expect(c, q, i, n):
    r = Rows(q[i : i + 1], *c.rows(i, n), [n], 1.0)
    r.keys, r.d = TARGETS, 1  # what its sums are made of
    return r


# (head size, GQA, sequences, prefix): one workgroup of four waves a KV head and range, eight waves,
# the prefix dequantized first, 32-bit kernels.
PATHS = [(128, 4, 3, 512), (64, 4, 3, 512), (256, 4, 3, 512), (128, 4, 40, 6400), (64, 8, 20, 6400),
         (128, 4, 200, 4096), (64, 4, 300, 2048), (96, 4, 3, 512)]


@pytest.mark.parametrize("d,gqa,seqs,prefix", PATHS)
@pytest.mark.parametrize("dtype", [F16, BF16, F32], ids=str)
def test_decode_holds_weights_and_values_exactly(device, d, gqa, seqs, prefix, dtype):
    """As paged decode does: into float32, and float16 beyond its own rounding."""
    print(f"[precision] decode {d} {gqa} {seqs} {prefix} {dtype}", flush=True)
    c = Probe(device, d, gqa, seqs, prefix, whole_values=False, vg=24 if d == 96 else 32, seed=d + seqs)
    q = c.q.to(dtype)
    outs = [torch.zeros(q.shape, dtype=t, device=device) for t in (F32, F16)]
    for out in outs:
        shared_prefix_decode(c.store, q, c.table, c.lens, prefix, 1.0, out=out, tier=4)
    torch.cuda.synchronize()
    for out in outs:
        for i in sorted({0, 1, seqs // 2, seqs - 1}):
            check(out[i : i + 1], expect(c, q, i, prefix + 5), weight=TWO_PARTS, value=TWO_PARTS)


@pytest.mark.parametrize("d,gqa,seqs,prefix", PATHS)
@pytest.mark.parametrize("dtype", [F16, BF16, F32], ids=str)
def test_prefix_weights(device, d, gqa, seqs, prefix, dtype):
    """Values exact in float16: what is left is the weights' rounding, none for float16 and float32
    queries, one of float16 for bfloat16 ones."""
    print(f"[precision] prefix {d} {gqa} {seqs} {prefix} {dtype}", flush=True)
    c = Probe(device, d, gqa, seqs, prefix, whole_values=True, vg=24 if d == 96 else 32, seed=d + seqs)
    q = c.q.to(dtype)
    part, lse = prefix_attention(c.store, q, c.table[0], prefix, 1.0)
    torch.cuda.synchronize()
    for i in sorted({0, 1, seqs // 2, seqs - 1}):
        r = expect(c, q, i, prefix)
        check(part[i : i + 1], r, weight=unit(F16) if dtype == BF16 else TWO_PARTS)
        assert float((lse[i] - r.lse).abs().max()) <= r.lse_bound()


@pytest.mark.parametrize("d,gqa,seqs,prefix", [(128, 4, 3, 512), (256, 4, 3, 512), (64, 8, 20, 6400), (128, 4, 200, 4096)])
@pytest.mark.parametrize("tier", [2, 4, 8])
def test_the_largest_values(device, d, gqa, seqs, prefix, tier):
    """Values of -65504 and 65504 in every V group: dequantized (65536 in INT4) they can pass float16."""
    print(f"[precision] largest {d} {gqa} {seqs} {prefix} INT{tier}", flush=True)
    c = Probe(device, d, gqa, seqs, prefix, whole_values=False, tier=tier, largest=65504.0, seed=d + seqs)
    q = c.q.half()
    got = shared_prefix_decode(c.store, q, c.table, c.lens, prefix, 1.0, tier=tier)
    torch.cuda.synchronize()
    passed = False
    for i in sorted({0, 1, seqs - 1}):
        r = expect(c, q, i, prefix + 5)
        passed = passed or r.vmax > 65504
        check(got[i : i + 1], r, weight=TWO_PARTS, value=TWO_PARTS)
    assert passed or tier != 4
