"""GPU: prefixes longer than a slab of the dequantized prefix, against float64."""

import pytest
import torch

from attend64 import Rows, check
from test_gpu_shared_prefix import BF16, BOUND, F16, Cache, check_prefix

from echokv_amd.kernels.shared import prefix_attention, prefix_workspace_bytes, shared_prefix_decode

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("h,d,rows,n,tiers", [(8, 128, 130, 50007, (4,)), (8, 128, 1100, 30000, (4, 8)),
                                              (4, 64, 600, 100032, (8,)), (4, 64, 2100, 90001, (4,))], ids=str)
def test_prefix_in_several_slabs(device, h, d, rows, n, tiers):
    """Several ranges, and one (1100 rows of 8 heads, 2100 of 4: the rows go on from the workspace there
    too). A workspace full of NaN changes nothing."""
    print(f"[slabs] {h} x {d}, {rows} behind {n}", flush=True)
    c = Cache(device, n, [], h=h, d=d, bs=64, kg=32, tiers=tiers, seed=n)
    gqa = 4 if d == 128 else 8
    q = c.queries(rows, gqa, BF16)
    need = prefix_workspace_bytes(c.store, h * gqa, rows, n)
    ws = torch.full((need,), 0xFF, dtype=torch.uint8, device=device)
    part, lse = prefix_attention(c.store, q, c.blocks, n, d ** -0.5)
    again = prefix_attention(c.store, q, c.blocks, n, d ** -0.5, workspace=ws)
    torch.cuda.synchronize()
    assert torch.equal(part, again[0]) and torch.equal(lse, again[1])
    some = [0, 1, rows // 2, rows - 1]
    check_prefix(c, q[some], part[some], lse[some], n, d ** -0.5)


def test_every_slab_counts_once(device):
    """Keys that take half of a row's weight at the ends of slabs, ranges and tiles: a lost or doubled
    one moves the row by a third of its value."""
    n, d = 50007, 128
    c = Cache(device, n, [], h=8, bs=64, kg=32)
    probes = [0, 63, 64, n // 2, n - 8, n - 1] + [x + e for x in (16768, 16704, 25088, 33536, 41856) for e in (-1, 0)]
    k, v = c.tokens(0, n)
    q = torch.zeros(130, 32, d, dtype=F16, device=device)
    for i in range(130):
        q[i] = (k[probes[i % len(probes)]].repeat_interleave(4, 0) * 1.2).half()
    part, lse = prefix_attention(c.store, q, c.blocks, n, d ** -0.5)
    torch.cuda.synchronize()
    some = list(range(len(probes)))
    check_prefix(c, q[some], part[some], lse[some], n, d ** -0.5)


def test_decode_behind_several_slabs(device):
    print("[slabs] decode", flush=True)
    c = Cache(device, 49984, [3, 70] * 70, h=8, bs=64, kg=32)
    q = c.queries(140, 4, F16)
    out = torch.full_like(q, 9.0)
    lens = torch.tensor(c.lens, device=device)
    lens[5], lens[7] = 0, 49983
    shared_prefix_decode(c.store, q, c.table, lens, c.prefix, c.d ** -0.5, out=out)
    torch.cuda.synchronize()
    for i in (0, 1, 77, 139):
        k, v = c.tokens(i, c.lens[i])
        check(out[i : i + 1], Rows(q[i : i + 1], k, v, [c.lens[i]], c.d ** -0.5), **BOUND)
    assert (out[5] == 9).all() and (out[7] == 9).all()


def test_slabs_in_a_graph(device):
    """Captured and replayed, the lengths changing, with eager calls between: every replay equals the eager
    result bit for bit."""
    print("[slabs] graph", flush=True)
    c = Cache(device, 32000, [3, 70] * 70, h=8, bs=64, kg=32)
    q = c.queries(140, 4, F16)
    lens = torch.tensor(c.lens, device=device)
    rows = torch.arange(139, 0, -1, device=device)
    out, part, lse = torch.zeros_like(q), torch.zeros_like(q, dtype=torch.float32), torch.zeros(140, 32, device=device)

    def call(o, p, x):
        shared_prefix_decode(c.store, q, c.table, lens, c.prefix, c.d ** -0.5, out=o, tier=4)
        prefix_attention(c.store, q, c.blocks, c.prefix, c.d ** -0.5, part=p, lse=x, q_rows=rows)

    call(out, part, lse)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(out, part, lse)
    for rep in range(3):
        lens.copy_(torch.tensor([max(c.prefix, n - 9 * rep) for n in c.lens], device=device))
        for t in (out, part, lse):
            t.zero_()
        g.replay()
        eager = [torch.zeros_like(t) for t in (out, part, lse)]
        call(*eager)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((out, part, lse), eager)), rep
        assert (part[0] == 0).all() and (out[0] != 0).any()
