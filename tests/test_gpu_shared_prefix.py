"""GPU: attention over a shared cached prefix and decode of a batch behind one (kernels.shared),
against float64 over the cache's own dequantized keys and values."""

import numpy as np
import pytest
import torch

from attend64 import Rows, check, unit
from echokv_amd.kernels import decode as dec
from echokv_amd.kernels.prompt import prompt_attention
from echokv_amd.kernels.shared import (prefix_attention, prefix_workspace_bytes, shared_prefix_decode,
                                       shared_workspace_bytes)
from echokv_amd.tiered_cache import TieredKVCache, TieredLayout

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


class Cache:
    """A store with a prefix of ``prefix`` tokens that every sequence begins with, and each
    sequence's own ``tails`` tokens behind it."""

    def __init__(self, device, prefix, tails, h=2, d=128, bs=16, kg=16, vg=32, mem_bits=8, tiers=(4,), dtype=F16,
                 seed=0, outliers=False, spare=0):
        g = torch.Generator(device=device)
        g.manual_seed(seed)
        rng = np.random.default_rng(seed)
        self.prefix, self.tails, self.h, self.d, self.bs, self.device = prefix, tails, h, d, bs, device
        shared = -(-prefix // bs)
        own = [-(-n // bs) for n in tails]
        nb = shared + sum(own) + 3 + spare
        perm = rng.permutation(nb)
        self.table_np = np.full((max(1, len(tails)), shared + max(own, default=0) + 1), perm[-1], np.int64)
        self.table_np[:, :shared] = perm[:shared]
        o = shared
        for i, n in enumerate(own):
            self.table_np[i, shared : shared + n] = perm[o : o + n]
            o += n
        layout = TieredLayout(h, d, bs, mem_bits, kg, vg)
        per = TieredLayout.per_token_bytes(h, d, mem_bits, kg, vg)
        pages = torch.zeros(nb, bs * per, dtype=torch.uint8, device=device)
        self.store = TieredKVCache(layout, pages, residual_slots=len(tails) + 4, residual_dtype=dtype)
        w = torch.ones(2, h, d, device=device)
        if outliers:
            w[:, :, :: 37] = 10.0

        def put(row, first, n, tier):
            k, v = (torch.randn(n, h, d, device=device, generator=g) * x for x in w)
            p = np.arange(first, first + n)
            slots = self.table_np[row][p // bs] * bs + p % bs
            self.store.write(k.to(dtype), v.to(dtype), torch.from_numpy(slots), tier)

        def put_blocks(row, first, n):  # block by block through the tiers
            for i, b in enumerate(range(0, n, bs)):
                put(row, first + b, min(bs, n - b), tiers[(first // bs + i) % len(tiers)])

        if len(tiers) == 1:
            if prefix:
                put(0, 0, prefix, tiers[0])
            for i, n in enumerate(tails):
                if n:
                    put(i, shared * bs, n, tiers[0])
        else:
            put_blocks(0, 0, prefix)
            for i, n in enumerate(tails):
                put_blocks(i, shared * bs, n)
        self.table = torch.from_numpy(self.table_np).to(device, torch.int32)
        self.blocks = self.table[0, : max(1, shared)].contiguous()
        self.lens = [prefix + n for n in tails]

    def tokens(self, row, n):
        p = np.arange(n)
        blk = torch.from_numpy(self.table_np[row][p // self.bs]).to(self.device)
        return self.store.gather(blk, torch.from_numpy(p % self.bs).to(self.device))

    def queries(self, n, gqa, dtype, seed=1):
        g = torch.Generator(device=self.device)
        g.manual_seed(seed)
        return torch.randn(n, self.h * gqa, self.d, device=self.device, generator=g).to(dtype)


# The matrix kernels take weights and values in float16, keys and float32 queries as two
# float16 parts (2^-22 of the value together, subnormal low parts 2^-25 of a unit).
BOUND = dict(weight=unit(F16), value=unit(F16), operands=2.0 ** -20)


def check_prefix(c, q, part, lse, n, scale):
    k, v = c.tokens(0, n)
    r = Rows(q, k, v, [n] * q.shape[0], scale)
    check(part, r, **BOUND)
    if n:
        assert float((lse.double() - r.lse).abs().max()) <= r.lse_bound(BOUND["operands"])
    else:
        assert (part == 0).all() and (lse == float("-inf")).all()


LAYOUTS = [dict(), dict(bs=64, kg=32, vg=64), dict(d=64), dict(d=256), dict(d=96, vg=24), dict(d=20, vg=4, kg=8),
           dict(bs=48, kg=16), dict(vg=4, h=3), dict(bs=128, kg=64, h=8)]


@pytest.mark.parametrize("kw", LAYOUTS, ids=str)
@pytest.mark.parametrize("tiers", [(4,), (8,), (2,), (4, 8, 2)], ids=str)
def test_prefix_matches_float64(device, kw, tiers):
    print(f"[prefix] {kw} {tiers}", flush=True)
    bs = kw.get("bs", 16)
    c = Cache(device, 7 * bs + 5, [], tiers=tiers, outliers=True, **kw)
    for gqa, rows, dtype in ((1, 1, F16), (4, 5, BF16), (7, 40, F16), (4, 3, F32)):
        q = c.queries(rows, gqa, dtype, seed=rows)
        for n in (0, 1, bs - 1, bs, 4 * bs + 3, 7 * bs + 5):  # the last: with the open K group
            part, lse = prefix_attention(c.store, q, c.blocks, n, c.d ** -0.5)
            torch.cuda.synchronize()
            check_prefix(c, q, part, lse, n, c.d ** -0.5)


@pytest.mark.parametrize("rows,gqa", [(1, 1), (3, 4), (64, 4), (65, 4), (300, 4), (33, 20)])
@pytest.mark.parametrize("n", [128, 129, 1000, 4096])
def test_prefix_rows_and_ranges(device, rows, gqa, n):
    print(f"[prefix] rows {rows} gqa {gqa} n {n}", flush=True)
    c = Cache(device, n, [], bs=64, kg=32, seed=n)
    q = c.queries(rows, gqa, BF16)
    part, lse = prefix_attention(c.store, q, c.blocks, n, c.d ** -0.5)
    torch.cuda.synchronize()
    check_prefix(c, q, part, lse, n, c.d ** -0.5)


@pytest.mark.parametrize("kw", [dict(), dict(d=64), dict(bs=64, kg=32, vg=64), dict(d=256)], ids=str)
@pytest.mark.parametrize("rows,n", [(4200, 200), (4200, 63), (300, 64), (300, 65), (300, 128), (300, 2100), (700, 1)])
def test_prefix_of_many_rows(device, kw, rows, n):
    """Rows enough that the prefix is dequantized into the workspace first, one range and several."""
    print(f"[prefix] many rows {kw} {rows} {n}", flush=True)
    c = Cache(device, n, [], tiers=(4,) if n > 500 else (4, 8, 2), outliers=True, seed=rows + n, **kw)
    for dtype in (BF16, F16):
        q = c.queries(rows, 4, dtype)
        part, lse = prefix_attention(c.store, q, c.blocks, n, c.d ** -0.5)
        torch.cuda.synchronize()
        check_prefix(c, q, part, lse, n, c.d ** -0.5)


@pytest.mark.parametrize("scale", [-0.088, 0.0, 0.9])
def test_prefix_scales(device, scale):
    c = Cache(device, 300, [], bs=64, kg=32)
    q = c.queries(9, 4, F16)
    part, lse = prefix_attention(c.store, q, c.blocks, 300, scale)
    torch.cuda.synchronize()
    check_prefix(c, q, part, lse, 300, scale)


def check_decode(c, q, got, lens, scale, rows=None):
    for i, n in enumerate(lens):
        if n < c.prefix or n == 0:
            continue
        k, v = c.tokens(i, n)
        j = i if rows is None else rows[i]
        r = Rows(q[j : j + 1], k, v, [n], scale)
        check(got[j : j + 1], r, **BOUND)


@pytest.mark.parametrize("kw", LAYOUTS, ids=str)
@pytest.mark.parametrize("tiers", [(4,), (8,), (2,), (4, 8)], ids=str)
def test_decode_matches_float64(device, kw, tiers):
    print(f"[shared] {kw} {tiers}", flush=True)
    bs = kw.get("bs", 16)
    tails = [1, bs, 5 * bs + 3, 0, 2, 40]
    c = Cache(device, 5 * bs, tails, tiers=tiers, **kw)
    lens = torch.tensor(c.lens, device=device)
    mask = "auto" if len(tiers) > 1 and c.d in (64, 128) and kw.get("bs", 16) != 48 else None
    for gqa, dtype in ((1, F16), (4, BF16), (7, F16), (20, F16), (4, F32)):
        q = c.queries(len(tails), gqa, dtype, seed=gqa)
        out = torch.full_like(q, 9.0)
        shared_prefix_decode(c.store, q, c.table, lens, c.prefix, c.d ** -0.5, out=out, tier_mask=mask)
        torch.cuda.synchronize()
        check_decode(c, q, out, c.lens, c.d ** -0.5)


@pytest.mark.parametrize("seqs", [1, 2, 17, 64, 130, 260])
@pytest.mark.parametrize("prefix", [64, 1024, 8192])
def test_decode_batches(device, seqs, prefix):
    print(f"[shared] {seqs} behind {prefix}", flush=True)
    tails = [1 + (37 * i) % 150 for i in range(seqs)]
    c = Cache(device, prefix, tails, h=4, bs=64, kg=32, dtype=BF16, seed=seqs, outliers=True)
    q = c.queries(seqs, 4, BF16)
    got = shared_prefix_decode(c.store, q, c.table, torch.tensor(c.lens, device=device), prefix, c.d ** -0.5)
    plain = dec.decode_attention(c.store, q, c.table, torch.tensor(c.lens, device=device), c.d ** -0.5)
    torch.cuda.synchronize()
    assert got.dtype == torch.float32
    check_decode(c, q, got, c.lens, c.d ** -0.5)
    # Plain decode is within 2e-3 of the exact result, this one within its bound: they differ by
    # both at most. (2e-3 does not hold here: values reach 40, where float16's half step is 2^-7.)
    for i, n in enumerate(c.lens):
        r = Rows(q[i : i + 1], *c.tokens(i, n), [n], c.d ** -0.5)
        assert ((got[i : i + 1] - plain[i : i + 1]).abs().double() <= r.bound(F32, **BOUND) + 2e-3).all()


def test_decode_rows_of_other_sequences_stay(device):
    """Padding (length 0), sequences shorter than the prefix, and rows that no sequence names."""
    print("[shared] rows", flush=True)
    c = Cache(device, 64, [30, 5, 8, 100], bs=16)
    q = c.queries(9, 4, F16)
    q_rows, bt_rows = [7, 0, 3, 5, 2, 8], [2, 1, 0, 3, 1, 1]
    lens = [64 + 8, 64 + 5, 64 + 30, 64 + 100, 0, 63]
    out = torch.full_like(q, 9.0)
    shared_prefix_decode(c.store, q, c.table, torch.tensor(lens, device=device), 64, c.d ** -0.5, out=out,
                         q_rows=torch.tensor(q_rows, device=device), bt_rows=torch.tensor(bt_rows, device=device),
                         blocks=c.blocks)
    torch.cuda.synchronize()
    for qr, br, n in list(zip(q_rows, bt_rows, lens))[:4]:
        k, v = c.tokens(br, n)
        check(out[qr : qr + 1], Rows(q[qr : qr + 1], k, v, [n], c.d ** -0.5), **BOUND)
    for row in (1, 2, 4, 6, 8):
        assert (out[row] == 9.0).all()


@pytest.mark.parametrize("d,seqs,prefix", [(128, 6, 64), (96, 6, 64), (128, 200, 4096)])
def test_padding_may_name_any_row(device, d, seqs, prefix):
    """Entries of length 0 or shorter than the prefix: their row indices are not followed."""
    print(f"[shared] padding {d} {seqs}", flush=True)
    c = Cache(device, prefix, [30, 5], d=d, vg=32 if d == 128 else 24)
    q = c.queries(2, 4, F16)
    q_rows, bt_rows, lens = [0, 1], [1, 0], [prefix + 5, prefix + 30]
    for i in range(seqs - 2):
        q_rows.append((-1, 1 << 40, -(1 << 40))[i % 3])
        bt_rows.append((1 << 40, -1, 7)[i % 3])
        lens.append((0, prefix - 1)[i % 2])
    out = torch.zeros_like(q)
    shared_prefix_decode(c.store, q, c.table, torch.tensor(lens, device=device), prefix, c.d ** -0.5, out=out,
                         q_rows=torch.tensor(q_rows, device=device), bt_rows=torch.tensor(bt_rows, device=device),
                         blocks=c.blocks)
    torch.cuda.synchronize()
    for row in range(2):
        k, v = c.tokens(bt_rows[row], lens[row])
        check(out[row : row + 1], Rows(q[row : row + 1], k, v, [lens[row]], c.d ** -0.5), **BOUND)


@pytest.mark.parametrize("d,dtype", [(128, F16), (128, BF16), (128, F32), (96, F16)], ids=str)
@pytest.mark.parametrize("prefix,rows", [(64, 3), (4096, 3), (4096, 200)])
def test_nan_queries_and_scales(device, d, dtype, prefix, rows):
    """A NaN in a query row, or as the softmax scale, makes its rows NaN and no others."""
    print(f"[shared] nan {d} {prefix} {rows}", flush=True)
    c = Cache(device, prefix, [0] * rows, d=d, vg=32 if d == 128 else 24)
    q = c.queries(rows, 4, dtype)
    q[1, 2, 5] = float("nan")
    bad = torch.zeros(rows, q.shape[1], dtype=torch.bool, device=device)
    bad[1, 2] = True
    lens = torch.tensor(c.lens, device=device)
    for scale, want in ((c.d ** -0.5, bad), (float("nan"), torch.ones_like(bad))):
        part, lse = prefix_attention(c.store, q, c.blocks, prefix, scale)
        out = shared_prefix_decode(c.store, q, c.table, lens, prefix, scale)
        torch.cuda.synchronize()
        assert torch.equal(lse.isnan(), want)
        for rows_out in (part, out):
            assert torch.equal(rows_out.isnan().all(-1), want) and torch.equal(rows_out.isnan().any(-1), want)


@pytest.mark.parametrize("d,seqs,prefix", [(128, 3, 512), (96, 3, 512), (128, 200, 4096)])
def test_pages_past_32_bits(device, d, seqs, prefix):
    """Blocks all over a cache of more than 2^32 bytes."""
    print(f"[shared] far pages {d} {seqs}", flush=True)
    h, vg = 8, 32 if d == 128 else 24
    spare = (6 << 30) // (16 * TieredLayout.per_token_bytes(h, d, 8, 16, vg))
    c = Cache(device, prefix, [5] * seqs, h=h, d=d, vg=vg, spare=spare)
    assert int(c.table_np.max()) * c.store.layout.page_bytes > 1 << 32
    q = c.queries(seqs, 4, F16)
    part, lse = prefix_attention(c.store, q, c.blocks, prefix, c.d ** -0.5)
    out = shared_prefix_decode(c.store, q, c.table, torch.tensor(c.lens, device=device), prefix, c.d ** -0.5)
    torch.cuda.synchronize()
    check_prefix(c, q[:3], part[:3], lse[:3], prefix, c.d ** -0.5)
    for i in (0, seqs - 1):
        k, v = c.tokens(i, c.lens[i])
        check(out[i : i + 1], Rows(q[i : i + 1], k, v, [c.lens[i]], c.d ** -0.5), **BOUND)


@pytest.mark.parametrize("d,dtype,seqs,prefix", [(128, F16, 5, 512), (128, F32, 5, 512), (96, BF16, 5, 512),
                                                 (128, BF16, 200, 4096), (256, F16, 5, 64)], ids=str)
def test_odd_strides(device, d, dtype, seqs, prefix):
    """Queries, outputs and parts whose rows are aligned to one element."""
    print(f"[shared] odd strides {d} {dtype} {seqs}", flush=True)
    c = Cache(device, prefix, [5] * seqs, d=d, vg=24 if d == 96 else 32)
    q = c.queries(seqs, 4, dtype)

    def odd(x, t):
        y = torch.full((x.shape[0], x.shape[1] + 1, d + 3), 7.0, dtype=t, device=device)
        return y, y[:, 1:, 1 : d + 1]

    qw, qo = odd(q, dtype)
    qo.copy_(q)
    lens = torch.tensor(c.lens, device=device)
    part, lse = prefix_attention(c.store, q, c.blocks, prefix, c.d ** -0.5)
    pw, po = odd(q, F32)
    prefix_attention(c.store, qo, c.blocks, prefix, c.d ** -0.5, part=po)
    out = shared_prefix_decode(c.store, q, c.table, lens, prefix, c.d ** -0.5, out=torch.empty_like(q))
    ow, oo = odd(q, dtype)
    shared_prefix_decode(c.store, qo, c.table, lens, prefix, c.d ** -0.5, out=oo)
    torch.cuda.synchronize()
    assert torch.equal(po, part) and torch.equal(oo, out)
    for w in (pw, ow):
        assert (w[:, 0] == 7).all() and (w[:, 1:, 0] == 7).all() and (w[:, 1:, d + 1 :] == 7).all()


@pytest.mark.parametrize("prefix", [64, 4096])
def test_large_gqa(device, prefix):
    """More query heads a KV head than a workgroup has rows."""
    print(f"[shared] gqa 300, {prefix}", flush=True)
    c = Cache(device, prefix, [30, 5], h=1)
    q = c.queries(2, 300, F16)
    part, lse = prefix_attention(c.store, q, c.blocks, prefix, c.d ** -0.5)
    out = shared_prefix_decode(c.store, q, c.table, torch.tensor(c.lens, device=device), prefix, c.d ** -0.5)
    torch.cuda.synchronize()
    check_prefix(c, q, part, lse, prefix, c.d ** -0.5)
    check_decode(c, q, out, c.lens, c.d ** -0.5)


def test_two_streams_at_once(device):
    """Calls on two streams side by side: each has a workspace of its own."""
    print("[shared] two streams", flush=True)
    c = Cache(device, 4096, [60, 33, 1, 90] * 16)
    qs = [c.queries(64, 4, F16, seed=i) for i in range(2)]
    lens = torch.tensor(c.lens, device=device)
    alone = [shared_prefix_decode(c.store, q, c.table, lens, 4096, 0.088) for q in qs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in qs], [[], []]
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(shared_prefix_decode(c.store, qs[i], c.table, lens, 4096, 0.088))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, alone[i]) for x in got[i])


@pytest.mark.parametrize("d,rows,prefix", [(128, 5, 500), (128, 60, 8192), (96, 5, 500), (128, 200, 4096)])
def test_blocks_outside_the_cache_are_zeros(device, d, rows, prefix):
    print(f"[shared] blocks outside {d} {rows}", flush=True)
    c = Cache(device, prefix, [], d=d, vg=24 if d == 96 else 32)
    q = c.queries(rows, 4, F16)
    bad = {3: -1, 7: c.store.pages.shape[0], 20: 1 << 30}
    blocks = c.blocks.clone()
    for i, b in bad.items():
        blocks[i] = b
    part, lse = prefix_attention(c.store, q, blocks, prefix, c.d ** -0.5)
    torch.cuda.synchronize()
    k, v = c.tokens(0, prefix)
    for i in bad:
        k[i * c.bs : (i + 1) * c.bs] = 0
        v[i * c.bs : (i + 1) * c.bs] = 0
    r = Rows(q[:8], k, v, [prefix] * min(8, rows), c.d ** -0.5)
    check(part[:8], r, **BOUND)
    assert float((lse[:8].double() - r.lse).abs().max()) <= r.lse_bound(BOUND["operands"])


def test_no_prefix_is_plain_decode(device):
    c = Cache(device, 0, [30, 5], bs=16)
    q = c.queries(2, 4, F16)
    lens = torch.tensor(c.lens, device=device)
    got = shared_prefix_decode(c.store, q, c.table, lens, 0, 0.088)
    assert torch.equal(got, dec.decode_attention(c.store, q, c.table, lens, 0.088))


def test_workspaces(device):
    """A workspace of the call's own and a caller's give the same bits; a smaller one is refused."""
    c = Cache(device, 512, [30, 5, 1], bs=16)
    q = c.queries(3, 4, F16)
    lens = torch.tensor(c.lens, device=device)
    args = (c.store, q, c.table, lens, 512, 0.088)
    need = shared_workspace_bytes(c.store, 8, 3, 512, 4)
    ws = torch.full((need + 64,), 0xFF, dtype=torch.uint8, device=device)  # NaN bits
    a = shared_prefix_decode(*args, num_splits=4)
    b = shared_prefix_decode(*args, num_splits=4, workspace=ws)
    assert torch.equal(a, b)
    with pytest.raises(ValueError):
        shared_prefix_decode(*args, num_splits=4, workspace=ws[: need - 1])
    need = prefix_workspace_bytes(c.store, 8, 3, 512)
    assert need > 0
    pa = prefix_attention(c.store, q, c.blocks, 512, 0.088)
    pb = prefix_attention(c.store, q, c.blocks, 512, 0.088, workspace=ws[:need])
    assert torch.equal(pa[0], pb[0]) and torch.equal(pa[1], pb[1])
    with pytest.raises(ValueError):
        prefix_attention(c.store, q, c.blocks, 512, 0.088, workspace=ws[: need - 1])


def test_graphs_replay_beside_each_other(device):
    """Two captured decodes and the eager call, replayed in turn with the lengths changing."""
    print("[shared] graphs", flush=True)
    c = Cache(device, 256, [60, 33, 1, 90], bs=16)
    q = [c.queries(4, 4, F16, seed=i) for i in range(2)]
    out = [torch.zeros_like(x) for x in q]
    lens = torch.tensor(c.lens, device=device)

    def call(i, o):
        shared_prefix_decode(c.store, q[i], c.table, lens, 256, 0.088, out=o, tier=4)

    call(0, out[0])
    torch.cuda.synchronize()
    graphs = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(i, out[i])
        graphs.append(g)
    for rep in range(4):
        lens.copy_(torch.tensor([max(256, n - 7 * rep) for n in c.lens], device=device))
        for o in out:
            o.zero_()
        graphs[0].replay()
        graphs[1].replay()
        for i in range(2):
            eager = torch.zeros_like(out[i])
            call(i, eager)
            torch.cuda.synchronize()
            assert torch.equal(eager, out[i]), (rep, i)


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 64), (F32, 96)], ids=str)
def test_prompts_behind_a_shared_prefix(device, dtype, d):
    """The two operators together: new prompts behind a cached prefix."""
    print(f"[joined] {dtype} D{d}", flush=True)
    pre, lens, gqa = 200, [90, 1, 33], 4
    c = Cache(device, pre, [], d=d, vg=16 if d != 96 else 24)
    t = sum(lens)
    q = c.queries(t, gqa, dtype)
    g = torch.Generator(device=device)
    g.manual_seed(3)
    k, v = (torch.randn(t, c.h, d, device=device, generator=g).to(dtype) for _ in range(2))
    entries, o = [], 0
    for n in lens:
        entries.append((o, o + n))
        o += n
    prefix = prefix_attention(c.store, q, c.blocks, pre, d ** -0.5)
    out = torch.empty_like(q)
    prompt_attention(q, k, v, out, entries, d ** -0.5, prefix=prefix)
    torch.cuda.synchronize()
    kp, vp = c.tokens(0, pre)
    for a, b in entries:
        kk, vv = (torch.cat([x.double(), y[a:b].double()]) for x, y in ((kp, k), (vp, v)))
        r = Rows(q[a:b], kk, vv, range(pre + 1, pre + b - a + 1), d ** -0.5)
        check(out[a:b], r, weight=max(unit(F16), unit(dtype)), value=unit(F16), operands=2.0 ** -20)
