"""GPU: attention over a shared prefix for some of the query rows, and a step of the backend in which
another request's chunk lies between the prompts behind it; against float64."""

import numpy as np
import pytest
import torch

from attend64 import Rows, check, unit
from test_gpu_backend import D, H, HQ, LAYERS, Batch, make_engine, run_layers, slots_for
from test_gpu_shared_backend import BS, F16, PREFIX, cached, settings  # noqa: F401
from test_gpu_shared_prefix import BF16, BOUND, Cache, check_prefix

from echokv_amd.kernels import shared as sh

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,rows,prefix", [(128, 9, 64), (128, 9, 1000), (96, 9, 1000), (64, 700, 4096), (256, 9, 300)])
def test_named_rows_alone(device, d, rows, prefix):
    print(f"[rows] {d} {rows} {prefix}", flush=True)
    c = Cache(device, prefix, [], d=d, vg=24 if d == 96 else 32)
    q = c.queries(rows, 4, BF16)
    named = [rows - 1, 0, 4, rows // 3, 4]  # one of them twice
    if rows > 100:
        named += list(range(200, 650))
    index = torch.tensor(named, device=device)
    part, lse = torch.full_like(q, 7.0, dtype=torch.float32), torch.full(q.shape[:2], 7.0, device=device)
    sh.prefix_attention(c.store, q, c.blocks, prefix, d ** -0.5, part=part, lse=lse, q_rows=index)
    alone = sh.prefix_attention(c.store, q, c.blocks, prefix, d ** -0.5, q_rows=index.int())
    torch.cuda.synchronize()
    check_prefix(c, q[named], part[named], lse[named], prefix, d ** -0.5)
    rest = sorted(set(range(rows)) - set(named))
    assert (part[rest] == 7).all() and (lse[rest] == 7).all()
    assert torch.equal(alone[0][named], part[named]) and torch.equal(alone[1][named], lse[named])
    assert (alone[1][rest] == float("-inf")).all()
    none = sh.prefix_attention(c.store, q, c.blocks, prefix, d ** -0.5, part=part, q_rows=index[:0])
    assert (none[1] == float("-inf")).all() and (part[rest] == 7).all()


def test_an_odd_number_of_partial_rows(device):
    """Head size 256, one sequence of 7 heads behind 5 ranges: the suffix's rows come behind 35 pairs."""
    print("[rows] odd pairs", flush=True)
    c = Cache(device, 640, [40], h=1, d=256)
    q = c.queries(1, 7, F16)
    out = sh.shared_prefix_decode(c.store, q, c.table, torch.tensor(c.lens, device=device), 640, 0.06)
    torch.cuda.synchronize()
    check(out, Rows(q, *c.tokens(0, c.lens[0]), [c.lens[0]], 0.06), **BOUND)


def test_another_chunk_between_the_prompts(device, settings, monkeypatch):  # noqa: F811
    """A chunk that continues a longer context lies between two prompts behind the shared prefix."""
    builder, layers, pool = make_engine(device, tiers=[4, 4, 4])
    shared = PREFIX // BS
    perm = np.random.default_rng(4).permutation(128)
    table_np = np.zeros((3, shared + 12), np.int64)
    table_np[:, :shared] = perm[:shared]
    table_np[:, shared:] = perm[shared : shared + 36].reshape(3, 12)
    table = torch.from_numpy(table_np).to(device, torch.int32)
    gen = torch.Generator(device=device)
    gen.manual_seed(9)

    def rand(n, heads):
        return [torch.randn(n, heads, D, device=device, generator=gen).half() for _ in range(LAYERS)]

    n0 = PREFIX + 40  # request 1 has the prefix and 40 tokens of its own
    first = table_np[1:2]
    md = builder.build(0, Batch(device, table[1:2], [0, n0], [n0], slots_for(first, [0], [n0]), n0))
    run_layers(layers, md, rand(n0, HQ), rand(n0, H), rand(n0, H))
    q_lens, ctx = [30, 90, 17], [PREFIX, n0, PREFIX]
    starts = np.concatenate([[0], np.cumsum(q_lens)])
    lens, t = [a + b for a, b in zip(ctx, q_lens)], int(starts[-1])
    md = builder.build(PREFIX, Batch(device, table, starts, lens, slots_for(table_np, ctx, q_lens), t))
    assert len(md.prefill.prompts) == 1 and len(md.prefill.entries) == 1
    asked, plain = [], sh.prefix_attention

    def counted(store, q, *args, **kw):
        asked.append(q.shape[0] if kw.get("q_rows") is None else kw["q_rows"].shape[0])
        return plain(store, q, *args, **kw)

    monkeypatch.setattr(sh, "prefix_attention", counted)
    q, k, v = rand(t, HQ), rand(t, H), rand(t, H)
    outs = run_layers(layers, md, q, k, v)
    torch.cuda.synchronize()
    assert asked == [47] * LAYERS  # the prompts' rows, none of the chunk's
    for li, layer in enumerate(layers):
        out = outs[li].view(-1, HQ, D)
        for r in (0, 2):
            a, b = int(starts[r]), int(starts[r + 1])
            kp, vp = cached(layer.impl, table_np[r], PREFIX)
            keys, vals = (torch.cat([x.double(), y[li][a:b].double()]) for x, y in ((kp, k), (vp, v)))
            ref = Rows(q[li][a:b], keys, vals, range(PREFIX + 1, PREFIX + b - a + 1), D ** -0.5)
            check(out[a:b], ref, weight=unit(F16), value=unit(F16), operands=2.0 ** -20)
        a, b = int(starts[1]), int(starts[2])
        keys, vals = cached(layer.impl, table_np[1], lens[1])
        check(out[a:b], Rows(q[li][a:b], keys, vals, range(n0 + 1, n0 + 91), D ** -0.5), weight=unit(F16),
              value=unit(F16), operands=2.0 ** -20)
