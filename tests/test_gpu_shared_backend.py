"""GPU: the backend with ECHOKV_PROMPT_EXACT=1 and ECHOKV_SHARED_PREFIX=1 -- a prompt alone, then
prompts behind its cached blocks in a step with its own decode, then shared decode steps -- against
float64 over this step's keys and values and over the cache's."""

import numpy as np
import pytest
import torch

from attend64 import Rows, check, unit
from echokv_amd import _vllm
from test_gpu_backend import D, H, HQ, LAYERS, Batch, check_decode, make_engine, run_layers, slots_for

pytestmark = pytest.mark.gpu

BS = 16
PREFIX = 1024
F16 = torch.float16


@pytest.fixture
def settings(monkeypatch):
    for k, v in {"ECHOKV_K_GROUP": "16", "ECHOKV_MEM_BITS": "8", "ECHOKV_RESIDUAL_SLOTS": "24",
                 "ECHOKV_PROMPT_EXACT": "1", "ECHOKV_SHARED_PREFIX": "1"}.items():
        monkeypatch.setenv(k, v)
    yield monkeypatch
    _vllm.set_forward_metadata(None)


def cached(impl, table_row, n):
    p = np.arange(n)
    dev = impl.store.device
    return impl.store.gather(torch.from_numpy(table_row[p // BS]).to(dev), torch.from_numpy(p % BS).to(dev))


@pytest.mark.parametrize("invariant", ["1", "0"])
def test_serving_behind_a_shared_prefix(device, settings, invariant):
    settings.setenv("ECHOKV_BATCH_INVARIANT", invariant)
    rng = np.random.default_rng(3)
    builder, layers, pool = make_engine(device, tiers=[4, 8, 2])
    perm = rng.permutation(128)
    shared = PREFIX // BS
    table_np = np.zeros((4, shared + 12), np.int64)
    table_np[:, :shared] = perm[:shared]
    table_np[:, shared:] = perm[shared : shared + 48].reshape(4, 12)
    table = torch.from_numpy(table_np).to(device, torch.int32)
    gen = torch.Generator(device=device)
    gen.manual_seed(5)

    def rand(n, heads):
        return [torch.randn(n, heads, D, device=device, generator=gen).half() for _ in range(LAYERS)]

    # A whole prompt: its own keys and values, nothing read back from the cache.
    n0 = PREFIX + 40
    print("[shared backend] prompt", flush=True)
    md = builder.build(0, Batch(device, table, [0, n0], [n0], slots_for(table_np, [0], [n0]), n0))
    assert md.prefill.prompts and not md.prefill.entries and md.prefill.prompts[0].prefix is None
    q, k, v = rand(n0, HQ), rand(n0, H), rand(n0, H)
    outs = run_layers(layers, md, q, k, v)
    torch.cuda.synchronize()
    for li in range(LAYERS):
        check(outs[li].view(-1, HQ, D), Rows(q[li], k[li], v[li], range(1, n0 + 1), D ** -0.5), weight=unit(F16))

    # Three prompts behind its first blocks, in a step with its decode and a chunk that continues
    # another context (read from the cache).
    new = [30, 1, 17]
    print("[shared backend] prompts behind the prefix", flush=True)
    q_lens = [1] + new
    lens = [n0 + 1] + [PREFIX + n for n in new]
    starts = np.concatenate([[0], np.cumsum(q_lens)])
    t = int(starts[-1])
    slots = slots_for(table_np, [n0] + [PREFIX] * 3, q_lens)
    assert builder.use_cascade_attention(PREFIX, q_lens, HQ, H)
    md = builder.build(PREFIX, Batch(device, table, starts, lens, slots, t))
    # (a prompt of one new token is a decode entry)
    assert md.decode.prefix.tokens == PREFIX and md.decode.lens.shape[0] == 2
    assert [w.prefix.tokens for w in md.prefill.prompts] == [PREFIX] and not md.prefill.entries
    q, k, v = rand(t, HQ), rand(t, H), rand(t, H)
    outs = run_layers(layers, md, q, k, v)
    torch.cuda.synchronize()
    for li, layer in enumerate(layers):
        out = outs[li].view(-1, HQ, D)
        for r in (1, 3):
            a, b = int(starts[r]), int(starts[r + 1])
            kp, vp = cached(layer.impl, table_np[r], PREFIX)
            keys, vals = (torch.cat([x.double(), y[li][a:b].double()]) for x, y in ((kp, k), (vp, v)))
            ref = Rows(q[li][a:b], keys, vals, range(PREFIX + 1, PREFIX + b - a + 1), D ** -0.5)
            check(out[a:b], ref, weight=unit(F16), value=unit(F16), operands=2.0 ** -20)
        for r in (0, 2):
            a = int(starts[r])
            keys, vals = cached(layer.impl, table_np[r], lens[r])
            ref = Rows(q[li][a : a + 1], keys, vals, [lens[r]], D ** -0.5)
            check(out[a : a + 1], ref, weight=unit(F16), value=unit(F16), operands=2.0 ** -20)

    # Decode steps of all four, padded to 6 rows; every other step without the common prefix.
    bt = torch.cat([table, torch.zeros(2, table.shape[1], dtype=table.dtype, device=device)])
    for layer, bits in zip(layers, (8, 2, 4)):
        layer.impl.controller.bits = bits  # blocks opened from now on: layers of two tiers
    for step in range(20):
        slots = np.concatenate([slots_for(table_np, lens, [1] * 4), -np.ones(2, np.int64)])
        lens = [x + 1 for x in lens]
        common = PREFIX if step % 2 == 0 else 0
        md = builder.build(common, Batch(device, bt, np.arange(7), lens + [0, 0], slots, 6))
        assert (md.decode.prefix is not None) == (common > 0)
        q, k, v = rand(6, HQ), rand(6, H), rand(6, H)
        outs = run_layers(layers, md, q, k, v)
        torch.cuda.synchronize()
        if step in (0, 1, 18, 19):
            check_decode(layers, table_np, lens, q, outs, f"shared decode {step}")
        for out in outs:
            assert (out[4:] == 0).all()  # padding rows stay
    assert any(len([b for b, n in l.impl.store.pool.live_tiers().items() if n]) > 1 for l in layers)


def test_chunks_behind_other_contexts_take_the_cache(device, settings):
    """A chunk that continues a longer context than the prefix, beside a whole prompt."""
    builder, layers, pool = make_engine(device, tiers=[4, 4, 4])
    table_np = np.random.default_rng(1).permutation(128)[:120].reshape(2, 60).astype(np.int64)
    table = torch.from_numpy(table_np).to(device, torch.int32)
    gen = torch.Generator(device=device)
    gen.manual_seed(7)

    def rand(n, heads):
        return [torch.randn(n, heads, D, device=device, generator=gen).half() for _ in range(LAYERS)]

    md = builder.build(0, Batch(device, table, [0, 100], [100], slots_for(table_np, [0], [100]), 100))
    run_layers(layers, md, rand(100, HQ), rand(100, H), rand(100, H))
    q_lens, lens = [20, 50], [120, 50]
    md = builder.build(0, Batch(device, table, [0, 20, 70], lens, slots_for(table_np, [100, 0], q_lens), 70))
    assert len(md.prefill.prompts) == 1 and len(md.prefill.entries) == 1
    q, k, v = rand(70, HQ), rand(70, H), rand(70, H)
    outs = run_layers(layers, md, q, k, v)
    torch.cuda.synchronize()
    for li, layer in enumerate(layers):
        out = outs[li].view(-1, HQ, D)
        keys, vals = cached(layer.impl, table_np[0], 120)
        check(out[:20], Rows(q[li][:20], keys, vals, range(101, 121), D ** -0.5), weight=unit(F16), value=unit(F16),
              operands=2.0 ** -20)
        check(out[20:], Rows(q[li][20:], k[li][20:], v[li][20:], range(1, 51), D ** -0.5), weight=unit(F16))
