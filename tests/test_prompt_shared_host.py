"""CPU: plans and refusals of prompt and shared-prefix attention; nothing here reaches a kernel."""

import ctypes as C
from types import SimpleNamespace

import pytest
import torch

from echokv_amd import _lib
from echokv_amd.kernels import shared as sh
from echokv_amd.kernels.prompt import build_prompt_plan, prompt_attention
from echokv_amd.tiered_cache import TieredLayout

CPU = torch.device("cpu")


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIB_PATH.exists():
        pytest.fail(f"{_lib.LIB_PATH} is not built")
    return _lib.lib()


def test_modules_under_the_reference_path():
    from echokv_vllm.kernels import prompt, shared

    assert prompt.prompt_attention is prompt_attention
    assert shared.shared_prefix_decode is sh.shared_prefix_decode


@pytest.mark.parametrize("gqa,d", [(1, 128), (4, 128), (7, 64), (300, 64), (4, 256), (4, 20)])
def test_plan_covers_every_row_once(lib, gqa, d):
    entries = [(5, 6), (10, 10), (20, 420), (7, 9), (500, 756)]
    plan = build_prompt_plan([(a, b, b - a, 0) for a, b in entries], gqa, d, CPU)
    seen = torch.zeros(800, dtype=torch.int64)
    for first, n, t0, tokens in plan.tiles.tolist():
        assert (first, first + n) in entries and 0 < tokens <= plan.tile_m and t0 + tokens <= n
        seen[first + t0 : first + t0 + tokens] += 1
    want = torch.zeros(800, dtype=torch.int64)
    for a, b in entries:
        want[a:b] = 1
    assert torch.equal(seen, want)
    assert plan.rows == 756
    keys = (plan.tiles[:, 2] + plan.tiles[:, 3]).tolist()
    assert keys == sorted(keys, reverse=True)


@pytest.mark.parametrize("entries", [[(3, 2)], [(0, 1 << 31)], [(-1, 4)], [(0, 10), (5, 20)], [(0, 4), (0, 4)], [(0, 9), (2, 3)]])
def test_plan_refuses_bad_rows(lib, entries):
    with pytest.raises(ValueError):
        build_prompt_plan(entries, 4, 128, CPU)


@pytest.mark.parametrize("d", [0, 3, 130, 260, 512])
def test_plan_refuses_head_sizes(lib, d):
    with pytest.raises(ValueError):
        build_prompt_plan([(0, 4)], 4, d, CPU)


def _qkv(t=8, hq=8, h=2, d=128, dtype=torch.bfloat16):
    return torch.zeros(t, hq, d, dtype=dtype), torch.zeros(t, h, d, dtype=dtype), torch.zeros(t, h, d, dtype=dtype)


def test_prompt_refuses_shapes_and_types(lib):
    q, k, v = _qkv()
    out = torch.empty_like(q)
    for bad in ((q, k, v[:4], out), (q, k[:, :1].expand(-1, 3, -1), v[:, :1].expand(-1, 3, -1), out),
                (q, k.half(), v, out), (q, k, v.float(), out), (q, k[..., :64], v[..., :64], out),
                (q[0], k, v, out), (q, k, v, out[:, :4]), (q, k, v, out.transpose(1, 2))):
        with pytest.raises((ValueError, RuntimeError)):
            prompt_attention(*bad, [(0, 8)], 0.1)
    with pytest.raises(RuntimeError, match="device"):  # never a fallback
        prompt_attention(q, k, v, out, [(0, 8)], 0.1)


def _prompt(lib, **kw):
    p = C.c_void_p(64)  # never dereferenced: every call below fails its checks first
    a = dict(dtype=_lib.BF16, hq=32, h=8, d=128, tiles=p, n=1, tile_m=32, part=None, part_lse=None, out=p, od=_lib.F16)
    a.update(kw)
    return lib.echokv_prompt(p, 4096, 128, p, 1024, 128, p, 1024, 128, a["dtype"], a["hq"], a["h"], a["d"], a["tiles"],
                             a["n"], a["tile_m"], 0.1, a["part"], 4096, 128, a["part_lse"], a["out"], 4096, 128, a["od"],
                             None, None)


def test_prompt_entry_rejects_bad_arguments(lib):
    assert lib.echokv_prompt_tile_m(32, 8, 128) == 32
    for bad in ((30, 8, 128), (32, 0, 128), (32, 8, 260), (32, 8, 30)):
        assert lib.echokv_prompt_tile_m(*bad) == -2
    for kw, code in ((dict(hq=30), 2), (dict(d=512), 2), (dict(tile_m=64), 2), (dict(dtype=7), 3), (dict(od=-1), 3),
                     (dict(n=-1), 1), (dict(n=1 << 40), 1), (dict(tiles=None), 1), (dict(out=None), 1),
                     (dict(part=C.c_void_p(64)), 1), (dict(n=0), 0)):
        assert _prompt(lib, **kw) == code, kw


def _layout(**kw):
    lay = TieredLayout(8, 128, 16, 8, 16, 32)
    L = lay.abi(100, lay.page_bytes)
    for k, v in kw.items():
        setattr(L, k, v)
    return L


def _shared(lib, entry, L=None, **kw):
    L = L if L is not None else _layout()
    p = C.c_void_p(64)
    res = _lib.Residual(C.c_void_p(16), 1, 2, 16 * 8 * 128, 8 * 128, 128)
    a = dict(dtype=_lib.F16, hq=32, n=4, blocks=p, prefix=64, splits=4, bps=16, tier=4, ws=p, bytes=1 << 40, out=p,
             od=_lib.F16, lse=p)
    a.update(kw)
    if entry == "prefix":
        return lib.echokv_prefix(C.byref(L), p, p, p, C.byref(res), p, 4096, 128, a["dtype"], a["hq"], None, a["n"],
                                 a["blocks"], a["prefix"], 0.1, a["ws"], a["bytes"], a["out"], 4096, 128, a["lse"],
                                 None)
    return lib.echokv_shared_decode(C.byref(L), p, p, p, C.byref(res), p, 4096, 128, a["dtype"], a["hq"], None, p, 64,
                                    None, p, a["n"], a["blocks"], a["prefix"], 0.1, a["splits"], a["bps"], a["tier"],
                                    None, a["ws"], a["bytes"], a["out"], 4096, 128, a["od"], None)


def test_prefix_entry_rejects_bad_arguments(lib):
    for kw, code in ((dict(hq=30), 2), (dict(n=-1), 2), (dict(prefix=-1), 2), (dict(prefix=1 << 40), 2), (dict(n=1 << 40), 2),
                     (dict(prefix=(1 << 31) - 16384), 2),
                     (dict(dtype=5), 3), (dict(blocks=None), 1), (dict(out=None), 1), (dict(lse=None), 1),
                     (dict(prefix=4096, bytes=1000), 1), (dict(prefix=4096, ws=None), 1),
                     (dict(prefix=4096, ws=C.c_void_p(8)), 1), (dict(n=0), 0)):
        assert _shared(lib, "prefix", **kw) == code, kw
    assert _shared(lib, "prefix", _layout(block_size=24)) == 2


def test_shared_entry_rejects_bad_arguments(lib):
    for kw, code in ((dict(hq=30), 2), (dict(n=-1), 2), (dict(prefix=0), 1), (dict(prefix=63), 1), (dict(splits=0), 1),
                     (dict(n=1 << 20, splits=1 << 20, bytes=1 << 62), 2),
                     (dict(splits=1 << 30), 1), (dict(bps=0), 1), (dict(tier=3), 1), (dict(dtype=5), 3), (dict(od=5), 3),
                     (dict(blocks=None), 1), (dict(out=None), 1), (dict(bytes=100), 1), (dict(ws=None), 1),
                     (dict(ws=C.c_void_p(8)), 1), (dict(n=0), 0)):
        assert _shared(lib, "decode", **kw) == code, kw


def test_shared_python_refusals(lib):
    lay = TieredLayout(2, 128, 16, 8, 16, 32)
    store = SimpleNamespace(layout=lay, abi=lay.abi(100, lay.page_bytes), pages=torch.zeros(1), res_k=None)
    q, table, lens = torch.zeros(3, 8, 128), torch.zeros(3, 8, dtype=torch.int32), torch.full((3,), 70)
    with pytest.raises(RuntimeError, match="device"):
        sh.shared_prefix_decode(store, q, table, lens, 64, 0.1)
    for bad in ((q, table, lens, 60), (q, table, lens, -16), (q[..., :64], table, lens, 64), (q[:, :3], table, lens, 64)):
        with pytest.raises(ValueError):
            sh.shared_prefix_decode(store, *bad, 0.1)
    two = torch.zeros(2, dtype=torch.int64)
    for kw in (dict(q_rows=two), dict(bt_rows=two), dict(out=torch.zeros(2, 8, 128)),
               dict(out=torch.zeros(0, 8, 128), q_rows=torch.zeros(3))):
        with pytest.raises(ValueError):
            sh.shared_prefix_decode(store, q, table, lens, 64, 0.1, **kw)
    with pytest.raises(ValueError, match="block-table"):
        sh.shared_prefix_decode(store, q, table[:2], lens, 64, 0.1)
    with pytest.raises(ValueError):
        sh.prefix_attention(store, q, table[0], -1, 0.1)
    with pytest.raises(ValueError):
        sh._blocks(store, table[0, :3], 64)
    assert sh._blocks(store, table[0], 49).numel() == 4
    with pytest.raises(ValueError):
        sh._workspace(torch.zeros(10, dtype=torch.uint8), 11, CPU)
    assert [sh.suffix_blocks(store, n) for n in (1, 64, 65)] == [8, 8, 16]
    assert sh.suffix_splits(8, 16, 64, 16, None) == 4
    assert sh.suffix_splits(4096, 16, 64, 16, None) == 64


# ---- the backend's side ----------------------------------------------------------------

def _builder(monkeypatch, **env):
    from echokv_amd.backend import EchoKVMetadataBuilder

    for k, v in env.items():
        monkeypatch.setenv(k, v)
    cfg = SimpleNamespace(model_config=SimpleNamespace(max_model_len=4096, dtype=torch.float16,
                                                       get_num_attention_heads=lambda pc: 8),
                          parallel_config=None, scheduler_config=SimpleNamespace(max_num_seqs=8),
                          compilation_config=SimpleNamespace(max_cudagraph_capture_size=8), speculative_config=None)
    spec = SimpleNamespace(block_size=64, num_kv_heads=2, head_size=128)
    return EchoKVMetadataBuilder(spec, ["l"], cfg, CPU)


def test_settings_are_off_by_default(monkeypatch):
    from echokv_amd.config import load_config

    for k in ("ECHOKV_PROMPT_EXACT", "ECHOKV_SHARED_PREFIX"):
        monkeypatch.delenv(k, raising=False)
    cfg = load_config()
    assert not cfg.prompt_exact and not cfg.shared_prefix
    assert load_config({"ECHOKV_PROMPT_EXACT": "1"}).prompt_exact
    assert load_config({"ECHOKV_SHARED_PREFIX": "1"}).shared_prefix
    b = _builder(monkeypatch)
    assert not b.use_cascade_attention(8192, [1, 1, 1], 8, 2, False, False, False, 256)


def test_cascade_is_taken_from_the_measured_length_on(monkeypatch):
    b = _builder(monkeypatch, ECHOKV_SHARED_PREFIX="1")
    assert b.use_cascade_attention(1024, [1, 1], 8, 2, False, False, False, 256, dcp_world_size=1)
    assert not b.use_cascade_attention(960, [1, 1], 8, 2)
    assert not b.use_cascade_attention(4096, [1], 8, 2)


def test_shared_prefix_of_a_step(monkeypatch):
    """Whole blocks, before every live request's first query token; padding rows do not count."""
    import numpy as np

    b = _builder(monkeypatch, ECHOKV_SHARED_PREFIX="1")
    table = torch.arange(4 * 40).view(4, 40)
    cm = SimpleNamespace(block_table_tensor=table)

    def of(starts, lens, common):
        return b._shared(cm, torch.tensor(lens), np.array(starts, np.int32), common)

    p = of([0, 0, 1, 8], [0, 2000, 1500], 1100)  # row 0 is padding
    assert p.tokens == 1088 and p.blocks.tolist() == list(range(40, 57)) and p.blocks.dtype == torch.int32
    assert of([0, 1, 11], [2000, 1098], 1088).tokens == 1088
    assert of([0, 1, 11], [2000, 1097], 1088).tokens == 1024  # 1087 cached: 16 whole blocks
    assert of([0, 1, 11], [2000, 1033], 1088) is None  # 1023 cached: 15, below the measured length
    assert of([0, 1, 11], [2000, 1100], 0) is None
    assert of([0, 0], [0], 2048) is None
    assert _builder(monkeypatch, ECHOKV_SHARED_PREFIX="0")._shared(cm, torch.tensor([2000]), np.array([0, 1]), 1088) is None


def test_prompt_chunks_are_told_apart(lib, monkeypatch):
    from echokv_amd.backend import SharedPrefix

    b = _builder(monkeypatch, ECHOKV_SHARED_PREFIX="1", ECHOKV_PROMPT_EXACT="1")
    prefix = SharedPrefix(1088, torch.zeros(17, dtype=torch.int32))
    chunks = [(3, 8, 5, 1), (8, 20, 1100, 2), (20, 30, 10, 3), (30, 40, 700, 4), (40, 41, 1089, 5)]
    work, rest = b._prompt_work(chunks, prefix)
    assert rest == [chunks[3]]
    assert [(w.rows, w.plan.entries, w.prefix is prefix) for w in work] == [
        ((3, 30), ((0, 5), (17, 27)), False), ((8, 41), ((0, 12), (32, 33)), True)]
    work, rest = b._prompt_work(chunks, None)
    assert len(work) == 1 and rest == [chunks[1], chunks[3], chunks[4]]
