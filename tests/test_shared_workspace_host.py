"""CPU: how much workspace calls behind a shared prefix ask for, and which rows take part."""

from types import SimpleNamespace

import pytest
import torch

from echokv_amd import _lib
from echokv_amd.kernels import shared as sh
from echokv_amd.tiered_cache import TieredLayout

MIB = 1 << 20


@pytest.fixture(scope="module", autouse=True)
def lib():
    if not _lib.LIB_PATH.exists():
        pytest.fail(f"{_lib.LIB_PATH} is not built")


def store(h=8, d=128, bs=16, kg=16, vg=32):
    lay = TieredLayout(h, d, bs, 8, kg, vg)
    return SimpleNamespace(layout=lay, abi=lay.abi(1000, lay.page_bytes))


@pytest.mark.parametrize("h,d,gqa", [(8, 128, 4), (2, 128, 8), (1, 64, 1), (32, 128, 1), (4, 64, 8)])
@pytest.mark.parametrize("rows", [64, 129, 256, 1000, 8000])
def test_workspace_does_not_grow_with_the_prefix(h, d, gqa, rows):
    """The dequantized prefix is held in slabs of at most 128 MiB; the rest goes by the rows: at most
    64 partial rows of an entry and head, and no more than one for each of the 256 CUs' 256 rows."""
    s, hq = store(h, d), h * gqa
    partial = max(rows * hq, 256 * 256 + 64 * rows) * (d + 2) * 4
    for tokens in (1 << 13, 1 << 15, 1 << 17, 1 << 20, 1 << 24, 1 << 30):
        assert sh.prefix_workspace_bytes(s, hq, rows, tokens) <= 128 * MIB + partial, tokens
        splits = 4
        suffix = splits * rows * hq * (d + 2) * 4 + 8 * rows + 64
        assert sh.shared_workspace_bytes(s, hq, rows, tokens, splits) <= 128 * MIB + partial + suffix, tokens


def test_one_more_sequence_costs_about_one_more():
    """128 to 129 sequences behind 131072 tokens: from where the prefix is dequantized first."""
    s = store()
    a, b = (sh.shared_workspace_bytes(s, 32, n, 1 << 17, 4) for n in (128, 129))
    assert b - a <= 128 * MIB


@pytest.mark.parametrize("h,gqa,seqs,tokens,ranges", [(1, 7, 1, 640, 5), (1, 1, 1, 128, 1), (2, 4, 3, 640, 5)])
def test_suffix_rows_are_aligned(h, gqa, seqs, tokens, ranges):
    """The suffixes' rows, read by 16-byte loads, lie behind the prefix's (max, sum) pairs: an odd number
    of those (5 ranges of 7 heads) is followed by 8 bytes of nothing."""
    s, rows, splits, d = store(h, 256), seqs * h * gqa, 4, 256
    size = sh.shared_workspace_bytes(s, h * gqa, seqs, tokens, splits)
    lengths, pairs = -(-seqs * 8 // 16) * 16, -(-ranges * rows * 8 // 16) * 16
    assert size == lengths + ranges * rows * d * 4 + pairs + splits * rows * d * 4 + splits * rows * 8


def test_prompt_refuses_half_a_prefix():
    from echokv_amd.kernels.prompt import build_prompt_plan, prompt_attention

    q, k = torch.zeros(4, 8, 128), torch.zeros(4, 2, 128)
    plan = build_prompt_plan([(0, 4)], 4, 128, torch.device("cpu"))
    for prefix in ((torch.zeros(4, 8, 128), None), (None, torch.zeros(4, 8))):
        with pytest.raises(ValueError, match="prefix"):
            prompt_attention(q, k, k, q, (), 0.1, plan=plan, prefix=prefix)


# ---- the backend's steps --------------------------------------------------------------------

def _builder(monkeypatch):
    from test_prompt_shared_host import _builder

    return _builder(monkeypatch, ECHOKV_SHARED_PREFIX="1", ECHOKV_PROMPT_EXACT="1")


def test_rows_of_other_requests_do_not_attend_to_the_prefix(monkeypatch):
    """A chunk of a longer context between two prompts behind the prefix: only the prompts' rows."""
    from echokv_amd.backend import SharedPrefix

    b = _builder(monkeypatch)
    prefix = SharedPrefix(1088, torch.zeros(17, dtype=torch.int32))
    chunks = [(3, 8, 1093, 1), (8, 20, 9000, 2), (20, 23, 1091, 3)]
    work, rest = b._prompt_work(chunks, prefix)
    assert rest == [chunks[1]] and work[0].rows == (3, 23)
    assert work[0].own.tolist() == [0, 1, 2, 3, 4, 17, 18, 19]
    work, rest = b._prompt_work([(3, 8, 1093, 1), (8, 20, 1100, 2)], prefix)  # nothing between them
    assert not rest and work[0].own is None


def test_prefix_refuses_row_indices():
    from echokv_amd.kernels.shared import prefix_attention

    s = store(2)
    s.pages, s.res_k = torch.zeros(1), None
    blocks = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="row index"):
        prefix_attention(s, torch.zeros(3, 8, 128), blocks, 64, 0.1, q_rows=torch.zeros(1, 3, dtype=torch.int64))
    with pytest.raises(ValueError, match="no query rows"):
        prefix_attention(s, torch.zeros(0, 8, 128), blocks, 64, 0.1, q_rows=torch.zeros(3, dtype=torch.int64))


def test_decode_takes_the_reserved_workspace_and_its_own_lengths(monkeypatch):
    """The plain decode's workspace where it is large enough, else memory of the step's own; the
    splits by the sequences that decode."""
    b = _builder(monkeypatch)
    s = store(2, bs=64, kg=32)
    group = SimpleNamespace(impls=[SimpleNamespace(store=s, num_heads=8)])
    from echokv_amd.backend import SharedPrefix

    prefix = SharedPrefix(1088, torch.zeros(17, dtype=torch.int32))
    need = sh.shared_workspace_bytes(s, 8, 3, 1088, 4)
    acc = torch.zeros(-(-need // (8 * 128 * 4)), 8, 128)
    got = b._decode_prefix(group, prefix, 3, 1300, (acc, None))
    assert got.num_splits == 4 and got.workspace.data_ptr() == acc.data_ptr() and got.workspace.numel() >= need
    for reserved in (None, (acc[:1], None)):
        got = b._decode_prefix(group, prefix, 3, 1300, reserved)
        assert got.workspace.data_ptr() != acc.data_ptr() and got.workspace.numel() == need


@pytest.mark.parametrize("chunk", [0, 3000])
def test_a_chunk_does_not_cut_the_decode(monkeypatch, chunk):
    """Two decodes of 1300 tokens, and a step that also prefills a request of 3000."""
    import numpy as np

    from echokv_amd import backend

    b = _builder(monkeypatch)
    n = 3 if chunk else 2
    starts = np.array([0, 1, 2, 202][: n + 1], np.int32)
    lens = torch.tensor([1300, 1290, chunk][:n])
    asked = []
    up = SimpleNamespace(decode=(torch.zeros(2),) * 3, prefill=[], tok=None, fin=None, fin_count=None, n_tokens=0, n_fin=0,
                         canary_rows=None, n_canary=0, canary_ctx=None, tier_masks=None, host_tier_masks=None)
    impl = SimpleNamespace(decode_workspace=lambda *a: None)
    group = SimpleNamespace(impls=[impl], driver=SimpleNamespace(run=lambda *a: up, apply=lambda *a: None), tiers=lambda: [4],
                            headers=None)
    monkeypatch.setattr(b, "_bound", lambda: group)
    monkeypatch.setattr(b, "_mapping", lambda cm, dummy: (lens, torch.zeros(int(starts[-1]), dtype=torch.int64)))
    monkeypatch.setattr(b, "_decode_prefix", lambda g, p, n_dec, longest, ws: asked.append((n_dec, longest)))
    monkeypatch.setattr(backend, "is_dummy_step", lambda cm: False)
    cm = SimpleNamespace(num_reqs=n, num_actual_tokens=int(starts[-1]), causal=True, slot_mapping=None,
                         query_start_loc_cpu=torch.from_numpy(starts),
                         block_table_tensor=torch.zeros(n, 60, dtype=torch.int32))
    b.build(1088, cm)
    assert asked == [(2, 1300)]
