"""CPU: how much workspace calls behind a shared prefix ask for."""

from types import SimpleNamespace

import pytest

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
