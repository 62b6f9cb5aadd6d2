"""GPU: long prompts against float64, row by row: the log-sum-exp, and queries that are the sum of two
keys, one of them at an end of a tile, step or prompt: the two share the weight, so that a key lost there
or counted twice moves the row by a large part of its value."""

import numpy as np
import pytest
import torch

from attend64 import Rows, check, unit
from test_gpu_prompt import BF16, F16, F32, make

from echokv_amd.kernels.prompt import build_prompt_plan, prompt_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,gqa,dtype", [(128, 4, BF16), (128, 4, F16), (64, 8, F16), (256, 4, BF16), (96, 4, F32),
                                         (128, 4, F32), (64, 1, BF16)], ids=str)
@pytest.mark.parametrize("lens", [[4099], [1500], [2000, 1, 321], [64] * 40], ids=str)
def test_no_key_is_lost_or_doubled(device, d, gqa, dtype, lens):
    print(f"[prompt ends] D{d} GQA{gqa} {dtype} {lens[:3]}", flush=True)
    q, k, v, entries = make(device, lens, 2, gqa, d, dtype, seed=sum(lens) + d)
    rng = np.random.default_rng(d)
    tile = build_prompt_plan(entries, gqa, d, device).tile_m
    wanted = []
    for a, b in entries[:3]:
        n = b - a
        cuts = {x for step in (32, 64, tile) for x in range(0, n, step)} | {n}
        at = sorted({p for x in cuts for p in (x - 1, x) if 0 <= p < n})
        for i in sorted({0, n - 1} | set(rng.integers(0, n, min(n, 24)).tolist()) | {p for p in at if n <= 330 or p % 5 == 0}):
            mine = [p for p in at if p <= i]
            for j in range(q.shape[1]):
                x, y = mine[(7 * i + j) % len(mine)], int(rng.integers(i + 1))
                q[a + i, j] = ((k[a + x, j // gqa].float() + k[a + y, j // gqa].float()) * (12 * d ** -0.5)).to(dtype)
            wanted.append((a, b, i))
    out, lse = torch.empty_like(q, dtype=F32), torch.empty(q.shape[:2], device=device)
    prompt_attention(q, k, v, out, entries, d ** -0.5, lse=lse)
    torch.cuda.synchronize()
    for a, b in entries[:3]:
        rows = [i for x, _, i in wanted if x == a]
        for o in range(0, len(rows), 64):
            some = rows[o : o + 64]
            at = [a + i for i in some]
            r = Rows(q[at], k[a:b], v[a:b], [i + 1 for i in some], d ** -0.5)
            check(out[at], r, weight=unit(dtype) if dtype != F32 and d in (64, 128, 256) else 0.0)
            assert float((lse[at].double() - r.lse).abs().max()) <= r.lse_bound()
