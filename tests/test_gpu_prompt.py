"""GPU: causal attention of packed prompts (kernels.prompt) against float64, at the sizes, types,
strides and values where it can go wrong."""

import pytest
import torch

from attend64 import Rows, check, unit
from echokv_amd.kernels.prompt import build_prompt_plan, prompt_attention

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def make(device, lens, h, gqa, d, dtype, seed=0, gap=0):
    """Packed tensors with ``gap`` rows between the prompts, and the prompts' row ranges."""
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    t = sum(lens) + gap * len(lens)
    q = torch.randn(t, h * gqa, d, device=device, generator=g).to(dtype)
    k, v = (torch.randn(t, h, d, device=device, generator=g).to(dtype) for _ in range(2))
    entries, o = [], 0
    for n in lens:
        entries.append((o, o + n))
        o += n + gap
    return q, k, v, entries


def weight_unit(dtype):
    """Rounding of the softmax weights: the matrix kernels take them in the input's type."""
    return unit(dtype)


def check_all(q, k, v, entries, out, lse, scale, untouched=None):
    for a, b in entries:
        if a == b:
            continue
        r = Rows(q[a:b], k[a:b], v[a:b], range(1, b - a + 1), scale)
        check(out[a:b].view(b - a, *q.shape[1:]), r, weight=weight_unit(q.dtype))
        if lse is not None:
            assert float((lse[a:b].double() - r.lse).abs().max()) <= r.lse_bound()


LENS = [[1], [1, 2, 3], [37, 64, 65], [130, 1, 257], [700]]


@pytest.mark.parametrize("lens", LENS, ids=str)
@pytest.mark.parametrize("h,gqa,d", [(2, 4, 128), (1, 1, 128), (3, 7, 128), (2, 8, 64), (1, 20, 64), (2, 4, 256),
                                     (2, 4, 96), (1, 3, 20), (2, 2, 80), (1, 300, 64)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
def test_matches_float64(device, lens, h, gqa, d, dtype):
    print(f"[prompt] {lens} H{h} GQA{gqa} D{d} {dtype}", flush=True)
    q, k, v, entries = make(device, lens, h, gqa, d, dtype, seed=len(lens) + d, gap=3)
    out = torch.full_like(q, 7.0)
    lse = torch.full(q.shape[:2], 7.0, device=device)
    prompt_attention(q, k, v, out, entries, d ** -0.5, lse=lse)
    torch.cuda.synchronize()
    check_all(q, k, v, entries, out, lse, d ** -0.5)
    for (_, b) in entries:  # the rows between the prompts
        assert (out[b : b + 3] == 7.0).all() and (lse[b : b + 3] == 7.0).all()


@pytest.mark.parametrize("h,gqa,d,lens", [(8, 4, 96, [1500, 3, 70]), (8, 5, 20, [40] * 50), (2, 4, 256, [2100]),
                                          (1, 160, 64, [300])])
def test_many_workgroups_in_32_bits(device, h, gqa, d, lens):
    """More than three workgroups of 64 rows a CU: each keeps all of its keys' steps."""
    print(f"[prompt] many workgroups D{d}", flush=True)
    q, k, v, entries = make(device, lens, h, gqa, d, F32, seed=71)
    out, lse = torch.empty_like(q), torch.empty(q.shape[:2], device=device)
    prompt_attention(q, k, v, out, entries, d ** -0.5, lse=lse)
    torch.cuda.synchronize()
    check_all(q, k, v, entries, out, lse, d ** -0.5)


@pytest.mark.parametrize("n", [255, 256, 1023, 1500, 4099])
def test_long_prompts(device, n):
    print(f"[prompt] one of {n}", flush=True)
    q, k, v, entries = make(device, [n], 2, 4, 128, BF16, seed=n)
    out = torch.empty_like(q)
    prompt_attention(q, k, v, out, entries, 128 ** -0.5)
    torch.cuda.synchronize()
    check_all(q, k, v, entries, out, None, 128 ** -0.5)


@pytest.mark.parametrize("scale", [-0.088, 0.0, 0.9])
@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
def test_softmax_scales(device, scale, dtype):
    print(f"[prompt] scale {scale} {dtype}", flush=True)
    q, k, v, entries = make(device, [90, 200], 2, 4, 128, dtype, seed=5)
    out, lse = torch.empty_like(q), torch.empty(q.shape[:2], device=device)
    prompt_attention(q, k, v, out, entries, scale, lse=lse)
    torch.cuda.synchronize()
    check_all(q, k, v, entries, out, lse, scale)


@pytest.mark.parametrize("out_dtype", [F32, F16, BF16], ids=str)
def test_output_types_and_flat_rows(device, out_dtype):
    print(f"[prompt] out {out_dtype}", flush=True)
    q, k, v, entries = make(device, [50, 130], 2, 4, 128, BF16, seed=9)
    out = torch.empty(q.shape[0], q.shape[1] * q.shape[2], dtype=out_dtype, device=device)
    prompt_attention(q, k, v, out, entries, 128 ** -0.5)
    torch.cuda.synchronize()
    check_all(q, k, v, entries, out, None, 128 ** -0.5)


@pytest.mark.parametrize("case", ["fused", "odd", "head_major", "channels"])
@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
def test_strides_and_alignment(device, case, dtype):
    print(f"[prompt] strides {case} {dtype}", flush=True)
    h, gqa, d, lens = 2, 4, 128, [70, 201]
    q, k, v, entries = make(device, lens, h, gqa, d, dtype, seed=11)
    t = q.shape[0]
    if case == "fused":  # slices of one projection's rows
        qkv = torch.cat([x.reshape(t, -1) for x in (q, k, v)], 1)
        q2, k2, v2 = (x.view(t, -1, d) for x in qkv.split([h * gqa * d, h * d, h * d], 1))
    elif case == "odd":  # rows that no 16-byte load is aligned for
        def shift(x):
            buf = torch.empty(x.numel() + 1 + t, dtype=dtype, device=device)
            y = buf.as_strided(x.shape, (x.shape[1] * d + 1, d, 1), 1)
            y.copy_(x)
            return y
        q2, k2, v2 = shift(q), shift(k), shift(v)
    elif case == "head_major":
        q2, k2, v2 = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v))
    else:  # channels apart: copied by the call
        q2, k2, v2 = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v))
    out = torch.empty_like(q)
    prompt_attention(q2, k2, v2, out, entries, d ** -0.5)
    torch.cuda.synchronize()
    check_all(q, k, v, entries, out, None, d ** -0.5)


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 64), (F32, 96), (BF16, 256)], ids=str)
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")], ids=str)
def test_later_tokens_never_reach_earlier_rows(device, dtype, d, bad):
    """Infinities and NaN in keys and values of tokens that a row does not see."""
    print(f"[prompt] {bad} behind, {dtype} D{d}", flush=True)
    q, k, v, entries = make(device, [150, 40], 2, 4, d, dtype, seed=13)
    clean = torch.empty_like(q)
    prompt_attention(q, k, v, clean, entries, d ** -0.5)
    k2, v2 = k.clone(), v.clone()
    for row in (0, 37, 149, 150, 189):
        for which, x in (("k", k2), ("v", v2)):
            kx, vx = (x, v) if which == "k" else (k, x)
            keep = x[row].clone()
            x[row, :, ::3] = bad
            out = torch.empty_like(q)
            prompt_attention(q, kx, vx, out, entries, d ** -0.5)
            torch.cuda.synchronize()
            lo = 0 if row < 150 else 150
            assert torch.equal(out[lo:row], clean[lo:row]), f"{which} row {row} reached rows before it"
            other = slice(150, 190) if row < 150 else slice(0, 150)
            assert torch.equal(out[other], clean[other])
            if which == "v":  # the channels of the value itself, from its row on
                hi = 150 if row < 150 else 190
                assert not torch.isfinite(out[row:hi, :, ::3]).any()
                assert torch.isfinite(out[row:hi, :, 1::3]).all()
            x[row] = keep


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 64), (F32, 96)], ids=str)
def test_joins_a_prefix(device, dtype, d):
    print(f"[prompt] prefix {dtype} D{d}", flush=True)
    h, gqa, lens, pre = 2, 4, [90, 1, 130], 77
    q, k, v, entries = make(device, lens, h, gqa, d, dtype, seed=17)
    _, kp, vp, _ = make(device, [pre], h, 1, d, dtype, seed=18)
    t = q.shape[0]
    r = Rows(q, kp, vp, [pre] * t, d ** -0.5)
    part, plse = r.out.float(), r.lse.float()
    none = torch.zeros(t, dtype=torch.bool, device=device)
    none[::5] = True  # rows with nothing before their prompt, whatever their part holds
    part[none], plse[none] = float("nan"), float("-inf")
    out, lse = torch.empty_like(q), torch.empty(t, h * gqa, device=device)
    prompt_attention(q, k, v, out, entries, d ** -0.5, lse=lse, prefix=(part.contiguous(), plse.contiguous()))
    torch.cuda.synchronize()
    for a, b in entries:
        for keys in (0, pre):
            sel = (none[a:b] if keys == 0 else ~none[a:b]).nonzero()[:, 0]
            if not sel.numel():
                continue
            kk, vv = (torch.cat([x[:keys], y[a:b]]) for x, y in ((kp, k), (vp, v)))
            ref = Rows(q[a:b][sel], kk, vv, (sel + keys + 1).tolist(), d ** -0.5)
            check(out[a:b][sel], ref, weight=weight_unit(dtype))
            assert float((lse[a:b][sel].double() - ref.lse).abs().max()) <= 2 * ref.lse_bound()


@pytest.mark.parametrize("t,step", [(40, 1 << 26), (300, 1 << 23)])  # a step of 64 rows past 2^31 bytes, and not
def test_offsets_past_32_bits(device, t, step):
    """Rows so far apart that the last ones lie past 2^31 elements."""
    print("[prompt] far rows", flush=True)
    d = 128
    q, k, v, entries = make(device, [t], 1, 2, d, BF16, seed=21)
    far = []
    buf = torch.empty(step * (t - 1) + 4 * d, dtype=BF16, device=device)
    for i, x in enumerate((k, v)):
        y = buf.as_strided((t, 1, d), (step, d, 1), i * d)
        y.copy_(x)
        far.append(y)
    qf = buf.as_strided((t, 2, d), (step, d, 1), 2 * d)
    qf.copy_(q)
    out = torch.empty_like(q)
    prompt_attention(qf, far[0], far[1], out, entries, d ** -0.5)
    torch.cuda.synchronize()
    check_all(q, k, v, entries, out, None, d ** -0.5)


def test_empty_steps_and_prompts(device):
    q, k, v, _ = make(device, [12], 2, 4, 128, BF16)
    out = torch.full_like(q, 3.0)
    prompt_attention(q, k, v, out, [], 0.1)
    prompt_attention(q, k, v, out, [(4, 4)], 0.1)
    plan = build_prompt_plan([], 4, 128, device)
    prompt_attention(q, k, v, out, [], 0.1, plan=plan)
    torch.cuda.synchronize()
    assert (out == 3.0).all()


def test_graph_replays_equal_eager_calls(device):
    print("[prompt] graph", flush=True)
    lens = [200, 3, 90]
    q, k, v, entries = make(device, lens, 2, 4, 128, BF16, seed=31)
    plan = build_prompt_plan(entries, 4, 128, device)
    out, eager = torch.empty_like(q), torch.empty_like(q)
    prompt_attention(q, k, v, out, entries, 0.088, plan=plan)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        prompt_attention(q, k, v, out, entries, 0.088, plan=plan)
    for seed in range(4):
        q2, k2, v2, _ = make(device, lens, 2, 4, 128, BF16, seed=40 + seed)
        for dst, src in ((q, q2), (k, k2), (v, v2)):
            dst.copy_(src)
        out.zero_()
        g.replay()
        prompt_attention(q, k, v, eager, entries, 0.088, plan=plan)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


def test_side_stream(device):
    q, k, v, entries = make(device, [300], 2, 4, 128, BF16, seed=51)
    out, ref = torch.empty_like(q), torch.empty_like(q)
    prompt_attention(q, k, v, ref, entries, 0.088)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        prompt_attention(q, k, v, out, entries, 0.088)
    s.synchronize()
    assert torch.equal(out, ref)


def test_same_bits_alone_and_in_a_batch(device):
    """A prompt's rows depend on nothing but the prompt."""
    q, k, v, entries = make(device, [90, 333, 10], 2, 4, 128, BF16, seed=61)
    out = torch.empty_like(q)
    prompt_attention(q, k, v, out, entries, 0.088)
    for a, b in entries:
        alone = torch.empty_like(q[a:b])
        prompt_attention(q[a:b], k[a:b], v[a:b], alone, [(0, b - a)], 0.088)
        torch.cuda.synchronize()
        assert torch.equal(alone, out[a:b])
