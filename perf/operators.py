"""Attention over whole prompts and over a prefix that a batch shares, as measured cases.

A case is a dict of plain values. ``prepare`` makes what a serving program holds before
the call (queries, keys, values, a filled cache, the step's plan), ``run`` makes one call,
and ``exact`` restates its result in float64.

Kinds:

* ``prompt``: causal attention of packed prompts over their own keys and values, grouped
  heads (``kernels.prompt.prompt_attention``);
* ``decode``: one new token for each sequence of a batch whose contexts begin with the same
  cached blocks (``kernels.shared.shared_prefix_decode``);
* ``joined``: new prompts behind a cached prefix that they share: the prefix from the cache
  for every query at once (``kernels.shared.prefix_attention``), the prompts' own tokens as in
  ``prompt``, both joined.

With ``own`` false ``run`` is plain torch in 32 bits over the same inputs (the cache as codes
and statistics in blocks); with ``own`` true it calls the package.

Queries, keys and values are N(0, 1); in the cached kinds 1% of the key and of the value
channels are ten times larger, as the repository's benchmark makes them.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
GOLDEN = 0.6180339887498949
SCORES = 1 << 28  # scores that the plain form holds at a time


# ---- the cases ---------------------------------------------------------------

def _prompt(name, seqs, lo, hi, **kw):
    return {**dict(kind="prompt", name=name, seqs=seqs, lo=lo, hi=hi, heads=8, gqa=4, dim=128, dtype="bf16"), **kw}


def _cached(kind, name, seqs, prefix, lo, hi, **kw):
    base = dict(kind=kind, name=name, seqs=seqs, prefix=prefix, lo=lo, hi=hi, heads=8, gqa=4, dim=128, block=64,
                k_group=32, v_group=32, mem_bits=4, tier=4, dtype="bf16")
    return {**base, **kw}


def listed() -> list:
    return [
        # A chat turn of a few words: one launch, latency counts.
        _prompt("prompt_tiny", 1, 37, 37),
        # One new prompt of ordinary length.
        _prompt("prompt_one", 1, 1500, 1500),
        # A full step of prompts of different lengths.
        _prompt("prompt_packed", 6, 100, 2600),
        # One long document.
        _prompt("prompt_long", 1, 16384, 16384),
        # Many short prompts at head size 64 and 8 query heads per KV head.
        _prompt("prompt_short64", 40, 16, 400, dim=64, gqa=8, heads=4, dtype="f16"),
        # 32-bit activations at a head size outside the matrix kernels' ones.
        _prompt("prompt_f32_96", 3, 100, 700, dim=96, dtype="f32"),
        # Four samples of one request: its prompt is the prefix. Latency counts.
        _cached("decode", "decode_samples", 4, 512, 1, 90),
        # A batch of chats behind one system prompt, the benchmark's page shape.
        _cached("decode", "decode_batch", 64, 4096, 64, 1024, block=16, k_group=16, mem_bits=8, dtype="f16"),
        # A large batch of questions about one long document, INT8.
        _cached("decode", "decode_large", 256, 16384, 16, 400, mem_bits=8, tier=8),
        # INT2, 8 query heads per KV head.
        _cached("decode", "decode_int2", 24, 8192, 100, 1500, tier=2, gqa=8),
        # Short questions behind a cached prompt.
        _cached("joined", "joined_short", 8, 2048, 9, 130),
        # A full step of prompts behind a long cached one.
        _cached("joined", "joined_large", 16, 8192, 300, 700),
    ]


def _log(rng, lo, hi) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choice(["prompt", "prompt", "decode", "decode", "joined"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    heads = rng.choice([2, 4, 8])
    if kind == "prompt":
        if rng.random() < 0.2:  # 32 bits, or a head size of no matrix kernel
            dim = rng.choice([64, 80, 96, 128])
            seqs = rng.randint(1, 8)
            hi = _log(rng, 20, 2000 // seqs + 20)
            return _prompt("", seqs, max(1, hi // 4), hi, heads=heads, gqa=rng.choice([1, 4, 7]), dim=dim, dtype="f32")
        dim, gqa = rng.choice([(64, 4), (64, 8), (128, 1), (128, 4), (128, 7), (128, 8), (256, 4)])
        seqs = _log(rng, 1, 32)
        hi = _log(rng, 1, 12000 // seqs)
        return _prompt("", seqs, max(1, hi // rng.choice([1, 3, 10])), hi, heads=heads, gqa=gqa, dim=dim, dtype=dtype)
    block, kg = rng.choice([(16, 16), (32, 32), (64, 32), (128, 64)])
    dim, vg, gqa = rng.choice([(64, 32, 4), (128, 32, 4), (128, 32, 4), (128, 32, 8), (128, 64, 7), (128, 32, 1)])
    tier = rng.choice([2, 4, 4, 8])
    prefix = _log(rng, 2, 16384 // block) * block
    kw = dict(heads=heads, gqa=gqa, dim=dim, v_group=vg, tier=tier, mem_bits=max(4, tier), dtype=dtype, block=block,
              k_group=kg)
    if kind == "decode":
        seqs = _log(rng, 2, 256)
        hi = _log(rng, 1, min(2000, 100000 // seqs))
        return _cached(kind, "", seqs, prefix, max(1, hi // rng.choice([1, 4, 16])), hi, **kw)
    seqs = rng.randint(1, 16)
    hi = _log(rng, 1, 8000 // seqs)
    return _cached(kind, "", seqs, prefix, max(1, hi // rng.choice([1, 4, 16])), hi, **kw)


# ---- sizes and inputs ------------------------------------------------------------

def _lens(case) -> list:
    """Prompt lengths, or for ``decode`` the tokens behind the prefix (the new one among them)."""
    lo, hi = case["lo"], case["hi"]
    return [lo + int((hi - lo + 1) * math.fmod(0.5 + i * GOLDEN, 1.0)) for i in range(case["seqs"])]


def _dev() -> torch.device:
    return torch.device("cuda", torch.cuda.current_device())


def _gen(*seed) -> torch.Generator:
    g = torch.Generator(device=_dev())
    g.manual_seed(int(np.random.SeedSequence([int(s) for s in seed]).generate_state(1, np.uint64)[0] >> 1))
    return g


def _normal(case, g, n, heads) -> torch.Tensor:
    return torch.randn(n, heads, case["dim"], device=_dev(), generator=g)


def _queries(case, seed: int, n: int) -> torch.Tensor:
    return _normal(case, _gen(seed, 3), n, case["heads"] * case["gqa"]).to(DTYPES[case["dtype"]])


def _tokens(case, seed: int, seq: int, n: int) -> tuple:
    """Keys and values ``[n, heads, dim]`` of the tokens of sequence ``seq`` (0: the prefix)."""
    out = []
    big, g = _gen(seed, 7), _gen(seed, 100 + seq)
    for _ in range(2):
        w = torch.ones(case["heads"] * case["dim"], device=_dev())
        some = torch.randperm(w.numel(), generator=big, device=_dev())[: max(1, round(0.01 * w.numel()))]
        if case["kind"] != "prompt":
            w[some] = 10.0
        x = _normal(case, g, n, case["heads"]) * w.view(case["heads"], case["dim"])
        out.append(x.to(DTYPES[case["dtype"]]))
    return tuple(out)


def _entries(lens: list) -> list:
    """(first row, last row + 1) of each prompt."""
    ends = np.cumsum(lens).tolist()
    return [(e - n, e) for e, n in zip(ends, lens)]


def _tables(case, lens: list, seed: int) -> tuple:
    """(block table, number of blocks): the prefix's blocks first in every row, the rest of
    its own; random blocks of the pool."""
    bs = case["block"]
    shared = case["prefix"] // bs
    own_blocks = [-(-n // bs) for n in lens]
    nb = shared + sum(own_blocks) + 5
    perm = np.random.default_rng(seed).permutation(nb)
    table = np.zeros((len(lens), shared + max(own_blocks)), np.int64)
    table[:, :shared] = perm[:shared]
    o = shared
    for i, n in enumerate(own_blocks):
        table[i, shared : shared + n] = perm[o : o + n]
        o += n
    return table, nb


def _cache_tokens(case, seed: int) -> list:
    """(sequence, first position, keys, values) of everything in the cache."""
    parts = [(0, 0, *_tokens(case, seed, 0, case["prefix"]))]
    if case["kind"] == "decode":
        parts += [(1 + i, case["prefix"], *_tokens(case, seed, 1 + i, n)) for i, n in enumerate(_lens(case))]
    return parts


def _slots(case, table: np.ndarray, row: int, first: int, n: int) -> np.ndarray:
    p = np.arange(first, first + n)
    return table[row][p // case["block"]] * case["block"] + p % case["block"]


# ---- prepare ----------------------------------------------------------------------

def _store(case, seed: int, table: np.ndarray, nb: int):
    """The package's cache holding the case's tokens."""
    from echokv_amd.tiered_cache import TieredKVCache, TieredLayout

    geometry = (case["heads"], case["dim"], case["block"], case["mem_bits"], case["k_group"], case["v_group"])
    layout = TieredLayout(*geometry)
    pages = layout.alloc_pages(nb, _dev(), zero=True)
    res = torch.zeros(case["seqs"] + 17, case["k_group"], case["heads"], case["dim"], dtype=DTYPES[case["dtype"]],
                      device=_dev())
    store = TieredKVCache(layout, pages, residual=res)
    pend: list = []

    def flush():
        if pend:
            k, v, s = zip(*pend)
            store.write(torch.cat(k), torch.cat(v), torch.from_numpy(np.concatenate(s)), case["tier"])
            pend.clear()

    for seq, first, k, v in _cache_tokens(case, seed):
        s = _slots(case, table, max(seq - 1, 0), first, k.shape[0])
        for o in range(0, k.shape[0], 8192):
            pend.append((k[o : o + 8192], v[o : o + 8192], s[o : o + 8192]))
            if sum(x[2].size for x in pend) >= 8192:
                flush()
    flush()
    return store


def _codes(x: torch.Tensor, bits: int, dim: int) -> tuple:
    """Codes, scale and minimum of groups along ``dim``: statistics in float16, codes by the
    rounded statistics, halves to even."""
    low = x.amin(dim, keepdim=True).half()
    top = float((1 << bits) - 1)
    scale = ((x.amax(dim, keepdim=True) - low.float()) / top).clamp_min(2.0 ** -14).half()
    q = ((x - low.float()) / scale.float()).round().clamp(0.0, top)
    return q.to(torch.uint8), scale, low


def _plain_cache(case, seed: int, table: np.ndarray, nb: int) -> dict:
    """The same cache for the plain form: codes and statistics of each block, the keys of each
    sequence's open group as they came."""
    bs, kg, vg, h, d = case["block"], case["k_group"], case["v_group"], case["heads"], case["dim"]
    dev, dt = _dev(), DTYPES[case["dtype"]]
    c = dict(kc=torch.zeros(nb, bs, h, d, dtype=torch.uint8, device=dev),
             vc=torch.zeros(nb, bs, h, d, dtype=torch.uint8, device=dev),
             ks=torch.zeros(nb, bs // kg, h, d, dtype=torch.half, device=dev),
             km=torch.zeros(nb, bs // kg, h, d, dtype=torch.half, device=dev),
             vs=torch.zeros(nb, bs, h, d // vg, dtype=torch.half, device=dev),
             vm=torch.zeros(nb, bs, h, d // vg, dtype=torch.half, device=dev),
             open=torch.zeros(case["seqs"], kg, h, d, dtype=dt, device=dev))
    for seq, first, k, v in _cache_tokens(case, seed):
        n = k.shape[0]
        slot = torch.from_numpy(_slots(case, table, max(seq - 1, 0), first, n)).to(dev)
        q, s, m = _codes(v.float().view(n, h, d // vg, vg), case["tier"], 3)
        for name, x in (("vc", q.view(n, h, d)), ("vs", s[..., 0]), ("vm", m[..., 0])):
            c[name].view(nb * bs, h, -1)[slot] = x
        full = n // kg * kg
        if full:
            q, s, m = _codes(k[:full].float().view(-1, kg, h, d), case["tier"], 1)
            c["kc"].view(nb * bs, h, d)[slot[:full]] = q.view(full, h, d)
            group = slot[:full:kg] // kg
            c["ks"].view(-1, h, d)[group] = s[:, 0]
            c["km"].view(-1, h, d)[group] = m[:, 0]
        if n > full:
            c["open"][seq - 1, : n - full] = k[full:]
    return c


def prepare(case, seed: int) -> dict:
    lens = _lens(case)
    dev = _dev()
    st = dict(case=case, scale=case["dim"] ** -0.5, entries=_entries(lens))
    if case["kind"] != "prompt":
        table, nb = _tables(case, lens, seed)
        st["table"] = torch.from_numpy(table).to(dev, torch.int32)
        st["lens"] = torch.tensor([case["prefix"] + n for n in lens], device=dev)
        if own:
            st["store"] = _store(case, seed, table, nb)
        else:
            st["cache"] = _plain_cache(case, seed, table, nb)
    if case["kind"] == "decode":
        st["q"] = _queries(case, seed, len(lens))
        st["max_len"] = case["prefix"] + max(lens)
    else:
        st["q"] = _queries(case, seed, sum(lens))
        kv = [_tokens(case, seed, 1 + i, n) for i, n in enumerate(lens)]
        st["k"], st["v"] = (torch.cat([x[j] for x in kv]) for j in range(2))
        if own:
            from echokv_amd.kernels.prompt import build_prompt_plan

            st["plan"] = build_prompt_plan(st["entries"], case["gqa"], case["dim"], dev)
    st["out"] = torch.zeros_like(st["q"])
    return st


# ---- run, by the package ------------------------------------------------------------

def _own_run(st):
    case = st["case"]
    if case["kind"] == "decode":
        from echokv_amd.kernels.shared import shared_prefix_decode

        return shared_prefix_decode(st["store"], st["q"], st["table"], st["lens"], case["prefix"], st["scale"],
                                    out=st["out"], max_len=st["max_len"], tier=case["tier"])
    from echokv_amd.kernels.prompt import prompt_attention

    prefix = None
    if case["kind"] == "joined":
        from echokv_amd.kernels.shared import prefix_attention

        prefix = prefix_attention(st["store"], st["q"], st["table"][0], case["prefix"], st["scale"])
    prompt_attention(st["q"], st["k"], st["v"], st["out"], st["entries"], st["scale"], plan=st["plan"], prefix=prefix)
    return st["out"]


# ---- run, in plain torch --------------------------------------------------------------

def _by_head(x: torch.Tensor, heads: int) -> torch.Tensor:
    """Rows ``[n, heads * g, dim]`` as ``[heads, n * g, dim]`` in 32 bits."""
    n, hq, d = x.shape
    return x.float().view(n, heads, hq // heads, d).transpose(0, 1).reshape(heads, -1, d)


def _blocks(cache: dict, ids: torch.Tensor, v_group: int) -> tuple:
    """Keys and values ``[..., blocks * block, heads, dim]`` of the named blocks, dequantized."""
    kc, vc = cache["kc"][ids], cache["vc"][ids]
    shape = kc.shape  # [..., blocks, block, heads, dim]
    groups = cache["ks"].shape[1]
    k = kc.float().unflatten(-3, (groups, -1))
    k = k * cache["ks"][ids].float().unsqueeze(-3) + cache["km"][ids].float().unsqueeze(-3)
    v = vc.float().unflatten(-1, (-1, v_group))
    v = v * cache["vs"][ids].float().unsqueeze(-1) + cache["vm"][ids].float().unsqueeze(-1)
    lead = shape[:-4] + (-1,) + shape[-2:]
    return k.reshape(lead), v.reshape(lead)


def _plain_prompt(st, cached: tuple | None) -> torch.Tensor:
    """Causal attention of each prompt, behind the cached keys and values if there are any."""
    case, out = st["case"], st["out"]
    h, gqa, d = case["heads"], case["gqa"], case["dim"]
    for a, b in st["entries"]:
        n = b - a
        k, v = st["k"][a:b].float().transpose(0, 1), st["v"][a:b].float().transpose(0, 1)
        first = 0
        if cached is not None:
            first = cached[0].shape[1]
            k, v = torch.cat([cached[0], k], 1), torch.cat([cached[1], v], 1)
        kt, v = k.transpose(1, 2).contiguous(), v.contiguous()
        rows = max(1, SCORES // (h * gqa * (first + n)))
        for r in range(0, n, rows):
            e = min(n, r + rows)
            seen = first + e
            s = torch.matmul(_by_head(st["q"][a + r : a + e], h), kt[:, :, :seen]) * st["scale"]
            s = s.view(h, e - r, gqa, seen)
            later = torch.arange(seen, device=s.device)[None] > torch.arange(first + r, seen, device=s.device)[:, None]
            s = s.masked_fill(later[:, None], -math.inf)
            p = (s - s.amax(-1, keepdim=True)).exp()
            o = torch.matmul(p.view(h, -1, seen), v[:, :seen]).view(h, e - r, gqa, d) / p.sum(-1, keepdim=True)
            out[a + r : a + e] = o.transpose(0, 1).reshape(e - r, h * gqa, d).to(out.dtype)
    return out


def _plain_decode(st) -> torch.Tensor:
    case, c, out = st["case"], st["cache"], st["out"]
    h, gqa, d, kg = case["heads"], case["gqa"], case["dim"], case["k_group"]
    shared = case["prefix"] // case["block"]
    n = st["q"].shape[0]
    kp, vp = (x.transpose(0, 1).contiguous() for x in _blocks(c, st["table"][0, :shared].long(), case["v_group"]))
    q = _by_head(st["q"], h)
    scores = (torch.matmul(q, kp.transpose(1, 2).contiguous()) * st["scale"]).view(h, n, gqa, -1)
    ks, vs = _blocks(c, st["table"][:, shared:].long(), case["v_group"])  # [n, tokens, heads, dim]
    lens = st["lens"] - case["prefix"]
    at = torch.arange(ks.shape[1], device=q.device)[None] - (lens // kg * kg)[:, None]  # place in the open group
    exact = c["open"].float()[torch.arange(n, device=q.device)[:, None], at.clamp(0, kg - 1)]
    ks = torch.where((at >= 0)[:, :, None, None] & (at < kg)[:, :, None, None], exact, ks)
    ks, vs = (x.permute(2, 0, 1, 3).contiguous() for x in (ks, vs))  # [heads, n, tokens, dim]
    tail = torch.matmul(q.view(h, n, gqa, d), ks.transpose(2, 3).contiguous()) * st["scale"]
    past = torch.arange(ks.shape[2], device=q.device)[None] >= lens[:, None]
    tail = tail.masked_fill(past[None, :, None], -math.inf)
    top = torch.maximum(scores.amax(-1, keepdim=True), tail.amax(-1, keepdim=True))
    p, pt = (scores - top).exp(), (tail - top).exp()
    o = torch.matmul(p.view(h, n * gqa, -1), vp).view(h, n, gqa, d) + torch.matmul(pt, vs)
    o = o / (p.sum(-1, keepdim=True) + pt.sum(-1, keepdim=True))
    out.copy_(o.transpose(0, 1).reshape(n, h * gqa, d))
    return out


def run(st):
    if own:
        return _own_run(st)
    case = st["case"]
    if case["kind"] == "decode":
        return _plain_decode(st)
    cached = None
    if case["kind"] == "joined":
        ids = st["table"][0, : case["prefix"] // case["block"]].long()
        cached = tuple(x.transpose(0, 1).contiguous() for x in _blocks(st["cache"], ids, case["v_group"]))
    return _plain_prompt(st, cached)


# ---- what a pass cannot do without ---------------------------------------------------

def _cached_bytes(case, n: int) -> int:
    """Codes and statistics of ``n`` cached tokens, the open group's keys in the model dtype."""
    hd, kg = case["heads"] * case["dim"], case["k_group"]
    full = n // kg * kg
    code = hd * case["tier"] // 8
    values = n * (code + 4 * hd // case["v_group"])
    return values + full * code + n // kg * hd * 4 + (n - full) * hd * DTYPES[case["dtype"]].itemsize


def work(case) -> dict:
    lens = _lens(case)
    es, hd = DTYPES[case["dtype"]].itemsize, case["heads"] * case["dim"]
    hq = case["heads"] * case["gqa"]
    if case["kind"] == "decode":
        nbytes = _cached_bytes(case, case["prefix"]) + sum(_cached_bytes(case, n) for n in lens)
        nbytes += 2 * len(lens) * hq * case["dim"] * es
        return {"bytes": nbytes, "flops": 4 * case["dim"] * hq * sum(case["prefix"] + n for n in lens)}
    t = sum(lens)
    nbytes = 2 * t * (hq * case["dim"] + hd) * es
    pairs = sum(n * (n + 1) // 2 for n in lens)
    if case["kind"] == "joined":
        nbytes += _cached_bytes(case, case["prefix"])
        pairs += t * case["prefix"]
    return {"bytes": nbytes, "flops": 4 * case["dim"] * hq * pairs}


# ---- results in 64 bits ------------------------------------------------------------------

def _round_trip(x: torch.Tensor, bits: int) -> torch.Tensor:
    """Values of groups (last axis) as the cache holds them."""
    lo = x.min(-1, keepdim=True).values.to(torch.float16)
    levels = 2 ** bits - 1
    step = torch.clamp((x.max(-1, keepdim=True).values - lo.float()) / levels, min=2.0 ** -14).to(torch.float16)
    code = torch.clamp(torch.round((x - lo.float()) / step.float()), 0, levels)
    return code.double() * step.double() + lo.double()


def _held(case, k: torch.Tensor, v: torch.Tensor) -> tuple:
    """A sequence's keys and values as the cache holds them, ``[heads, n, dim]`` in float64."""
    n, h, d = k.shape
    full = n - n % case["k_group"]
    keys = k.double()
    if full:
        g = k[:full].float().reshape(-1, case["k_group"], h, d).movedim(1, 3)
        keys[:full] = _round_trip(g, case["tier"]).movedim(3, 1).reshape(full, h, d)
    vals = _round_trip(v.float().reshape(n, h, -1, case["v_group"]), case["tier"]).reshape(n, h, d)
    return keys.movedim(1, 0).contiguous(), vals.movedim(1, 0).contiguous()


def _attend64(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, before: int) -> torch.Tensor:
    """Softmax attention of the queries ``[n, hq, dim]`` (query i sees ``before + i + 1`` keys)
    over ``[heads, keys, dim]``, in float64, head by head and in runs of queries."""
    n, hq, d = q.shape
    gqa = hq // k.shape[0]
    out = torch.empty(n, hq, d, dtype=torch.float64, device=q.device)
    run_len = max(1, (SCORES // 2) // max(1, k.shape[1]))
    for j in range(hq):
        kt, vj = k[j // gqa].t().contiguous(), v[j // gqa]
        for a in range(0, n, run_len):
            b = min(n, a + run_len)
            keys = min(k.shape[1], before + b)
            s = q[a:b, j].double() @ kt[:, :keys] / math.sqrt(d)
            limit = torch.arange(before + a + 1, before + b + 1, device=q.device)
            s[torch.arange(keys, device=q.device)[None, :] >= limit[:, None]] = -math.inf
            out[a:b, j] = torch.softmax(s, 1) @ vj[:keys]
    return out


def exact(case, seed: int):
    lens = _lens(case)
    if case["kind"] == "prompt":
        q = _queries(case, seed, sum(lens))
        rows = []
        for i, (a, b) in enumerate(_entries(lens)):
            k, v = (x.double().movedim(1, 0).contiguous() for x in _tokens(case, seed, 1 + i, b - a))
            rows.append(_attend64(q[a:b], k, v, 0))
        return torch.cat(rows)
    kp, vp = _held(case, *_tokens(case, seed, 0, case["prefix"]))
    decode = case["kind"] == "decode"
    q = _queries(case, seed, len(lens) if decode else sum(lens))
    rows = []
    for i, (a, b) in enumerate([(i, i + 1) for i in range(len(lens))] if decode else _entries(lens)):
        k, v = _tokens(case, seed, 1 + i, lens[i])
        k, v = _held(case, k, v) if decode else (x.double().movedim(1, 0) for x in (k, v))
        before = case["prefix"] + (lens[i] - 1 if decode else 0)
        rows.append(_attend64(q[a:b], torch.cat([kp, k], 1), torch.cat([vp, v], 1), before))
    return torch.cat(rows)
