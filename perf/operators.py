"""Measured operators of the paged serving path: their plain forms, their cases and their work.

Four kinds of case, each one pass of what a serving program does:

* ``attention``: the attention of one decode step over a 4-bit paged cache (the step's plan, then one
  call a layer).
* ``write``: new tokens' keys and values rounded to 4 bits and written into the cache, and all of the
  pool's slots read back as 16-bit keys and values.
* ``rotary``: rotary positions with several axes (time, height, width) applied to queries and keys.
* ``fork`` (some branches of requests dropped, others forked over shared blocks) and ``compact`` (a
  fragmented pool's live blocks moved to its lowest ids).

A 4-bit cache is (blocks, layers, KV heads, 1152) elements of the model's 16-bit type. One such tile
holds 16 tokens of one head: 1024 bytes of key codes, 1024 bytes of value codes, then the
(scale, minimum) pairs of the keys' and of the values' two 64-dimension groups per token. An element
stands for ``code * scale + minimum``; scale is ``(max - min) / 15`` of the group, rounded once to the
type, and code is ``(x - min) / scale`` rounded to the nearest, ties to even, within 0..15. A group that
holds no finite span has NaN for both.
"""
import math

import torch

own = False

BLOCK = 16
DIM = 128
TILE = 1152  # 16-bit elements of one (block, layer, head) tile
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ---- cases ------------------------------------------------------------------------------------------


def listed():
    return [
        # one layer of a 28/4-head model serving four short requests: the smallest call, launches count
        dict(name="attention_4_short", kind="attention", dtype="fp16", batch=4, hq=28, hkv=4, layers=1, mode="uniform", lo=17, hi=300),
        # a chat batch of the same model
        dict(name="attention_64_chat", kind="attention", dtype="fp16", batch=64, hq=28, hkv=4, layers=4, mode="log", mu=5.5, lo=4, hi=4096),
        # a full batch of a 32/4-head model, lengths spread over three decades
        dict(name="attention_256_ragged", kind="attention", dtype="bf16", batch=256, hq=32, hkv=4, layers=4, mode="log", mu=6.0, lo=4, hi=4096),
        # two long documents: the split over the cache's length is all the parallelism there is
        dict(name="attention_2_long", kind="attention", dtype="bf16", batch=2, hq=32, hkv=4, layers=2, mode="uniform", lo=40001, hi=65535),
        # multi-head attention without sharing: one query head a tile
        dict(name="attention_16_mha", kind="attention", dtype="fp16", batch=16, hq=40, hkv=40, layers=2, mode="uniform", lo=2048, hi=4096),
        # a decode step's new tokens, one of each of 64 requests
        dict(name="write_64_tokens", kind="write", dtype="fp16", tokens=64, hkv=4, blocks=64, scattered=True),
        # a prompt batch
        dict(name="write_11348_prompt", kind="write", dtype="bf16", tokens=11348, hkv=4, blocks=720, scattered=False),
        # queries and keys of a decode batch over a video's context
        dict(name="rotary_256_tokens", kind="rotary", dtype="bf16", tokens=256, hq=32, hkv=4, dim=128, sections="16,24,24", deal=False, far=100000),
        # a prompt batch with images, frequencies dealt to the axes in turn
        dict(name="rotary_11348_prompt", kind="rotary", dtype="fp16", tokens=11348, hq=28, hkv=4, dim=128, sections="24,20,20", deal=True, far=20000),
        # a beam step: 24 branches dropped, 24 forked from 8 requests
        dict(name="fork_24_branches", kind="fork", dtype="fp16", blocks=700, layers=4, hkv=4, parents=8, children=24, lo=60, hi=700),
        # parallel samples of a batch of prompts, whole blocks of 28 layers
        dict(name="fork_192_samples", kind="fork", dtype="fp16", blocks=2100, layers=28, hkv=4, parents=48, children=192, lo=30, hi=600),
        # a pool half freed, before its tail is given to another model
        dict(name="compact_2048_blocks", kind="compact", dtype="bf16", blocks=2048, layers=28, hkv=4, rows=60, width=40, live=0.5),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "write", "rotary", "fork", "compact"])
    dtype = rng.choice(["fp16", "bf16"])
    if kind == "attention":
        hkv = rng.choice([1, 2, 4, 5, 8])
        group = rng.choice([1, 2, 3, 4, 6, 7, 8, 12, 16])
        hi = _log(rng, 40, 30000)
        batch = max(1, min(_log(rng, 1, 256), 400000 // hi))
        mode = rng.choice(["uniform", "log"])
        return dict(kind=kind, dtype=dtype, batch=batch, hq=hkv * group, hkv=hkv, layers=rng.choice([1, 2, 3]), mode=mode,
                    mu=round(rng.uniform(3.0, 7.0), 2), lo=rng.randint(1, 17), hi=hi)
    if kind == "write":
        tokens = _log(rng, 1, 11348)
        scattered = rng.random() < 0.5
        blocks = (tokens if scattered and tokens <= 512 else -(-tokens // BLOCK)) + rng.randint(1, 20)
        return dict(kind=kind, dtype=dtype, tokens=tokens, hkv=rng.choice([1, 2, 3, 4]), blocks=blocks, scattered=scattered and tokens <= 512)
    if kind == "rotary":
        dim = rng.choice([64, 80, 96, 128])
        half = dim // 2 if rng.random() < 0.7 else dim // 4
        a = rng.randint(1, half - 2)
        b = rng.randint(1, half - a - 1)
        hkv = rng.choice([1, 2, 4, 8])
        return dict(kind=kind, dtype=dtype, tokens=_log(rng, 1, 8000), hq=hkv * rng.choice([1, 3, 4, 7]), hkv=hkv, dim=dim,
                    sections="%d,%d,%d" % (a, b, half - a - b), deal=rng.random() < 0.5, far=_log(rng, 1000, 200000))
    layers, hkv = rng.choice([2, 5, 16, 28]), rng.choice([1, 4])
    if kind == "fork":
        parents = _log(rng, 1, 48)
        children = min(192, parents * rng.randint(1, 4) + rng.randint(0, 3))
        hi = _log(rng, 20, 600)
        return dict(kind=kind, dtype=dtype, blocks=parents * (hi // BLOCK + 2) + 2 * children + rng.randint(0, 99), layers=layers, hkv=hkv,
                    parents=parents, children=children, lo=rng.randint(1, 16), hi=hi)
    blocks = _log(rng, 64, 2048)
    rows = max(2, blocks // rng.randint(8, 40))
    return dict(kind=kind, dtype=dtype, blocks=blocks, layers=layers, hkv=hkv, rows=rows, width=rng.randint(20, 45),
                live=round(rng.uniform(0.1, 0.8), 2))


# ---- the 4-bit format -------------------------------------------------------------------------------


def _power(k):
    """2 ** k for whole k within the normal range of 64 bits, exactly."""
    return ((k.to(torch.int64) + 1023) << 52).view(torch.float64)


def _round_once(v, dtype):
    """64-bit values rounded to a 16-bit type in one step (a cast goes through 32 bits)."""
    digits, least = (11, -13) if dtype == torch.float16 else (8, -125)
    unit = _power(torch.frexp(v)[1].clamp(min=least) - digits)
    return (torch.round(v / unit) * unit).to(dtype)


def _quantise(x):
    """Codes (whole numbers 0..15, 64 bits) and (scale, minimum) pairs of vectors of 128."""
    groups = x.double().unflatten(-1, (2, 64))
    low, high = groups.amin(-1), groups.amax(-1)
    bad = ~torch.isfinite(high.float() - low.float())
    scale = _round_once(torch.where(bad, 0.0, high - low) / 15, x.dtype)
    steps = (groups - low.unsqueeze(-1)) / scale.double().unsqueeze(-1)
    flat = (bad | (scale == 0)).unsqueeze(-1)
    codes = torch.round(torch.where(flat, 0.0, steps)).clamp(0, 15).to(torch.uint8).flatten(-2)
    nan = torch.full((), math.nan, dtype=x.dtype, device=x.device)
    return codes, torch.stack([torch.where(bad, nan, scale), torch.where(bad, nan, low.to(x.dtype))], -1)


def _pack_rows(codes_k, codes_v, par_k, par_v):
    """Tiles [n, TILE] of whole blocks from codes [n, 16, 128] and pairs [n, 16, 2, 2]."""
    n = codes_k.shape[0]
    k = codes_k.view(n, 16, 4, 4, 4, 2).permute(0, 1, 3, 2, 4, 5)  # token, word, quad, byte, nibble -> token, quad, word, ...
    k = (k[..., 0] | (k[..., 1] << 4)).reshape(n, 1024)
    v = codes_v.view(n, 8, 2, 2, 8, 2, 2, 2)  # pair, parity, group, row, word, byte, nibble
    v = v.permute(0, 1, 4, 3, 5, 2, 6, 7)  # pair, row, group, word, parity, byte, nibble
    v = (v[..., 0] | (v[..., 1] << 4)).reshape(n, 1024)
    return torch.cat([k.view(par_k.dtype), v.view(par_v.dtype), par_k.reshape(n, 64), par_v.reshape(n, 64)], 1)


def _unpack_rows(tiles):
    """Keys and values [..., 16, 128] in 32 bits that tiles [..., TILE] stand for."""
    lead = tiles.shape[:-1]
    codes = tiles[..., :1024].contiguous().view(torch.uint8)
    codes = torch.stack([codes & 15, codes >> 4], -1)
    k = codes[..., :1024, :].reshape(*lead, 16, 4, 4, 4, 2).transpose(-4, -3).reshape(*lead, 16, 2, 64)
    v = codes[..., 1024:, :].reshape(*lead, 8, 8, 2, 2, 2, 2, 2)  # pair, row, group, word, parity, byte, nibble
    m = len(lead)
    v = v.permute(*range(m), m, m + 4, m + 2, m + 1, m + 3, m + 5, m + 6).reshape(*lead, 16, 2, 64)
    pairs = tiles[..., 1024:].float().reshape(*lead, 2, 16, 2, 2, 1)
    k = k.float() * pairs[..., 0, :, :, 0, :] + pairs[..., 0, :, :, 1, :]
    v = v.float() * pairs[..., 1, :, :, 0, :] + pairs[..., 1, :, :, 1, :]
    return k.flatten(-2), v.flatten(-2)


def _exact_tiles(tiles):
    """Keys and values [n, 16, 128] in 64 bits of tiles [n, TILE], element by element from the byte and the bit that hold it."""
    raw = tiles.contiguous().view(torch.uint8).long()
    t = torch.arange(16, device=tiles.device).view(16, 1)
    d = torch.arange(128, device=tiles.device).view(1, 128)
    k_at = t * 64 + (d % 32) // 8 * 16 + d // 32 * 4 + d % 8 // 2
    v_at = 1024 + t // 2 * 128 + d % 64 // 8 * 16 + (2 * (d // 64) + d % 8 // 4) * 4 + t % 2 * 2 + d % 4 // 2
    wide = tiles.double()
    got = []
    for at, pairs in ((k_at, 1024), (v_at, 1088)):
        code = torch.bitwise_right_shift(raw[:, at.flatten()].view(-1, 16, 128), 4 * (d % 2)) & 15
        p = (pairs + t * 4 + d // 64 * 2).flatten()
        got.append(code.double() * wide[:, p].view(-1, 16, 128) + wide[:, p + 1].view(-1, 16, 128))
    return got


# ---- inputs -----------------------------------------------------------------------------------------


def _generators(seed):
    return torch.Generator().manual_seed(seed), torch.Generator("cuda").manual_seed(seed)


def _normal(shape, dtype, g, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * std).to(dtype)


def _lengths(case, n, g):
    if case.get("mode") == "log":
        x = torch.empty(n, dtype=torch.float64).log_normal_(case["mu"], 1.0, generator=g).round()
        return x.clamp(case["lo"], case["hi"]).to(torch.int32)
    return torch.randint(case["lo"], case["hi"] + 1, (n,), generator=g).to(torch.int32)


def _scattered_tables(lens, n_blocks, width, g):
    """Block tables of rows that share nothing, their blocks spread over the pool."""
    used = (lens.long() + BLOCK - 1) // BLOCK
    mask = torch.arange(width).view(1, -1) < used.view(-1, 1)
    tables = torch.zeros(len(lens), width, dtype=torch.int32)
    tables[mask] = torch.randperm(n_blocks, generator=g)[: int(used.sum())].to(torch.int32)
    return tables


def _prepare_attention(case, g, gd):
    dtype = TYPES[case["dtype"]]
    lens = _lengths(case, case["batch"], g)
    used = int(((lens.long() + BLOCK - 1) // BLOCK).sum())
    n_blocks = used + 7
    tables = _scattered_tables(lens, n_blocks, int((lens.max() + BLOCK - 1) // BLOCK), g)
    cache = torch.empty(n_blocks, case["layers"], case["hkv"], TILE, dtype=dtype, device="cuda")
    rows, step = cache.view(-1, TILE), 1 << 15
    shift = _normal((2, 1, 1, DIM), torch.float32, gd)  # channels that keep an offset over all tokens, as keys do
    for i in range(0, rows.shape[0], step):
        n = min(step, rows.shape[0] - i)
        x = (torch.randn((2, n, 16, DIM), generator=gd, device="cuda") + shift).to(dtype)
        codes, pairs = _quantise(x)
        rows[i:i + n] = _pack_rows(codes[0], codes[1], pairs[0], pairs[1])
    return dict(kind="attention", cache=cache, tables=tables.cuda(), lens=lens.cuda(), scale=1.0 / math.sqrt(DIM),
                query=_normal((case["layers"], case["batch"], case["hq"], DIM), dtype, gd), hkv=case["hkv"])


def _prepare_write(case, g, gd):
    dtype, n = TYPES[case["dtype"]], case["tokens"]
    if case["scattered"]:  # one token in a block of its own, at any place of it
        slots = torch.randperm(case["blocks"], generator=g)[:n] * BLOCK + torch.randint(0, BLOCK, (n,), generator=g)
    else:  # prompts over scattered blocks
        at = torch.arange(n)
        slots = torch.randperm(case["blocks"], generator=g)[at // BLOCK] * BLOCK + at % BLOCK
    shift = _normal((1, case["hkv"], DIM), torch.float32, gd)
    key = (_normal((n, case["hkv"], DIM), torch.float32, gd) + shift).to(dtype)
    value = _normal((n, case["hkv"], DIM), dtype, gd)
    return dict(kind="write", key=key, value=value, slots=slots.cuda(), all=torch.arange(case["blocks"] * BLOCK, device="cuda"),
                cache=torch.zeros(case["blocks"], 1, case["hkv"], TILE, dtype=dtype, device="cuda"))


def _axis_of(sections, deal):
    """The axis of each frequency: sections one after another, or dealt in turn until an axis has its number."""
    if not deal:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    left, order = list(sections), []
    while any(left):
        for a in range(len(left)):
            if left[a]:
                left[a] -= 1
                order.append(a)
    return order


def _prepare_rotary(case, g, gd):
    dtype, n = TYPES[case["dtype"]], case["tokens"]
    sections = [int(s) for s in case["sections"].split(",")]
    # runs of text, where all axes agree, and pictures 16 wide, where time stands still
    start = int(torch.randint(0, case["far"], (1,), generator=g))
    at = torch.arange(n)
    picture = (at // 256) % 2 == 1
    text = start + at
    pos = torch.stack([torch.where(picture, start + at // 256 * 256, text), torch.where(picture, start + at // 256 * 256 + at % 256 // 16, text),
                       torch.where(picture, start + at // 256 * 256 + at % 16, text)])
    half = sum(sections)
    inv = (1.0 / (1000000.0 ** (torch.arange(half, dtype=torch.float64) / half))).float()
    return dict(kind="rotary", query=_normal((n, case["hq"], case["dim"]), dtype, gd), key=_normal((n, case["hkv"], case["dim"]), dtype, gd),
                positions=pos.cuda(), inv_freq=inv.cuda(), sections=sections, deal=case["deal"],
                axis=torch.tensor(_axis_of(sections, case["deal"]), device="cuda"))


def _prepare_fork(case, g, gd):
    dtype, parents, children = TYPES[case["dtype"]], case["parents"], case["children"]
    lens = _lengths(case, parents, g)
    width = (case["hi"] + BLOCK - 1) // BLOCK
    used = (lens.long() + BLOCK - 1) // BLOCK
    perm = torch.randperm(case["blocks"], generator=g).to(torch.int32)
    own_blocks = int(used.sum())
    tables = torch.zeros(parents + children, width, dtype=torch.int32)
    mask = torch.arange(width).view(1, -1) < used.view(-1, 1)
    tables[:parents][mask] = perm[:own_blocks]
    # the children of the step before, which this one drops: forks of any of the parents
    old = torch.randint(0, parents, (children,), generator=g)
    tables[parents:] = tables[old]
    at = own_blocks
    all_lens = torch.cat([lens, lens[old]])
    for i in range(children):
        if int(lens[old[i]]) % BLOCK:
            tables[parents + i, int(used[old[i]]) - 1] = perm[at]
            at += 1
    used = (all_lens.long() + BLOCK - 1) // BLOCK
    held = tables[torch.arange(width).view(1, -1) < used.view(-1, 1)].long()
    kv = _normal((case["blocks"], case["layers"], 2, BLOCK, case["hkv"], DIM), dtype, gd)
    return dict(kind="fork", kv=kv, counts=torch.bincount(held, minlength=case["blocks"]).to(torch.int32).cuda(), tables=tables.cuda(),
                lens=all_lens.cuda(), src=torch.randint(0, parents, (children,), generator=g).cuda(),
                dst=(parents + torch.arange(children)).cuda())


def _prepare_compact(case, g, gd):
    n, rows, width = case["blocks"], case["rows"], case["width"]
    want = max(1, int(n * case["live"]))
    lens = torch.randint(1, width * BLOCK + 1, (rows,), generator=g).to(torch.int32)
    used = (lens.long() + BLOCK - 1) // BLOCK
    mask = torch.arange(width).view(1, -1) < used.view(-1, 1)
    tables = torch.zeros(rows, width, dtype=torch.int32)
    # rows share some of their blocks: entries drawn from the live ones
    live = torch.randperm(n, generator=g)[:want].to(torch.int32)
    tables[mask] = live[torch.randint(0, want, (int(used.sum()),), generator=g)]
    counts = torch.bincount(tables[mask].long(), minlength=n).to(torch.int32)
    kv = _normal((n, case["layers"], 2, BLOCK, case["hkv"], DIM), TYPES[case["dtype"]], gd)
    return dict(kind="compact", kv=kv, counts=counts.cuda(), tables=tables.cuda(), lens=lens.cuda())


def prepare(case, seed):
    g, gd = _generators(seed)
    return {"attention": _prepare_attention, "write": _prepare_write, "rotary": _prepare_rotary, "fork": _prepare_fork,
            "compact": _prepare_compact}[case["kind"]](case, g, gd)


# ---- plain forms ------------------------------------------------------------------------------------


def _plain_attention(s):
    lens, tables, scale = s["lens"].long(), s["tables"].long(), s["scale"]
    batch, width = tables.shape
    hkv = s["hkv"]
    seen = (torch.arange(width * BLOCK, device="cuda").view(1, -1) < lens.view(-1, 1)).view(batch, 1, 1, -1)
    outs = []
    for layer in range(s["cache"].shape[1]):
        k, v = _unpack_rows(s["cache"][tables, layer])  # batch, width, head, 16, 128
        k = k.permute(0, 2, 1, 3, 4).reshape(batch, hkv, width * BLOCK, DIM)
        v = v.permute(0, 2, 1, 3, 4).reshape(batch, hkv, width * BLOCK, DIM)
        q = s["query"][layer].float().view(batch, hkv, -1, DIM)
        scores = torch.where(seen, q @ k.transpose(-1, -2) * scale, -math.inf)
        e = torch.exp(scores - scores.amax(-1, keepdim=True))
        v = torch.where(seen.view(batch, 1, -1, 1), v, 0.0)
        outs.append((e @ v / e.sum(-1, keepdim=True)).view(batch, -1, DIM).to(s["query"].dtype))
    return outs


def _plain_write(s):
    cache, slots = s["cache"], s["slots"]
    block, row = slots // BLOCK, slots % BLOCK
    heads = cache.shape[2]
    codes, pairs = _quantise(torch.stack([s["key"], s["value"]]))
    tokens = torch.zeros(2, cache.shape[0], 16, heads, DIM, dtype=torch.uint8, device="cuda")
    params = torch.zeros(2, cache.shape[0], 16, heads, 2, 2, dtype=cache.dtype, device="cuda")
    tokens[:, block, row] = codes
    params[:, block, row] = pairs
    touched = torch.zeros(cache.shape[0], 16, dtype=torch.uint8, device="cuda")
    touched[block, row] = 15
    touched = touched.view(-1, 1, 16, 1).expand(-1, heads, 16, DIM).reshape(-1, 16, DIM)
    tokens, params = tokens.transpose(2, 3).flatten(1, 2), params.transpose(2, 3).flatten(1, 2)
    new = _pack_rows(tokens[0], tokens[1], params[0], params[1])
    ones = (touched[:, :, ::32] > 0).view(-1, 16, 2, 2)
    at = _pack_rows(touched, touched, ones.to(cache.dtype), ones.to(cache.dtype))
    keep = torch.where(at[:, 1024:] != 0, -1, 0).to(torch.int16)
    mask = torch.cat([at[:, :1024].view(torch.int16), keep], 1)
    old = cache.view(torch.int16).view(-1, TILE)
    old.copy_((new.view(torch.int16) & mask) | (old & ~mask))
    k, v = _unpack_rows(cache[s["all"] // BLOCK, 0])
    pick = (s["all"] % BLOCK).view(-1, 1, 1, 1).expand(-1, heads, 1, DIM)
    return [x.gather(2, pick).squeeze(2).to(cache.dtype) for x in (k, v)]


def _plain_rotary(s):
    half = s["inv_freq"].numel()
    angle = s["positions"].double()[s["axis"]].T * s["inv_freq"].double()
    cos, sin = torch.cos(angle).float().unsqueeze(1), torch.sin(angle).float().unsqueeze(1)
    outs = []
    for x in (s["query"], s["key"]):
        a, b, rest = x[..., :half].float(), x[..., half:2 * half].float(), x[..., 2 * half:]
        outs.append(torch.cat([(a * cos - b * sin).to(x.dtype), (b * cos + a * sin).to(x.dtype), rest], -1))
    return outs


def _plain_fork(s):
    counts, tables, lens, kv = s["counts"], s["tables"], s["lens"], s["kv"]
    src, dst = s["src"], s["dst"]
    at = torch.arange(tables.shape[1], device="cuda").view(1, -1)
    held = at < ((lens[dst].long() + BLOCK - 1) // BLOCK).view(-1, 1)
    counts.index_add_(0, tables[dst].long().flatten(), -held.to(torch.int32).flatten())
    n = lens[src].long()
    blocks = (n + BLOCK - 1) // BLOCK
    need = n % BLOCK > 0
    free = torch.argsort((counts > 0).to(torch.int8), stable=True)
    new = torch.where(need, free[(torch.cumsum(need, 0) - 1).clamp(min=0)], -1)
    rows = tables[src]
    tail = (blocks - 1).clamp(min=0).view(-1, 1)
    old = rows.gather(1, tail).squeeze(1).long()
    rows = torch.where((at == tail) & need.view(-1, 1), new.view(-1, 1).to(torch.int32), rows)
    tables[dst] = torch.where(at < blocks.view(-1, 1), rows, tables[dst])
    lens[dst] = lens[src]
    counts.index_add_(0, rows.long().flatten(), (at < blocks.view(-1, 1)).to(torch.int32).flatten())
    kv[new[need]] = kv[old[need]]
    return [counts, tables, lens, new.to(torch.int32), kv]


def _plain_compact(s):
    counts, tables, kv = s["counts"], s["tables"], s["kv"]
    at = torch.arange(counts.numel(), device="cuda")
    live = counts > 0
    n_live = live.sum()
    holes, movers = at[~live & (at < n_live)], at[live & (at >= n_live)]
    kv[holes] = kv[movers]
    remap = torch.where(live, at, -1).to(torch.int32)
    remap[movers] = holes.to(torch.int32)
    new_counts = torch.where(at < n_live, counts, 0)
    new_counts[holes] = counts[movers]
    used = torch.arange(tables.shape[1], device="cuda").view(1, -1) < ((s["lens"].long() + BLOCK - 1) // BLOCK).view(-1, 1)
    new_tables = torch.where(used, remap[tables.long()], tables)
    return [new_tables, new_counts, remap, n_live.to(torch.int32).view(1), kv]


def _own_attention(s):
    from aegaeon_b200 import ops
    plan = ops.DecodePlan(s["query"].shape[1], s["query"].shape[2], s["hkv"], DIM, s["cache"].device, cache="int4").plan(s["lens"], s["tables"])
    outs = []
    for layer in range(s["cache"].shape[1]):
        out = torch.empty_like(s["query"][layer])
        ops.paged_attention_decode_int4(out, s["query"][layer], s["cache"], layer, s["tables"], s["lens"], s["scale"], plan=plan, prefetch=True)
        outs.append(out)
    return outs


def _own_write(s):
    from aegaeon_b200 import ops
    ops.reshape_and_cache_int4(s["key"], s["value"], s["cache"], 0, s["slots"])
    return list(ops.gather_cache_int4(s["cache"], 0, s["all"]))


def _own_rotary(s):
    from aegaeon_b200 import ops
    return list(ops.rotary_multi_axis(s["query"], s["key"], s["positions"], s["inv_freq"], s["sections"], interleaved=s["deal"]))


def _own_fork(s):
    from aegaeon_b200 import ops
    ops.free_blocks(s["counts"], s["tables"], s["lens"], s["dst"])
    new = ops.fork_blocks(s["kv"], s["counts"], s["tables"], s["lens"], s["src"], s["dst"])
    return [s["counts"], s["tables"], s["lens"], new, s["kv"]]


def _own_compact(s):
    from aegaeon_b200 import ops
    got = ops.compact_blocks(s["kv"], s["counts"], s["tables"], s["lens"])
    return [got.block_tables, got.ref_counts, got.remap, got.num_live, s["kv"]]


def run(state):
    if own:
        return {"attention": _own_attention, "write": _own_write, "rotary": _own_rotary, "fork": _own_fork,
                "compact": _own_compact}[state["kind"]](state)
    return {"attention": _plain_attention, "write": _plain_write, "rotary": _plain_rotary, "fork": _plain_fork,
            "compact": _plain_compact}[state["kind"]](state)


# ---- work -------------------------------------------------------------------------------------------


def _mean_length(case):
    """The mean context of a case: the lengths of one fixed seed."""
    return float(_lengths(case, 4096, torch.Generator().manual_seed(0)).double().mean())


def work(case):
    kind = case["kind"]
    if kind == "attention":
        tokens = case["batch"] * _mean_length(case)
        per_layer = tokens * case["hkv"] * 144 + 2 * case["batch"] * case["hq"] * DIM * 2 + 4 * tokens / BLOCK + 4 * case["batch"]
        return {"bytes": case["layers"] * per_layer, "flops": case["layers"] * 4 * tokens * case["hq"] * DIM}
    if kind == "write":
        n, slots, h = case["tokens"], case["blocks"] * BLOCK, case["hkv"]
        # the tokens in, their tiles out; all slots' tiles in, their keys and values out
        return {"bytes": n * h * (512 + 144) + 8 * n + slots * h * (144 + 512) + 8 * slots, "flops": 8 * (n + slots) * h * 2 * DIM}
    if kind == "rotary":
        n, heads = case["tokens"], case["hq"] + case["hkv"]
        return {"bytes": 2 * n * heads * case["dim"] * 2 + 24 * n, "flops": 3 * n * heads * case["dim"]}
    page = case["layers"] * 2 * BLOCK * case["hkv"] * DIM * 2
    if kind == "fork":
        copied = case["children"] * 15 / 16
        entries = case["children"] * (case["lo"] + case["hi"]) / 2 / BLOCK
        return {"bytes": 2 * copied * page + 24 * entries + 4 * case["blocks"], "flops": 0}
    # the live blocks beyond the number of live ones move; with random places a share 1 - live of them
    entries = case["rows"] * case["width"] / 2
    live = max(1, int(case["blocks"] * case["live"]))
    live *= 1 - math.exp(-entries / live)
    return {"bytes": 2 * live * (1 - live / case["blocks"]) * page + 8 * entries + 12 * case["blocks"], "flops": 0}


# ---- from the definitions, in 64 bits ---------------------------------------------------------------


def _exact_attention(s):
    outs = [torch.empty(s["query"][0].shape, dtype=torch.float64, device="cuda") for _ in range(s["cache"].shape[1])]
    group = s["query"].shape[2] // s["hkv"]
    for b, n in enumerate(s["lens"].tolist()):
        ids = s["tables"][b, :(n + BLOCK - 1) // BLOCK].long()
        for layer, out in enumerate(outs):
            k, v = (x.view(-1, s["hkv"], 16, DIM).transpose(0, 1).reshape(s["hkv"], -1, DIM)[:, :n] for x in
                    _exact_tiles(s["cache"][ids, layer].reshape(-1, TILE)))
            p = torch.softmax(torch.einsum("hgd,htd->hgt", s["query"][layer, b].double().view(s["hkv"], group, DIM), k) * s["scale"], -1)
            out[b] = torch.einsum("hgt,htd->hgd", p, v).reshape(-1, DIM)
    return outs


def _nearest(v, dtype):
    """The values of a 16-bit type nearest to 64-bit ones: of a cast's result and its two neighbours the nearest, the even one of two."""
    first = v.to(dtype)
    bits = first.view(torch.int16).long()
    around = torch.stack([bits - 1, bits, bits + 1]).clamp(min=0)
    values = around.to(torch.int16).view(dtype).double()
    off = (values - v).abs()
    off = torch.where(torch.isfinite(values), off, math.inf)
    best = torch.where(off == off.amin(0), (around % 2).double(), 9.0).argmin(0, keepdim=True)
    return values.gather(0, best).squeeze(0)


def _exact_write(s):
    out = []
    dtype, heads = s["cache"].dtype, s["cache"].shape[2]
    for x in (s["key"], s["value"]):
        rows = x.double().reshape(-1, 64)
        low = rows.min(1).values
        step = _nearest((rows.max(1).values - low) / 15, dtype)
        below = torch.floor((rows - low[:, None]) / step[:, None]).clamp(0, 15)  # then the nearer of two levels, the even one of a tie
        rest = (rows - low[:, None]) - below * step[:, None]
        up = (2 * rest > step[:, None]) | ((2 * rest == step[:, None]) & (below % 2 == 1))
        code = torch.where(step[:, None] > 0, (below + up).clamp(0, 15), 0.0)
        all_slots = torch.zeros(s["all"].numel(), heads, DIM, dtype=torch.float64, device="cuda")
        all_slots[s["slots"]] = (code * step[:, None] + low[:, None]).view(-1, heads, DIM)
        out.append(all_slots)
    return out


def _exact_rotary(s):
    half = s["inv_freq"].numel()
    outs = []
    order = _axis_of(s["sections"], s["deal"])
    theta = torch.stack([s["positions"][a].double() * f for a, f in zip(order, s["inv_freq"].double())], 1)
    turn = torch.polar(torch.ones_like(theta), theta)[:, None]
    for x in (s["query"], s["key"]):
        w = x.double()
        z = torch.complex(w[..., :half].contiguous(), w[..., half:2 * half].contiguous()) * turn
        outs.append(torch.cat([z.real, z.imag, w[..., 2 * half:]], -1))
    return outs


def _exact_fork(s):
    counts, tables, lens = s["counts"].tolist(), s["tables"].tolist(), s["lens"].tolist()
    kv = s["kv"].double()
    for row in s["dst"].tolist():
        for j in range(-(-lens[row] // BLOCK)):
            counts[tables[row][j]] -= 1
        lens[row] = 0
    free = [b for b, c in enumerate(counts) if c == 0]
    new = []
    for a, row in zip(s["src"].tolist(), s["dst"].tolist()):
        n = -(-lens[a] // BLOCK)
        tables[row][:n] = tables[a][:n]
        lens[row] = lens[a]
        new.append(-1)
        if lens[a] % BLOCK:
            new[-1] = tables[row][n - 1] = free.pop(0)
            kv[new[-1]] = s["kv"][tables[a][n - 1]].double()
        for j in range(n):
            counts[tables[row][j]] += 1
    return [torch.tensor(x) for x in (counts, tables, lens, new)] + [kv]


def _exact_compact(s):
    counts, tables = s["counts"].tolist(), s["tables"].tolist()
    kv = s["kv"].double()
    n_live = sum(c > 0 for c in counts)
    remap = [b if c > 0 else -1 for b, c in enumerate(counts)]
    new = counts[:n_live] + [0] * (len(counts) - n_live)
    hole = 0
    for b in range(n_live, len(counts)):
        if counts[b] > 0:
            while counts[hole] > 0:
                hole += 1
            kv[hole] = s["kv"][b].double()
            remap[b], new[hole] = hole, counts[b]
            hole += 1
    for row, n in zip(tables, s["lens"].tolist()):
        for j in range(-(-n // BLOCK)):
            row[j] = remap[row[j]]
    return [torch.tensor(x) for x in (tables, new, remap, [n_live])] + [kv]


def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "write": _exact_write, "rotary": _exact_rotary, "fork": _exact_fork,
            "compact": _exact_compact}[case["kind"]](s)
