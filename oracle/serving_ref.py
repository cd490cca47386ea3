"""CPU oracle of the 4-bit KV cache, the multi-axis rotary positions and the shared-block calls —
TEST INFRASTRUCTURE ONLY, written from their definitions in 64 bits (torch on the CPU, plain Python
for the block bookkeeping), one element or entry at a time where that is affordable."""
from __future__ import annotations

import math
from fractions import Fraction

import torch

TILE, DIM, GROUP = 1152, 128, 64

DIGITS = {torch.float16: (11, -14), torch.bfloat16: (8, -126)}  # significant bits, least normal exponent


def half_step(dtype: torch.dtype) -> float:
    """A rounding's largest relative error."""
    return torch.finfo(dtype).eps / 2


def round_fraction(x: Fraction, dtype: torch.dtype) -> Fraction:
    """The value of ``dtype`` nearest to a positive ``x``, ties to even, in exact arithmetic."""
    if x == 0:
        return x
    bits, least = DIGITS[dtype]
    e = math.floor(math.log2(x)) if x > 0 else 0
    while Fraction(2) ** e > x:
        e -= 1
    while Fraction(2) ** (e + 1) <= x:
        e += 1
    unit = Fraction(2) ** (max(e, least) - bits + 1)
    return Fraction(round(x / unit)) * unit  # Python rounds a Fraction half to even


def quantise_fraction(row: list[float], dtype: torch.dtype):
    """(codes, scale, minimum) of one 64-dim group in exact arithmetic."""
    x = [Fraction(v) for v in row]
    lo = min(x)
    scale = round_fraction((max(x) - lo) / 15, dtype)
    codes = [min(15, round((v - lo) / scale)) if scale else 0 for v in x]
    return codes, float(scale), float(lo)


def round_once(v: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """64-bit values rounded to ``dtype`` in one step (a cast goes through 32 bits)."""
    bits, least = DIGITS[dtype]
    unit = torch.ldexp(torch.ones_like(v), (torch.frexp(v)[1] - 1).clamp(min=least) - bits + 1)
    return (torch.round(v / unit) * unit).to(dtype)


def quantise(x: torch.Tensor):
    """Codes uint8 [..., 128] and pairs [..., 2 groups, (scale, minimum)] of 16-bit rows [..., 128]."""
    g = x.double().unflatten(-1, (2, GROUP))
    lo, hi = g.amin(-1), g.amax(-1)
    bad = ~torch.isfinite(hi.float() - lo.float())
    scale = round_once(torch.where(bad, 0.0, hi - lo) / 15, x.dtype)
    steps = (g - lo.unsqueeze(-1)) / scale.double().unsqueeze(-1)
    flat = (bad | (scale == 0)).unsqueeze(-1)
    codes = torch.round(torch.where(flat, 0.0, steps)).clamp(0, 15).to(torch.uint8)
    pairs = torch.stack([scale, lo.to(x.dtype)], -1)
    pairs[bad] = math.nan
    return codes.flatten(-2), pairs


def _offsets():
    """Byte offsets [16 tokens, 128 dims] of the key and value codes within a tile (nibble d % 2)."""
    t = torch.arange(16).view(16, 1)
    d = torch.arange(DIM).view(1, DIM)
    key = t * 64 + d % 32 // 8 * 16 + d // 32 * 4 + d % 8 // 2
    value = 1024 + t // 2 * 128 + d % 64 // 8 * 16 + d // 64 * 8 + d % 8 // 4 * 4 + t % 2 * 2 + d % 4 // 2
    return key, value


KEY_AT, VALUE_AT = _offsets()


def write(cache: torch.Tensor, layer: int, key: torch.Tensor, value: torch.Tensor, slots) -> None:
    """reshape_and_cache_int4 on a CPU cache (N, L, Hkv, 1152): byte by byte, token by token."""
    raw = cache.view(torch.uint8).view(cache.size(0), cache.size(1), cache.size(2), 2 * TILE)
    for what, (x, at, pairs_at) in enumerate(((key, KEY_AT, 2048), (value, VALUE_AT, 2176))):
        codes, pairs = quantise(x)
        packed = codes[..., 0::2] | (codes[..., 1::2] << 4)
        pair_bytes = pairs.contiguous().view(torch.uint8).reshape(*pairs.shape[:2], 8)
        for i, s in enumerate(slots):
            s = int(s)
            if 0 <= s < cache.size(0) * 16:
                tile = raw[s // 16, layer]
                tile[:, at[s % 16, 0::2]] = packed[i]
                tile[:, pairs_at + s % 16 * 8:pairs_at + s % 16 * 8 + 8] = pair_bytes[i]


def values(tiles: torch.Tensor):
    """Keys and values [..., 16, 128] in 64 bits that CPU tiles [..., 1152] hold."""
    lead = tiles.shape[:-1]
    raw = tiles.contiguous().view(torch.uint8).reshape(-1, 2 * TILE)
    wide = tiles.double().reshape(-1, TILE)
    nib = 4 * (torch.arange(DIM) % 2)
    out = []
    for at, first in ((KEY_AT, 1024), (VALUE_AT, 1088)):
        code = (raw[:, at].to(torch.int64) >> nib) & 15
        p = first + torch.arange(16).view(16, 1) * 4 + torch.arange(DIM).view(1, DIM) // GROUP * 2
        out.append((code.double() * wide[:, p] + wide[:, p + 1]).view(*lead, 16, DIM))
    return out


def gather(cache: torch.Tensor, layer: int, slots) -> list[torch.Tensor]:
    """gather_cache_int4: one rounding to fp32, one to the cache's type; zeros for slots outside."""
    k, v = values(cache[:, layer])  # N, Hkv, 16, 128
    out = []
    for x in (k, v):
        rows = torch.zeros(len(slots), cache.size(2), DIM, dtype=torch.float64)
        for i, s in enumerate(slots):
            if 0 <= int(s) < cache.size(0) * 16:
                rows[i] = x[int(s) // 16, :, int(s) % 16]
        out.append(rows.float().to(cache.dtype))
    return out


def attention(q: torch.Tensor, cache: torch.Tensor, layer: int, tables, lens, scale: float) -> torch.Tensor:
    """Decode attention over a CPU 4-bit cache, in 64 bits; a length of 0 gives a zero row."""
    B, Hq, _ = q.shape
    Hkv = cache.size(2)
    out = torch.zeros(B, Hq, DIM, dtype=torch.float64)
    for b in range(B):
        n = int(lens[b])
        if n <= 0:
            continue
        ids = torch.as_tensor([int(i) for i in tables[b][:(n + 15) // 16]])
        k, v = values(cache[ids, layer])
        k, v = (x.transpose(0, 1).reshape(Hkv, -1, DIM)[:, :n] for x in (k, v))
        s = torch.einsum("hgd,htd->hgt", q[b].double().view(Hkv, -1, DIM), k) * scale
        out[b] = torch.einsum("hgt,htd->hgd", torch.softmax(s, -1), v).reshape(Hq, DIM)
    return out


def axes_of(sections, interleaved: bool) -> list[int]:
    if not interleaved:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    left, order = list(sections), []
    while sum(left):
        for a in range(len(left)):
            if left[a] > 0:
                left[a] -= 1
                order.append(a)
    return order


def rotary(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, sections, interleaved: bool,
           scaling: float = 1.0) -> torch.Tensor:
    half = inv_freq.numel()
    order = axes_of(sections, interleaved)
    theta = torch.stack([positions[a].double() * float(f) for a, f in zip(order, inv_freq)], 1).unsqueeze(1)
    a, b = x[..., :half].double(), x[..., half:2 * half].double()
    cos, sin = torch.cos(theta) * scaling, torch.sin(theta) * scaling
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:].double()], -1)


class Pool:
    """The shared-block calls on plain lists, entry by entry."""

    def __init__(self, counts, tables, lens, blocks):
        self.counts, self.tables, self.lens = [int(c) for c in counts], [list(map(int, r)) for r in tables], [int(n) for n in lens]
        self.blocks = blocks  # a CPU tensor of the pool's blocks, or None
        self.width = len(self.tables[0]) if self.tables else 0

    def fork(self, src, dst):
        before, counts = list(self.lens), list(self.counts)
        taken, new, errors = set(), [], set()
        free = [b for b, c in enumerate(self.counts) if c == 0]
        copies = []
        for s, d in zip(src, dst):
            new.append(-1)
            if not (0 <= s < len(before) and 0 <= d < len(before)) or not 0 <= before[s] <= 16 * self.width or before[d] != 0:
                errors.add("entry")
                continue
            n = (before[s] + 15) // 16
            if before[s] % 16 and not 0 <= self.tables[s][n - 1] < len(self.counts):
                errors.add("id")
                continue
            if before[s] % 16 and counts[self.tables[s][n - 1]] <= 0:
                errors.add("entry")
                continue
            if d in taken:
                errors.add("entry")
                continue
            taken.add(d)
            if before[s] % 16:
                if not free:
                    errors.add("empty")
                    continue
                new[-1] = free.pop(0)
            row = self.tables[s][:n]
            if new[-1] >= 0:
                copies.append((row[-1], new[-1]))
                row[-1] = new[-1]
            self.tables[d][:n] = row
            self.lens[d] = before[s]
            for b in row:
                if 0 <= b < len(self.counts):
                    self.counts[b] += 1
                else:
                    errors.add("id")
        if self.blocks is not None:
            for a, b in copies:
                self.blocks[b] = self.blocks[a]
        return new, errors

    def free(self, rows):
        errors = set()
        for r in rows:
            if not 0 <= r < len(self.lens):
                errors.add("entry")
                continue
            for b in self.tables[r][:(self.lens[r] + 15) // 16]:
                if not 0 <= b < len(self.counts):
                    errors.add("id")
                elif self.counts[b] > 0:
                    self.counts[b] -= 1
                else:
                    errors.add("entry")
            self.lens[r] = 0
        return errors

    def compact(self):
        live = [b for b, c in enumerate(self.counts) if c > 0]
        n = len(live)
        remap = [b if c > 0 else -1 for b, c in enumerate(self.counts)]
        counts = [max(c, 0) if b < n else 0 for b, c in enumerate(self.counts)]
        holes = [b for b in range(n) if self.counts[b] <= 0]
        for b, to in zip([b for b in live if b >= n], holes):
            remap[b], counts[to] = to, self.counts[b]
            if self.blocks is not None:
                self.blocks[to] = self.blocks[b]
        tables = []
        for row, length in zip(self.tables, self.lens):
            used = (min(max(length, 0), 16 * self.width) + 15) // 16
            tables.append([remap[b] if j < used and 0 <= b < len(remap) and remap[b] >= 0 else b for j, b in enumerate(row)])
        return tables, counts, remap, n
