"""Plain statement, in 64 bits and on the CPU, of the cache of e4m3 codes: the codes' numbers, the append, the maps of a step and
attention over the numbers.  Shares no code with the package under test."""

import math

import torch

F64 = torch.float64
BLOCK = 16


def numbers():
    """What the 256 codes stand for (1 sign, 4 exponent, 3 fraction bits, bias 7; no infinity, one NaN of each sign)."""
    out = []
    for c in range(256):
        e, f = (c >> 3) & 15, c & 7
        x = math.nan if c & 127 == 127 else f / 8 * 2.0 ** -6 if e == 0 else (1 + f / 8) * 2.0 ** (e - 7)
        out.append(-x if c & 128 else x)
    return torch.tensor(out, dtype=F64)


NUMBERS = numbers()


def nearest(x):
    """The nearest number that a code has, ties to the even code, within the format's range; x float64."""
    steps = NUMBERS[:127]
    size = x.abs().clamp(max=448.0)
    up = torch.searchsorted(steps, size).clamp(1, 126)
    low, high = steps[up - 1], steps[up]
    take = (size - low > high - size) | ((size - low == high - size) & (up % 2 == 0))
    return torch.copysign(torch.where(take, high, low), x)


def exponent(largest: float) -> int:
    """The smallest e in -100 .. 119 with largest <= 448 * 2^e (119 where there is none)."""
    if largest == 0:
        return -100
    m, k = math.frexp(largest)
    return min(max(k - 9 + (1 if m > 0.875 else 0), -100), 119)


class Cache:
    """One sequence's keys and values as the cache holds them: `codes` float64 numbers of the codes and `scales` per 16 positions, each
    [2, kv heads, ...]; grows by `append`."""

    def __init__(self, kv_heads, dim):
        self.kv_heads, self.dim, self.length = kv_heads, dim, 0
        self.codes = torch.zeros(2, kv_heads, 0, dim, dtype=F64)
        self.scales = torch.zeros(2, kv_heads, 0, dtype=F64)

    def append(self, k, v):
        """k, v float64 [new, kv heads, dim], as they are before rounding."""
        new = torch.stack([k, v]).transpose(1, 2)                 # [2, kv heads, new, dim]
        n, start = new.shape[2], self.length
        end = start + n
        self.codes = torch.cat([self.codes, torch.zeros(2, self.kv_heads, n, self.dim, dtype=F64)], 2)
        blocks = -(-end // BLOCK)
        more = blocks - self.scales.shape[2]
        self.scales = torch.cat([self.scales, torch.zeros(2, self.kv_heads, more, dtype=F64)], 2)
        for b in range(start // BLOCK, blocks):
            lo, hi = max(b * BLOCK, start), min((b + 1) * BLOCK, end)
            held = lo - b * BLOCK
            for h in range(self.kv_heads):
                spoilt = False
                for w in (0, 1):
                    x = new[w, h, lo - start: hi - start]
                    fine = x.isfinite()
                    spoilt |= not bool(fine.all())
                    x = torch.where(fine, x, 0.0)
                    e = exponent(float(x.abs().max()))
                    was = float(self.scales[w, h, b]) if held else 0.0
                    if held and math.isnan(was):
                        spoilt = True
                    elif held:
                        before = math.frexp(was)[1] - 1
                        e = max(e, before)
                        if e > before:
                            self.codes[w, h, b * BLOCK: lo] = nearest(self.codes[w, h, b * BLOCK: lo] * 2.0 ** (before - e))
                    self.scales[w, h, b] = 2.0 ** e
                    self.codes[w, h, lo:hi] = nearest(x * 2.0 ** -e)
                if spoilt:
                    self.scales[0, h, b] = math.nan
        self.length = end

    def values(self):
        """[2, kv heads, length, dim] numbers that the cache stands for."""
        return self.codes * self.scales.repeat_interleave(BLOCK, -1)[..., : self.length, None]


def rotate(x, positions, inv_freq):
    """x [tokens, heads, dim] turned by position * inv_freq, halves paired; 64 bits."""
    angle = positions.to(F64)[:, None, None] * inv_freq.to(F64)
    half = x.shape[-1] // 2
    lo, hi = x[..., :half], x[..., half:]
    return torch.cat([lo * angle.cos() - hi * angle.sin(), hi * angle.cos() + lo * angle.sin()], -1)


def attention(q, k, v, first, scale, window=0, chunk=0, sink=None, gate=None):
    """q [new, heads, dim] at positions first, first + 1, ...; k, v [kv heads, length, dim]; returns (out, the sum of the
    weights times the values' sizes), both [new, heads, dim].  A row that sees nothing is zero."""
    new, heads, _dim = q.shape
    kv_heads, length, _ = k.shape
    group = heads // kv_heads
    position = torch.arange(first, first + new)[:, None]
    key = torch.arange(length)[None]
    visible = key <= position
    if window:
        visible &= key > position - window
    if chunk:
        visible &= key >= position // chunk * chunk
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    for h in range(heads):
        s = q[:, h] @ k[h // group].t() * scale
        s = torch.where(visible, s, -math.inf)
        if sink is not None:
            s = torch.cat([s, sink[h].expand(new, 1)], 1)
        top = s.max(1, keepdim=True).values
        p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
        total = p.sum(1, keepdim=True)
        w = torch.where(total == 0, 0.0, p / total)[:, :length]
        mine = v[h // group]
        out[:, h] = torch.where(visible[..., None], w[..., None] * mine[None], 0.0).sum(1)
        bound[:, h] = torch.where(visible[..., None], w[..., None] * mine[None].abs(), 0.0).sum(1)
        if gate is not None:
            g = torch.sigmoid(gate[:, h])[:, None]
            out[:, h] *= g
            bound[:, h] *= g
    return out, bound


def maps(cached, q_len, pages, page, group, tile_rows, few_rows, max_blocks, n_rows):
    """The maps of a step as lists, request by request (cached < 0: an idle row)."""
    out = {name: [] for name in ("seq_q_start", "seq_q_len", "seq_kv_len", "positions", "row_seq", "slots", "block_table", "write_seq",
                                 "write_block", "tile_seq", "tile_index")}
    row = at = 0
    for s, (c, n) in enumerate(zip(cached, q_len)):
        idle = c < 0
        kv = 0 if idle else c + n
        blocks = 0 if idle else -(-kv // page)
        mine = pages[at: at + blocks]
        at += blocks
        out["seq_q_start"].append(row)
        out["seq_q_len"].append(0 if idle else n)
        out["seq_kv_len"].append(kv)
        out["block_table"].append((mine + [-1] * max_blocks)[:max_blocks])
        for i in range(n):
            p = 0 if idle else c + i
            held = -1 if idle or p // page >= max_blocks else mine[p // page]
            out["positions"].append(p)
            out["row_seq"].append(s)
            out["slots"].append(held * page + p % page if held >= 0 else -1)
        if not idle and n:
            for b in range(c // BLOCK, (kv - 1) // BLOCK + 1):
                out["write_seq"].append(s)
                out["write_block"].append(b)
            if n * group > few_rows:
                for t in range(-(-n * group // tile_rows)):
                    out["tile_seq"].append(s)
                    out["tile_index"].append(t)
        row += n
    for name, fill, n in (("positions", 0, n_rows), ("row_seq", -1, n_rows), ("slots", -1, n_rows)):
        out[name] += [fill] * (n - len(out[name]))
    seqs = len(cached)
    out["order"] = sorted(range(seqs), key=lambda s: (-out["seq_kv_len"][s], s))
    for name, fill, n in (("write_seq", -1, min(n_rows, n_rows // BLOCK + 2 * seqs)), ("write_block", 0, min(n_rows, n_rows // BLOCK + 2 * seqs)),
                          ("tile_seq", -1, n_rows * group // tile_rows + seqs), ("tile_index", 0, n_rows * group // tile_rows + seqs)):
        assert len(out[name]) <= n, (name, len(out[name]), n)
        out[name] += [fill] * (n - len(out[name]))
    return out
