"""Plain float64 arithmetic and byte-by-byte layout of the ops between the q / k / v projections and the o projection: what the GPU tests
check against.  Nothing here is fast, and nothing is shared with the library."""
import numpy as np


def slices(x):
    """[tokens][heads][head_dim] -> [channels / 4][tokens][4]"""
    x = np.asarray(x)
    return np.ascontiguousarray(x.reshape(x.shape[0], -1, 4).transpose(1, 0, 2))


def unslices(x, head_dim):
    return np.ascontiguousarray(x.transpose(1, 0, 2)).reshape(x.shape[1], -1, head_dim)


def norm_rope(x, positions, rotary, interleaved, weight=None, offset=0.0, eps=1e-6, base=10000.0, frequencies=None):
    x = np.asarray(x, np.float64)
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + np.float64(np.float32(eps))) * (offset + weight.astype(np.float64))
    r = rotary
    if r == 0:
        return x
    if frequencies is None:
        frequencies = np.longdouble(base) ** (-2 * np.arange(r // 2, dtype=np.longdouble) / r)
    turns = np.asarray(positions, np.longdouble)[:, None] * (np.asarray(frequencies, np.longdouble) / (2 * np.longdouble("3.14159265358979323846264338327950288")))
    t = (2 * np.pi * (turns - np.floor(turns)).astype(np.float64))[:, None]
    y = x.copy()
    one, two = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    a, b = x[..., one], x[..., two]
    y[..., one], y[..., two] = a * np.cos(t) - b * np.sin(t), b * np.cos(t) + a * np.sin(t)
    return y


# every scale there is: 7 significant bits, multiples of 2^-20 at the small end
SCALES = np.unique(np.concatenate([np.arange(64) * 2.0**-20] + [np.arange(64, 128) * 2.0**e for e in range(-20, 10)]))


def quantized(x, group):
    """codes [..., head_dim], scales and zero points [..., head_dim / group] of float64 values."""
    with np.errstate(invalid="ignore"):
        x = np.where(np.isnan(x), 0.0, np.clip(x, -57344.0, 57344.0))
    g = x.reshape(*x.shape[:-1], -1, group)
    low, high = np.minimum(g.min(-1), 0), np.maximum(g.max(-1), 0)
    scale = SCALES[np.searchsorted(15 * SCALES, high - low)]
    safe = np.where(scale > 0, scale, 1.0)
    zero = np.rint(-low / safe)
    codes = np.clip(np.rint(g / safe[..., None]) + zero[..., None], 0, 15)
    return codes.reshape(x.shape).astype(int), scale, zero.astype(int)


def kept(x, group):
    codes, scale, zero = quantized(np.asarray(x, np.float64), group)
    g = codes.reshape(*codes.shape[:-1], -1, group)
    return (scale[..., None] * (g - zero[..., None])).reshape(codes.shape)


class Cache:
    """The bytes of a cache, written nibble by nibble where the layout's description puts them."""

    def __init__(self, kv_heads, head_dim, group, page, pages):
        self.kv_heads, self.head_dim, self.group, self.page, self.pages = kv_heads, head_dim, group, page, pages
        self.block = page * (head_dim + 4 * (head_dim // group))
        self.bytes = np.zeros(pages * kv_heads * self.block, np.uint8)
        p = min(head_dim, 128)
        c = np.arange(head_dim)
        i1, i = c // p, c % p
        # nibble inside a tile's codes for (token, channel), and the word of (token, group) inside a tile's words
        t = np.arange(16)[:, None]
        key = (i1 * 16 + t) * p + i % 32 // 8 * (p // 4) + i // 32 * 8 + i % 8
        per = p // 16
        value = ((i1 * 4 + t // 4) * 16 + i // per) * (4 * per) + i % per // 4 * 16 + t % 4 // 2 * 8 + t % 2 * 4 + i % 4
        self.nibble = {"k": key, "v": value}
        g = np.arange(head_dim // group)
        self.word = g[None] * 16 + t

    def _at(self, page, head):
        return (int(page) * self.kv_heads + head) * self.block

    def _codes(self, which, offset):
        return (0 if which == "k" else self.page * self.head_dim // 2) + offset // 16 * 8 * self.head_dim

    def _words(self, which, offset):
        n = self.head_dim // self.group
        return self.page * self.head_dim + (0 if which == "k" else 2 * self.page * n) + offset // 16 * 32 * n

    def set_token(self, page, offset, k, v):
        """k, v: [kv_heads][head_dim]"""
        for which, x in (("k", k), ("v", v)):
            codes, scale, zero = quantized(np.asarray(x, np.float64), self.group)
            words = (scale.astype(np.float16).view(np.uint16) | zero.astype(np.uint16)).astype("<u2")
            for h in range(self.kv_heads):
                at = self._at(page, h)
                nib = self.nibble[which][offset % 16]
                byte = at + self._codes(which, offset) + nib // 2
                low = nib % 2 == 0
                self.bytes[byte[low]] = (self.bytes[byte[low]] & 0xF0) | codes[h][low]
                self.bytes[byte[~low]] = (self.bytes[byte[~low]] & 0x0F) | (codes[h][~low] << 4)
                w = at + self._words(which, offset) + 2 * self.word[offset % 16]
                self.bytes[w], self.bytes[w + 1] = words[h] & 255, words[h] >> 8

    def set_all(self, k, v):
        """k, v: [pages][kv_heads][page][head_dim]"""
        blocks = self.bytes.reshape(self.pages, self.kv_heads, self.block)
        for which, x in (("k", k), ("v", v)):
            codes, scale, zero = quantized(np.asarray(x, np.float64), self.group)
            words = scale.astype(np.float16).view(np.uint16) | zero.astype(np.uint16)
            for tile in range(self.page // 16):
                nibbles = np.zeros((self.pages, self.kv_heads, 16 * self.head_dim), np.uint8)
                nibbles[..., self.nibble[which].ravel()] = codes[:, :, 16 * tile:16 * tile + 16].reshape(self.pages, self.kv_heads, -1)
                at = self._codes(which, 16 * tile)
                blocks[..., at:at + 8 * self.head_dim] = nibbles[..., 0::2] | (nibbles[..., 1::2] << 4)
                w = np.zeros((self.pages, self.kv_heads, self.word.size), "<u2")
                w[..., self.word.ravel()] = words[:, :, 16 * tile:16 * tile + 16].reshape(self.pages, self.kv_heads, -1)
                at = self._words(which, 16 * tile)
                blocks[..., at:at + 2 * self.word.size] = w.view(np.uint8)

    def spoil(self, table, lengths):
        """NaN words and other codes at every position that no sequence holds."""
        held = np.zeros((self.pages, self.page), bool)
        for row, n in zip(table, lengths):
            for p in range(min(n, len(row) * self.page)):
                if 0 <= row[p // self.page] < self.pages:
                    held[row[p // self.page], p % self.page] = True
        blocks = self.bytes.reshape(self.pages, self.kv_heads, self.block)
        for page, offset in np.argwhere(~held):
            for which in "kv":
                w = self._words(which, offset) + 2 * self.word[offset % 16]
                blocks[page][:, w], blocks[page][:, w + 1] = 0xF3, 0x7F

    def values(self):
        """keys, values [pages][kv_heads][page][head_dim]"""
        blocks = self.bytes.reshape(self.pages, self.kv_heads, self.block)
        found = []
        for which in "kv":
            x = np.zeros((self.pages, self.kv_heads, self.page, self.head_dim))
            for offset in range(self.page):
                nib = self.nibble[which][offset % 16]
                b = blocks[..., self._codes(which, offset) + nib // 2]
                code = np.where(nib % 2 == 0, b & 15, b >> 4).astype(np.float64)
                w = self._words(which, offset) + 2 * self.word[offset % 16]
                bits = blocks[..., w].astype(np.uint16) | (blocks[..., w + 1].astype(np.uint16) << 8)
                scale = np.repeat((bits & 0xFFF0).astype(np.uint16).view(np.float16).astype(np.float64), self.group, -1)
                x[:, :, offset] = scale * (code - np.repeat((bits & 15).astype(np.float64), self.group, -1))
            found.append(x)
        return found


def attention(q, cache, table, lengths, starts, scale, causal, window, fill=0.0):
    """-> (outputs [tokens][heads][head_dim], the largest |v| that a row sees, the largest scale * sum |q||k|), the last two to be
    broadcast against the outputs; rows of no sequence hold `fill`."""
    q = np.asarray(q, np.float64)
    keys, values = cache.values()
    tokens, heads, d = q.shape
    share = heads // cache.kv_heads
    out, largest, score = np.full(q.shape, fill), np.zeros((tokens, heads, 1)), np.zeros((tokens, heads, 1))
    scale = np.float64(np.float32(scale))
    for s in range(len(lengths)):
        n = starts[s + 1] - starts[s]
        held = min(int(lengths[s]), table.shape[1] * cache.page)
        at = np.arange(held)
        page = table[s][at // cache.page] if held else np.zeros(0, int)
        there = (page >= 0) & (page < cache.pages)
        at, page = at[there], page[there]
        k, v = keys[page, :, at % cache.page], values[page, :, at % cache.page]  # [positions][kv_heads][head_dim]
        for i in range(n):
            row = starts[s] + i
            position = lengths[s] - n + i
            seen = np.ones(len(at), bool)
            if causal:
                seen &= at <= position
            if window:
                seen &= at > position - window
            if not seen.any():
                out[row] = 0
                continue
            for h in range(heads):
                ks, vs = k[seen, h // share], v[seen, h // share]
                z = scale * (ks @ q[row, h])
                w = np.exp(z - z.max())
                out[row, h] = (w / w.sum()) @ vs
                largest[row, h] = np.abs(vs).max()
                score[row, h] = (scale * np.abs(ks) @ np.abs(q[row, h])).max()
    return out, largest, score
