"""The ops between the q / k / v projections and the o projection against plain arithmetic in 64 bits."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

import mldhip as M
import workloads as W
from kv4math import Cache, attention, kept, norm_rope, slices, unslices

torch = pytest.importorskip("torch")


def stream():
    return torch.cuda.current_stream().cuda_stream


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


# ---- norms and rotation ------------------------------------------------------------------------------------------------------

def run_norm_rope(q, k, positions, rotary, interleaved, dtype, norm=None, base=10000.0, frequencies=None, eps=1e-6, offset=0.0, in_place=False):
    """q, k: [tokens][heads][head_dim]; norm: (q weight, k weight) or None."""
    t, h, d = q.shape
    hk = k.shape[1]
    sq, sk = dev(slices(q).astype(dtype)), dev(slices(k).astype(dtype))
    oq, ok = (sq, sk) if in_place else (torch.full_like(sq, 7.0), torch.full_like(sk, 7.0))
    op = M.qk_norm_rope_create(M.FLOAT16 if dtype == np.float16 else M.FLOAT32, h, hk, d, rotary_dim=rotary, base=base, frequencies=frequencies,
                               interleaved=interleaved, norm=norm is not None, eps=eps, weight_offset=offset, max_tokens=t)
    srcs = [sq, sk, dev(positions.astype(np.int32))]
    if norm is not None:
        srcs += [dev(norm[0].astype(dtype)), dev(norm[1].astype(dtype))]
    op.bind(srcs, [oq, ok])
    op.set_shape(1, 1, t)
    print("norm_rope", t, h, hk, d, rotary, interleaved, dtype.__name__, norm is not None, flush=True)
    op.launch(stream())
    torch.cuda.synchronize()
    assert op.kernel_name == "qk_norm_rope_kernel"
    return unslices(oq.cpu().numpy(), d), unslices(ok.cpu().numpy(), d)


# What the kernel may be off by, relative to the length of a pair (a rotation keeps it): the rounding of the result, half a step
# (2^-11 / 2^-24 of it); the sine's and cosine's own error (hardware ones 2^-19 for halfs, 4 ulp of fp32 plus 2 pi 2^-26 of the angle
# otherwise); with norms the sum of head_dim squares, the root, the reciprocal and three products, 12 roundings of 2^-24 at most where
# the sum is of positive terms (its own error is at most 64 additions of a lane and 4 across, half of them by the root).
def rope_tolerance(dtype, norm):
    eps = 2.0**-11 + 2.0**-19 if dtype == np.float16 else 2.0**-24 + 8 * 2.0**-24 + 2 * math.pi * 2.0**-26
    return eps + (12 + 34) * 2.0**-24 * (norm is not None) + 3 * 2.0**-24


def check_rope(got, exact, tol, rotary, interleaved):
    mag = np.abs(exact).copy()
    r = rotary
    a, b = (exact[..., 0:r:2], exact[..., 1:r:2]) if interleaved else (exact[..., :r // 2], exact[..., r // 2:r])
    length = np.sqrt(a * a + b * b)
    if interleaved:
        mag[..., 0:r:2] = mag[..., 1:r:2] = length
    else:
        mag[..., :r // 2] = mag[..., r // 2:r] = length
    err = np.abs(got.astype(np.float64) - exact)
    bad = err > tol * mag + 2.0**-25  # (subnormal halves: half a step is 2^-25)
    assert not bad.any(), (np.argwhere(bad)[:3], got[bad][:3], exact[bad][:3])


@pytest.mark.parametrize("tokens,heads,kv_heads,head_dim,rotary", [
    (1, 8, 1, 256, 256), (3, 4, 2, 128, 128), (15, 2, 2, 64, 32), (16, 5, 1, 64, 64), (17, 3, 3, 128, 64), (63, 2, 1, 256, 128),
    (65, 4, 4, 80, 80), (200, 6, 2, 96, 96), (513, 5, 2, 128, 128), (700, 3, 1, 8, 8), (530, 1, 1, 256, 0), (33, 2, 1, 24, 16)])
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("with_norm", [False, True])
def test_norm_rope(tokens, heads, kv_heads, head_dim, rotary, dtype, interleaved, with_norm):
    rng = np.random.default_rng(tokens * 7 + heads)
    q = rng.standard_normal((tokens, heads, head_dim)).astype(dtype)
    k = rng.standard_normal((tokens, kv_heads, head_dim)).astype(dtype)
    norm = tuple(rng.standard_normal(head_dim).astype(dtype) for _ in range(2)) if with_norm else None
    positions = rng.integers(0, 5000, tokens)
    got = run_norm_rope(q, k, positions, rotary, interleaved, dtype, norm, offset=1.0 if with_norm else 0.0)
    for x, y, w in zip((q, k), got, norm or (None, None)):
        exact = norm_rope(x, positions, rotary, interleaved, weight=w, offset=1.0)
        # (what the norm multiplies by is at most |1 + w|: the same factor for error and value)
        check_rope(y, exact, rope_tolerance(dtype, norm), rotary, interleaved)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_norm_rope_far_and_negative_positions(dtype):
    rng = np.random.default_rng(5)
    q, k = rng.standard_normal((40, 2, 64)).astype(dtype), rng.standard_normal((40, 1, 64)).astype(dtype)
    positions = np.concatenate([[0, 1, -1, -77777, 2**31 - 1, -2**31, 2**24 + 1, 10**9], rng.integers(-2**31, 2**31, 32)])
    # float64 angles lose 2^-53 of up to 2^31 radians: 2^-22; the reference takes whole turns out in extended precision
    got = run_norm_rope(q, k, positions, 64, False, dtype)
    for x, y in zip((q, k), got):
        check_rope(y, norm_rope(x, positions, 64, False), rope_tolerance(dtype, None), 64, False)


def test_norm_rope_given_frequencies_and_in_place():
    rng = np.random.default_rng(6)
    q, k = rng.standard_normal((70, 3, 128)).astype(np.float16), rng.standard_normal((70, 2, 128)).astype(np.float16)
    positions = np.arange(70) + 1000
    frequencies = rng.uniform(0, 9, 64)  # (above 2 pi too)
    a = run_norm_rope(q, k, positions, 128, False, np.float16, frequencies=frequencies)
    b = run_norm_rope(q, k, positions, 128, False, np.float16, frequencies=frequencies, in_place=True)
    for x, y, z in zip((q, k), a, b):
        check_rope(y, norm_rope(x, positions, 128, False, frequencies=frequencies), rope_tolerance(np.float16, None), 128, False)
        assert np.array_equal(y, z)


def test_norm_rope_zero_rows_and_neighbours_of_infinities():
    x = np.zeros((20, 2, 64), np.float16)
    x[1, 0, 60], x[2, 1, 61] = np.inf, np.nan  # behind the rotary channels: their neighbours keep their values
    x[1, 0, :8] = 1
    got, _ = run_norm_rope(x, x[:, :1], np.zeros(20, int), 32, False, np.float16)
    assert np.array_equal(got, x, equal_nan=True)
    w = np.ones(64, np.float16)
    got, _ = run_norm_rope(np.zeros((20, 2, 64), np.float16), x[:, :1] * 0, np.arange(20), 64, False, np.float16, (w, w), eps=1e-6)
    assert np.array_equal(got, np.zeros_like(got))


# ---- the cache -----------------------------------------------------------------------------------------------------------------

def batch(rng, counts, lengths, page, extra=2):
    """starts, lengths, page_table (random distinct pages), pages."""
    s = len(counts)
    per = max(1, max((l + page - 1) // page for l in lengths))
    pages = s * per + extra
    table = rng.permutation(pages)[:s * per].reshape(s, per)
    return np.concatenate([[0], np.cumsum(counts)]), np.array(lengths), table, pages


class Device:
    """A cache on the device with its sequences."""

    def __init__(self, kv_heads, head_dim, group, page, pages, starts, lengths, table, tokens=None):
        self.desc = M.kv4_cache_desc(kv_heads, head_dim, group, page, pages, len(lengths), table.shape[1])
        self.host = Cache(kv_heads, head_dim, group, page, pages)
        assert M.kv4_cache_bytes(self.desc) == self.host.bytes.size
        self.cache = torch.full((self.host.bytes.size,), 0xFF, dtype=torch.uint8, device="cuda")  # words of NaN scales: what no test reads
        self.starts, self.lengths, self.table = starts, lengths, table
        self.tokens = tokens or int(starts[-1])
        self.where = [dev(np.asarray(a).astype(np.int32)) for a in (table, lengths, starts)]
        self.most = int(max(1, np.max(np.diff(starts))))

    def fill(self, rng, scale=1.0):
        """Every page of random keys and values, through the host's layout."""
        k, v = [rng.standard_normal((self.host.pages, self.host.kv_heads, self.host.page, self.host.head_dim)) * scale for _ in range(2)]
        self.host.set_all(k, v)
        self.cache.copy_(torch.from_numpy(self.host.bytes))

    def append(self, k, v, dtype, most=None):
        op = M.kv4_append_create(self.desc, M.FLOAT16 if dtype == np.float16 else M.FLOAT32, self.tokens, most or self.most)
        a = [dev(slices(x).astype(dtype)) for x in (k, v)]
        op.bind(a + self.where, [self.cache])
        op.set_shape(1, 1, self.tokens)
        print("append", self.desc.kv_heads, self.desc.head_dim, self.desc.group_size, self.desc.page_size, self.tokens, dtype.__name__, flush=True)
        op.launch(stream())
        torch.cuda.synchronize()

    def read(self, dtype, most=None, fill=5.0):
        op = M.kv4_read_create(self.desc, M.FLOAT16 if dtype == np.float16 else M.FLOAT32, self.tokens, most or self.most)
        c = self.desc.kv_heads * self.desc.head_dim
        out = [torch.full((c // 4, self.tokens, 4), fill, dtype=torch.float16 if dtype == np.float16 else torch.float32, device="cuda") for _ in range(2)]
        op.bind([self.cache] + self.where, out)
        op.set_shape(1, 1, self.tokens)
        print("read", self.desc.kv_heads, self.desc.head_dim, self.desc.group_size, self.desc.page_size, self.tokens, flush=True)
        op.launch(stream())
        torch.cuda.synchronize()
        return [unslices(o.cpu().numpy(), self.desc.head_dim) for o in out]

    def attend(self, q, heads, causal=True, window=0, scale=None, most=None, fill=5.0, launches=1):
        op = M.kv4_attention_create(self.desc, heads, scale=scale, causal=causal, window=window, max_tokens=self.tokens, max_new_tokens=most or self.most)
        src = dev(slices(q).astype(np.float16))
        out = torch.full_like(src, fill)
        op.bind([src, self.cache] + self.where, [out])
        op.set_shape(1, 1, self.tokens)
        print("attend", heads, self.desc.kv_heads, self.desc.head_dim, self.desc.group_size, self.desc.page_size, self.tokens, causal, window, most, flush=True)
        for _ in range(launches):
            op.launch(stream())
        torch.cuda.synchronize()
        self.op = op
        return unslices(out.cpu().numpy(), self.desc.head_dim)


def edges(rng, shape, dtype):
    """Rows of every kind: zeros, one sign only, tiny, huge, ties, infinities and NaN."""
    x = rng.standard_normal(shape)
    flat = x.reshape(-1, shape[-1])
    for i, row in enumerate(flat):
        kind = i % 11
        if kind == 1:
            row[:] = 0
        elif kind == 2:
            row[:] = np.abs(row)
        elif kind == 3:
            row[:] = -np.abs(row)
        elif kind == 4:
            row *= 2.0**-22
        elif kind == 5:
            row *= 30000
        elif kind == 6:  # ties: halves of the step of a span of 15
            row[:] = rng.integers(-14, 15, row.shape) / 2.0
            row[0::32], row[1::32] = 8.0, -7.0
        elif kind == 7:
            row[3], row[5], row[9] = np.inf, -np.inf, np.nan
        elif kind == 8:
            row[:] = 0.1
        elif kind == 9:
            row *= 10.0 ** rng.uniform(-8, 4, row.shape)
    with np.errstate(over="ignore"):
        return x.astype(dtype)


SHAPES = [(1, 64, 32, 16), (2, 64, 64, 32), (1, 128, 32, 64), (3, 128, 64, 16), (1, 128, 128, 128), (1, 256, 32, 16), (2, 256, 64, 64), (1, 256, 128, 1024)]


@pytest.mark.parametrize("kv_heads,head_dim,group,page", SHAPES)
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_append_writes_the_defined_bytes_and_no_others(kv_heads, head_dim, group, page, dtype):
    rng = np.random.default_rng(head_dim + group + page)
    # first tokens of a page, its last ones, a page border inside, single tokens, an empty sequence, more than one page
    counts, lengths = [1, 0, 5, 37, 1, 16, 33], [1, 9, page, page + 20, 17, 16, 70]
    starts, lengths, table, pages = batch(rng, counts, lengths, page)
    tokens = int(starts[-1]) + 3  # (rows behind the last sequence)
    d = Device(kv_heads, head_dim, group, page, pages, starts, lengths, table, tokens)
    k, v = edges(rng, (tokens, kv_heads, head_dim), dtype), edges(rng, (tokens, kv_heads, head_dim), dtype)
    d.host.bytes[:] = 0xFF
    for s, n in enumerate(counts):
        for i in range(n):
            p = lengths[s] - n + i
            if p >= 0:
                d.host.set_token(table[s][p // page], p % page, k[starts[s] + i], v[starts[s] + i])
    d.append(k, v, dtype)
    got = d.cache.cpu().numpy()
    bad = np.nonzero(got != d.host.bytes)[0]
    assert bad.size == 0, (bad.size, bad[:5], got[bad[:5]], d.host.bytes[bad[:5]])


@pytest.mark.parametrize("kv_heads,head_dim,group,page", SHAPES)
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_read_gives_the_values(kv_heads, head_dim, group, page, dtype):
    rng = np.random.default_rng(head_dim + group + page + 1)
    counts, lengths = [1, 0, 5, 37, 1, 16, 33], [1, 9, page, page + 20, 17, 16, 70]
    starts, lengths, table, pages = batch(rng, counts, lengths, page)
    tokens = int(starts[-1]) + 3
    d = Device(kv_heads, head_dim, group, page, pages, starts, lengths, table, tokens)
    d.fill(rng)
    got = d.read(dtype)
    ek, ev = d.host.values()
    for x, y in zip(got, (ek, ev)):
        want = np.full((tokens, kv_heads, head_dim), 5.0)
        for s, n in enumerate(counts):
            for i in range(n):
                p = lengths[s] - n + i
                want[starts[s] + i] = y[table[s][p // page], :, p % page] if p >= 0 else 0
        assert np.array_equal(x.astype(np.float64), want)


def test_append_and_read_of_rows_that_have_no_place():
    """A length shorter than the new rows, one behind the table's room, pages that are not the cache's, a sequence of more rows than the
    launch is sized for: the rows without a place are appended nowhere and read as zeros."""
    rng = np.random.default_rng(3)
    starts, lengths = np.array([0, 6, 10, 30, 230]), np.array([4, 40, 20, 200])
    table = np.array([[0, 1], [2, 3], [4, 99], [5, 6]])
    table = np.concatenate([table, np.full((4, 12), -1)], 1)
    table[3, :14] = 7 + np.arange(14)
    table[1, 2:] = 6  # (positions from 32 on: one page for many positions, written by no row of this test)
    d = Device(2, 64, 32, 16, 21, starts, lengths, table)
    d.cache.zero_()
    k, v = [rng.standard_normal((230, 2, 64)).astype(np.float16) for _ in range(2)]
    starts[1] = 6
    # sequence 1: rows at 36 .. 39 on page 6; sequence 2: positions 0 .. 19, 16 .. 19 on page 99; sequence 3: 0 .. 199
    d.append(k, v, np.float16, most=1)
    got = d.read(np.float16, most=1)
    for x, y in zip(got, (k, v)):
        want = kept(y.astype(np.float64), 32)
        want[0:2] = 0  # positions -2, -1
        want[26:30] = 0
        assert np.array_equal(x.astype(np.float64), want)


# ---- attention -------------------------------------------------------------------------------------------------------------------

# The kernels' scores are fp32 sums of exact products (halfs by integers); of a score of magnitude S = scale * sum |q||k| they are off by
# at most about 2^-16 S (sums of up to 256 terms, codes on a base of 1024), which scales a probability by as much.  Probabilities are
# rounded to halfs (2^-11), their products summed in fp32, the result rounded to a half (2^-11).  An output is an average of the values
# seen, so all of it is relative to the largest |v| seen: 2^-11 + 2 * 2^-16 S for the weights (numerator and sum), 2^-11 of the output.
def check_attention(got, exact, largest, score):
    tol = (2.0**-11 + 2 * 2.0**-16 * score + 2.0**-18) * largest + 2.0**-11 * np.abs(exact) + 2.0**-24
    err = np.abs(got.astype(np.float64) - exact)
    bad = ~(err <= tol)
    assert not bad.any(), (np.argwhere(bad)[:3], got[bad][:3], exact[bad][:3], (err / tol).max())


def attention_case(kv_heads, share, head_dim, group, page, counts, lengths, causal=True, window=0, seed=0, behind=0, q_scale=1.0, most=None):
    rng = np.random.default_rng(seed)
    starts, lengths, table, pages = batch(rng, counts, lengths, page)
    tokens = int(starts[-1]) + behind
    d = Device(kv_heads, head_dim, group, page, pages, starts, lengths, table, tokens)
    d.fill(rng)
    # what lies behind a sequence's last token is never looked at: NaN words there
    d.host.spoil(table, lengths)
    d.cache.copy_(torch.from_numpy(d.host.bytes))
    q = (rng.standard_normal((tokens, kv_heads * share, head_dim)) * q_scale).astype(np.float16)
    got = d.attend(q, kv_heads * share, causal, window, most=most)
    exact, largest, score = attention(q, d.host, table, lengths, starts, head_dim**-0.5, causal, window, fill=5.0)
    check_attention(got, exact, largest, score)
    return d


@pytest.mark.parametrize("kv_heads,head_dim,group,page", SHAPES)
@pytest.mark.parametrize("share", [1, 4, 8])
def test_attention_one_token(kv_heads, head_dim, group, page, share):
    attention_case(kv_heads, share, head_dim, group, page, [1] * 9, [1, 2, 15, 16, 17, 63, 64, 65, 300], seed=share)


@pytest.mark.parametrize("kv_heads,head_dim,group,page", SHAPES)
@pytest.mark.parametrize("window", [0, 1, 40])
def test_attention_few_tokens(kv_heads, head_dim, group, page, window):
    attention_case(kv_heads, 3, head_dim, group, page, [4, 1, 0, 2, 3, 6], [4, 1, 0, 2, 100, 333], window=window, behind=2, seed=window)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("share", [1, 2, 7, 16, 20])
def test_attention_row_tiles(causal, share):
    attention_case(2, share, 64, 32, 16, [1, 5, 13, 21], [200, 5, 77, 129], causal=causal, window=0 if causal else 50, seed=share)


@pytest.mark.parametrize("kv_heads,head_dim,group,page", SHAPES)
@pytest.mark.parametrize("share,causal,window", [(1, True, 0), (4, True, 0), (3, True, 40), (2, False, 0), (2, False, 70)])
def test_attention_many_tokens(kv_heads, head_dim, group, page, share, causal, window):
    d = attention_case(kv_heads, share, head_dim, group, page, [70, 1, 0, 130, 33, 16], [70, 90, 3, 200, 95, 400], causal, window, behind=2, seed=share)
    assert d.op.kernel_name == "kv4_attention_many_kernel" and d.op.kernel_variant == "many"


@pytest.mark.parametrize("head_dim,group", [(64, 32), (128, 64), (256, 128)])
@pytest.mark.parametrize("parts", [-1, 3])
def test_attention_of_prompts_and_single_tokens_together(head_dim, group, parts):
    counts, lengths = [1, 70, 16, 0, 2, 33, 1, 20, 1, 1], [90, 90, 16, 3, 333, 200, 1, 400, 64, 77]
    with M.tuning(kv4_parts=parts):
        d = attention_case(8, 2, head_dim, group, 32, counts, lengths, behind=1)
    assert d.op.kernel_name == "kv4_attention_many_kernel" and d.op.kernel_variant == "many, few"


@pytest.mark.parametrize("kv_heads,head_dim,group,page", SHAPES)
@pytest.mark.parametrize("many", [0, 1])
@pytest.mark.parametrize("parts", [1, 2, 3, 7])
def test_attention_in_parts(kv_heads, head_dim, group, page, many, parts):
    """Both kernels with the keys in any number of parts, some of which see nothing."""
    with M.tuning(kv4_many=many, kv4_parts=parts):
        d = attention_case(kv_heads, 3, head_dim, group, page, [1, 40, 5, 90], [700, 333, 5, 1024], window=500 if parts == 3 else 0, seed=parts)
        assert d.op.kernel_variant == ("many" if many else "few") and d.op.kernel_tiles[2] == parts
        d = attention_case(kv_heads, 2, head_dim, group, page, [300], [900], seed=parts)
        assert d.op.kernel_variant == ("many" if many else "few")


def test_attention_of_many_heads_for_a_key_head():
    """More heads on a key head than rows that the kernel for few takes: every row of a ragged batch is the other kernel's."""
    d = attention_case(8, 56, 64, 32, 16, [1, 3, 0, 2, 1, 1, 1, 1], [90, 40, 3, 333, 200, 1, 17, 64])
    assert d.op.kernel_variant == "many"
    with M.tuning(kv4_parts=3):
        attention_case(8, 56, 64, 32, 16, [1, 3, 0, 2, 1, 1, 1, 1], [90, 40, 3, 333, 200, 1, 17, 64])


def test_attention_parts_of_one_kernel_beside_whole_rows_of_the_other():
    """Long tables: sequences of few rows in parts, prompts not, and the other way round."""
    for parts in (-1, 2):
        with M.tuning(kv4_parts=parts):
            d = attention_case(1, 4, 128, 64, 64, [1, 80, 2, 1], [5000, 200, 4400, 70], seed=parts + 1)
        assert d.op.kernel_variant == "many, few"


@pytest.mark.parametrize("parts", [-1, 5, 256])
def test_attention_shares_over_many_sequences(parts):
    """More sequences than lanes, shares that begin and end inside sequences, and launches again with other lengths."""
    rng = np.random.default_rng(21)
    counts = list(rng.integers(0, 3, 150))
    lengths = [int(c + rng.integers(0, 500)) if c else 0 for c in counts]
    with M.tuning(kv4_many=0, kv4_parts=parts):
        d = attention_case(1, 9, 64, 32, 16, counts, lengths, seed=5)
        q = rng.standard_normal((d.tokens, 9, 64)).astype(np.float16)
        src, out = dev(slices(q)), torch.zeros((9 * 16, d.tokens, 4), dtype=torch.float16, device="cuda")
        op = M.kv4_attention_create(d.desc, 9, max_tokens=d.tokens, max_new_tokens=2)
        op.bind([src, d.cache] + d.where, [out])
        op.set_shape(1, 1, d.tokens)
        for turn in range(3):
            now = [l if turn == 0 else max(int(c), l // (turn + 1)) for c, l in zip(counts, lengths)]
            d.where[1].copy_(torch.tensor(now, dtype=torch.int32))
            op.launch(stream())
            torch.cuda.synchronize()
            exact, largest, score = attention(q, d.host, d.table, np.array(now), d.starts, 64**-0.5, True, 0)
            check_attention(unslices(out.cpu().numpy(), 64), exact, largest, score)


@pytest.mark.parametrize("head_dim,group,page", [(64, 32, 16), (64, 64, 64), (128, 32, 16), (128, 128, 32), (256, 64, 16), (256, 128, 64)])
@pytest.mark.parametrize("sequences,kv_heads,parts", [(16, 16, 1), (8, 8, 4)])
def test_attention_by_work_groups_of_whole_compute_units(head_dim, group, page, sequences, kv_heads, parts):
    """As many tiles as compute units, or a share of them: all the waves of a unit take one tile's keys."""
    waves = {64: 16, 128: 12, 256: 8}[head_dim]
    most = parts * 32 * waves
    lengths = [1 + (most + 40) * i // (sequences - 1) for i in range(sequences)]
    counts = [min(l, 1 + i % 2) for i, l in enumerate(lengths)]
    d = attention_case(kv_heads, 3, head_dim, group, page, counts, lengths, window=most // 2 if page == 32 else 0, behind=1, seed=head_dim + parts)
    # (in a window of half the positions 4 parts have not a step for each of their waves: work-groups of 4 waves then)
    form = (16, 4, 7) if page == 32 and parts == 4 else (16, waves, parts)
    assert d.op.kernel_variant == "few" and d.op.kernel_tiles == form


def test_attention_of_more_than_a_thousand_sequences():
    attention_case(2, 2, 64, 64, 16, [1] * 1100, [1 + i % 40 for i in range(1100)], seed=6)


def test_attention_of_starts_that_decrease_stays_in_bounds():
    """Not a batch that means anything: whatever is written, it is written into the output, and what is in front of and behind it stays."""
    starts, lengths = np.array([0, 60, 0, 60, 5, 60, -7, 90]), np.array([60, 0, 60, 0, 60, 0, 60])
    d = Device(2, 64, 32, 16, 30, starts, lengths, np.arange(28).reshape(7, 4), tokens=60)
    d.fill(np.random.default_rng(1))
    size, room = 4 * 16 * 60 * 4, 4096
    around = torch.full((size + 2 * room,), 7.0, dtype=torch.float16, device="cuda")
    src = torch.zeros((64, 60, 4), dtype=torch.float16, device="cuda")
    for many in (0, 1):
        for parts in (1, 5):
            with M.tuning(kv4_many=many, kv4_parts=parts):
                op = M.kv4_attention_create(d.desc, 4, max_tokens=60, max_new_tokens=60)
            op.bind([src, d.cache] + d.where, [around[room:room + size]])
            op.set_shape(1, 1, 60)
            op.launch(stream())
            torch.cuda.synchronize()
            assert (around[:room] == 7).all() and (around[room + size:] == 7).all()


def test_attention_of_more_rows_than_it_is_sized_for():
    attention_case(1, 4, 64, 32, 16, [90, 200], [90, 230], most=1)
    attention_case(1, 4, 64, 32, 16, [90, 700], [90, 730], most=20)
    attention_case(64, 1, 64, 32, 16, [90, 1, 300], [90, 9, 330], most=33)


def test_attention_of_pages_that_are_not_there():
    """Pages in the middle that are not the cache's, for every kernel."""
    rng = np.random.default_rng(12)
    starts, lengths = np.array([0, 3, 80]), np.array([200, 160])
    for page, head_dim in ((16, 128), (64, 64), (32, 256)):
        per = -(-200 // page)
        table = np.arange(2 * per).reshape(2, per)
        table[0, 1], table[1, 0], table[1, 2] = -5, 10**6, 2 * per + 1
        d = Device(2, head_dim, 32, page, 2 * per + 1, starts, lengths, table)
        d.fill(rng)
        d.host.spoil(table, lengths)
        d.cache.copy_(torch.from_numpy(d.host.bytes))
        q = rng.standard_normal((80, 4, head_dim)).astype(np.float16)
        for many in (0, 1):
            for window in (0, 30):
                with M.tuning(kv4_many=many):
                    got = d.attend(q, 4, window=window)
                exact, largest, score = attention(q, d.host, table, lengths, starts, head_dim**-0.5, True, window, fill=5.0)
                check_attention(got, exact, largest, score)


def test_attention_of_nothing():
    """No positions at all, a length shorter than the new rows, pages that are not the cache's."""
    rng = np.random.default_rng(8)
    starts, lengths = np.array([0, 2, 6, 9]), np.array([0, 2, 40])
    table = np.array([[0, 1, 2], [3, 4, 5], [6, -1, 70]])
    d = Device(1, 128, 64, 16, 8, starts, lengths, table)
    d.fill(rng)
    q = rng.standard_normal((9, 4, 128)).astype(np.float16)
    got = d.attend(q, 4)
    assert not got[:4].any()  # (sequence 1's first two rows have positions -2 and -1)
    exact, largest, score = attention(q, d.host, table, lengths, starts, 128**-0.5, True, 0, fill=5.0)
    check_attention(got, exact, largest, score)


def test_attention_sharp_and_far_apart_scores():
    """Scores of hundreds: one position takes all; and a long cache in which every position counts the same."""
    for q_scale in (60.0, 0.0):
        attention_case(1, 8, 128, 64, 64, [1, 1], [1000, 4097], q_scale=q_scale)
        attention_case(1, 2, 128, 64, 64, [65, 100], [1000, 100], q_scale=q_scale)


@pytest.mark.parametrize("head_dim,group,page", [(64, 32, 16), (128, 64, 32), (256, 128, 64)])
@pytest.mark.parametrize("many,parts", [(0, 1), (0, 3), (1, 1), (1, 2)])
@pytest.mark.parametrize("size", [30.0, 1000.0, 60000.0])
def test_attention_of_the_largest_scores(head_dim, group, page, many, parts, size):
    """Two equal keys in far apart steps whose scores, up to 1e10, leave all others nothing: the output is the mean of their values, whatever
    ulps of such scores are."""
    rng = np.random.default_rng(head_dim + many + parts)
    counts, lengths = [70, 2, 1], [700, 600, 555]
    starts, lengths, table, pages = batch(rng, counts, lengths, page)
    d = Device(2, head_dim, group, page, pages, starts, lengths, table)
    d.fill(rng)
    u = rng.choice([-1.0, 1.0], head_dim)
    v = rng.standard_normal((2, 2, head_dim)) * 4
    for s in range(3):
        for i, p in enumerate((300, 17)):
            d.host.set_token(table[s][p // page], p % page, np.stack([size * u] * 2), v[i])
    d.cache.copy_(torch.from_numpy(d.host.bytes))
    q = (size * u * np.ones((d.tokens, 6, 1))).astype(np.float16)
    with M.tuning(kv4_many=many, kv4_parts=parts):
        got = d.attend(q, 6)
    exact, largest, _ = attention(q, d.host, table, lengths, starts, head_dim**-0.5, True, 0)
    mean = np.repeat(kept(v, group).mean(0), 3, 0)  # [6][head_dim]
    assert np.abs(exact - mean).max() < 1e-9
    # two equal probabilities (rounded alike) and their sum, fp32 sums, one rounding to half
    assert (np.abs(got - exact) <= 2.0**-11 * np.abs(exact) + 2.0**-20 * largest).all()


@pytest.mark.parametrize("many", [0, 1])
def test_attention_of_many_small_probabilities(many):
    """One key far above 66000 others, whose probabilities are subnormal halfs and yet add up to a hundredth of its own: they count in the outputs
    and in their sum alike."""
    rng = np.random.default_rng(31)
    starts, lengths, table, pages = batch(rng, [50], [66000], 64)
    d = Device(1, 64, 32, 64, pages, starts, lengths, table)
    v = rng.uniform(-1, 1, 64) + np.where(np.arange(64) % 2, 2.0, -2.0)
    shape = (pages, 1, 64, 64)
    d.host.set_all(np.zeros(shape), np.broadcast_to(v, shape))
    one = np.ones((1, 64))
    d.host.set_token(table[0][500], 0, one, -v[None])
    d.cache.copy_(torch.from_numpy(d.host.bytes))
    q = np.full((50, 2, 64), 22.4 / math.log2(math.e) / 64 * 8).astype(np.float16)  # (the score of the one key is 22.4 in powers of two)
    with M.tuning(kv4_many=many):
        got = d.attend(q, 2)
    exact, largest, score = attention(q, d.host, table, lengths, starts, 64**-0.5, True, 0)
    assert np.abs(exact + kept(v[None], 32)).max() > 0.02  # (without the others it would be -v)
    check_attention(got, exact, largest, score)


@pytest.mark.parametrize("many,parts", [(0, 1), (0, 3), (0, 12), (1, 1), (1, 2), (-1, -1)])
def test_rows_in_front_of_the_first_sequence_stay(many, parts):
    rng = np.random.default_rng(17)
    starts, lengths, table, pages = batch(rng, [2, 0, 60, 1], [900, 5, 1700, 1], 32)
    starts = starts + 3
    tokens = int(starts[-1]) + 2
    d = Device(2, 64, 32, 32, pages, starts, lengths, table, tokens)
    d.fill(rng)
    q = rng.standard_normal((tokens, 6, 64)).astype(np.float16)
    with M.tuning(kv4_many=many, kv4_parts=parts):
        got = d.attend(q, 6)
    exact, largest, score = attention(q, d.host, table, lengths, starts, 64**-0.5, True, 0, fill=5.0)
    check_attention(got, exact, largest, score)
    assert (got[:3] == 5.0).all() and (got[-2:] == 5.0).all()
    for most in (1, 60):
        for x in d.read(np.float32, most=most):
            assert (x[:3] == 5.0).all() and (x[-2:] == 5.0).all() and (x[3:-2] != 5.0).any(-1).all()


def test_attention_of_rows_that_are_not_finite():
    rng = np.random.default_rng(9)
    starts, lengths, table, pages = batch(rng, [3, 1], [90, 70], 16)
    d = Device(1, 64, 32, 16, pages, starts, lengths, table)
    d.fill(rng)
    q = rng.standard_normal((4, 2, 64)).astype(np.float16)
    q[1, 0, 5] = np.nan
    got = d.attend(q, 2)
    assert np.isnan(got[1, 0]).all()
    q2 = q.copy()
    q2[1, 0] = 0
    same = np.ones((4, 2), bool)
    same[1, 0] = False
    for many in (0, 1):
        with M.tuning(kv4_many=many):
            got, rest = d.attend(q, 2), d.attend(q2, 2)
        assert np.isnan(got[1, 0]).all() and np.array_equal(got[same], rest[same])


# ---- launches ------------------------------------------------------------------------------------------------------------------------

def decode_step(rng, kv_heads=2, share=4, head_dim=128, group=32, page=16, counts=(1, 1, 2, 1), lengths=(40, 300, 65, 1)):
    """The ops of one layer's step over one batch, bound one behind the other, and the host's copies of what they read."""
    starts, lengths, table, pages = batch(rng, list(counts), list(lengths), page, extra=5)
    d = Device(kv_heads, head_dim, group, page, pages, starts, lengths, table)
    d.fill(rng)
    heads, t = kv_heads * share, d.tokens
    host = [rng.standard_normal((t, h, head_dim)).astype(np.float16) for h in (heads, kv_heads, kv_heads)]
    q, k, v = [dev(slices(x)) for x in host]
    positions = np.concatenate([np.arange(l - c, l) for c, l in zip(counts, lengths)])
    weights = [rng.standard_normal(head_dim).astype(np.float16) for _ in range(2)]
    most = max(counts)
    rope = M.qk_norm_rope_create(M.FLOAT16, heads, kv_heads, head_dim, norm=True, weight_offset=1.0, max_tokens=t)
    d.keep = [dev(positions.astype(np.int32))] + [dev(w) for w in weights]  # (an op holds raw pointers)
    rope.bind([q, k] + d.keep, [q, k])
    append = M.kv4_append_create(d.desc, M.FLOAT16, t, most)
    append.bind([k, v] + d.where, [d.cache])
    out = torch.zeros_like(q)
    attend = M.kv4_attention_create(d.desc, heads, max_tokens=t, max_new_tokens=most)
    attend.bind([q, d.cache] + d.where, [out])
    for op in (rope, append, attend):
        op.set_shape(1, 1, t)
    return d, host, positions, weights, (q, k, v), out, (rope, append, attend), table, starts


def check_step(d, host, positions, weights, out, table, starts):
    """The step's output against 64 bits throughout, but for what the step itself rounds to halfs on the way."""
    head_dim = d.desc.head_dim
    q, k = [norm_rope(x, positions, head_dim, False, weight=w, offset=1.0).astype(np.float16) for x, w in zip(host[:2], weights)]
    for s in range(len(d.lengths)):
        for i in range(starts[s], starts[s + 1]):
            p = positions[i]
            d.host.set_token(table[s][p // d.desc.page_size], p % d.desc.page_size, k[i], host[2][i])
    exact, largest, score = attention(q, d.host, table, d.lengths, starts, head_dim**-0.5, True, 0)
    # The step's q and k may be a half's step off these where the rounding falls the other way, and a key's code with it: a scale (of at most
    # 2 max|k| / 15) of one key channel and 2^-10 of q, of which a score of `score` is at most (1/4 + 2^-10) off, in all but a few rows much
    # less; an output moves by at most twice that of the values' range.
    tol = 2 * (0.25 + 2.0**-10) * score * largest + 2.0**-10 * largest
    err = np.abs(unslices(out.cpu().numpy(), head_dim).astype(np.float64) - exact)
    rms = np.sqrt((err**2).mean()) / np.sqrt((exact**2).mean())
    assert (err <= tol).all() and rms < 2.0**-7, rms


def test_a_step_captured_and_replayed():
    """The step in a graph: replays with other inputs in the same buffers, eager work in between, every one against the eager launches."""
    rng = np.random.default_rng(31)
    d, host, positions, weights, (q, k, v), out, ops, table, starts = decode_step(rng)
    first = [x.clone() for x in (q, k, v)]
    cache = d.cache.clone()

    def reset(scale):
        for x, y in zip((q, k, v), first):
            x.copy_(y * scale)
        d.cache.copy_(cache)

    def run():
        for op in ops:
            op.launch(stream())

    eager = []
    for scale in (1.0, 0.5, 2.0):
        reset(scale)
        run()
        torch.cuda.synchronize()
        eager.append((out.clone(), d.cache.clone()))
    check_step(d, [x.astype(np.float64) * 2 for x in host], positions, weights, out, table, starts)
    reset(1.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        run()
    for turn in range(6):
        reset((1.0, 0.5, 2.0)[turn % 3])
        out.fill_(3.0)
        graph.replay()
        if turn % 2:
            torch.cuda.synchronize()
            (out * 2).sum().item()
        torch.cuda.synchronize()
        assert torch.equal(out, eager[turn % 3][0]) and torch.equal(d.cache, eager[turn % 3][1])


def test_a_step_on_another_stream():
    rng = np.random.default_rng(32)
    d, host, positions, weights, tensors, out, ops, table, starts = decode_step(rng)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for op in ops:
            op.launch(side.cuda_stream)
    side.synchronize()
    check_step(d, host, positions, weights, out, table, starts)


def test_two_ops_at_the_same_time():
    """Two batches on two streams, each with ops (and workspaces) of its own."""
    steps = [decode_step(np.random.default_rng(40 + i), page=64, counts=(1, 1), lengths=(2000, 777)) for i in range(2)]
    alone = []
    for s in steps:
        keep = [x.clone() for x in s[4]] + [s[0].cache.clone()]
        for op in s[6]:
            op.launch(stream())
        torch.cuda.synchronize()
        alone.append(s[5].clone())
        for x, y in zip(list(s[4]) + [s[0].cache], keep):
            x.copy_(y)
        s[5].zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in steps]
    for k in range(3):
        for s, st in zip(steps, streams):
            s[6][k].launch(st.cuda_stream)
    torch.cuda.synchronize()
    for s, want in zip(steps, alone):
        assert torch.equal(s[5], want)


@pytest.mark.parametrize("many", [0, 1])
def test_attention_is_the_same_every_time(many):
    rng = np.random.default_rng(33)
    starts, lengths, table, pages = batch(rng, [3, 40, 1], [2000, 300, 1500], 16)
    d = Device(2, 64, 32, 16, pages, starts, lengths, table)
    d.fill(rng)
    q = rng.standard_normal((44, 6, 64)).astype(np.float16)
    with M.tuning(kv4_many=many):
        a = d.attend(q, 6)
        assert all(np.array_equal(d.attend(q, 6, launches=n), a) for n in (1, 2, 3))


def test_a_cache_of_more_than_four_gigabytes():
    """Pages whose bytes lie behind 2^32: written, read and attended there."""
    kv_heads, head_dim, group, page = 8, 256, 32, 1024
    per_page = kv_heads * page * (head_dim + 4 * head_dim // group)
    pages = (9 << 30) // per_page
    cache = M.kv4_cache_desc(kv_heads, head_dim, group, page, pages, 2, 1)
    assert M.kv4_cache_bytes(cache) > 8 << 30
    rng = np.random.default_rng(34)
    big = torch.zeros(M.kv4_cache_bytes(cache), dtype=torch.uint8, device="cuda")
    starts, lengths, table = np.array([0, 20, 30]), np.array([20, 10]), np.array([[pages - 1], [pages // 2 + 1]])
    where = [dev(np.asarray(a).astype(np.int32)) for a in (table, lengths, starts)]
    k, v = [rng.standard_normal((30, kv_heads, head_dim)).astype(np.float16) for _ in range(2)]
    q = rng.standard_normal((30, kv_heads * 2, head_dim)).astype(np.float16)
    src = [dev(slices(x)) for x in (k, v, q)]
    append = M.kv4_append_create(cache, M.FLOAT16, 30, 20)
    append.bind(src[:2] + where, [big])
    back = [torch.zeros_like(x) for x in src[:2]]
    read = M.kv4_read_create(cache, M.FLOAT16, 30, 20)
    read.bind([big] + where, back)
    for op in (append, read):
        op.set_shape(1, 1, 30)
        op.launch(stream())
    torch.cuda.synchronize()
    for x, y in zip(back, (k, v)):
        assert np.array_equal(unslices(x.cpu().numpy(), head_dim).astype(np.float64), kept(y.astype(np.float64), group))
    small = Cache(kv_heads, head_dim, group, 32, 2)
    for s in range(2):
        for i in range(lengths[s]):
            small.set_token(s, i, k[starts[s] + i], v[starts[s] + i])
    exact, largest, score = attention(q, small, np.array([[0], [1]]), lengths, starts, head_dim**-0.5, True, 0)
    for many in (0, 1):
        with M.tuning(kv4_many=many):
            op = M.kv4_attention_create(cache, kv_heads * 2, max_tokens=30, max_new_tokens=20)
        out = torch.zeros_like(src[2])
        op.bind([src[2], big] + where, [out])
        op.set_shape(1, 1, 30)
        op.launch(stream())
        torch.cuda.synchronize()
        check_attention(unslices(out.cpu().numpy(), head_dim), exact, largest, score)
    op = None
    del big
    torch.cuda.empty_cache()


# ---- together --------------------------------------------------------------------------------------------------------------------

def test_a_sequence_token_by_token_is_the_prompt_at_once():
    """Appending and attending one token at a time gives what the prompt gives in one launch each, and both what the arithmetic gives."""
    rng = np.random.default_rng(11)
    heads, kv_heads, head_dim, group, page, n = 4, 2, 64, 32, 16, 45
    q, k, v = [rng.standard_normal((n, h, head_dim)).astype(np.float16) for h in (heads, kv_heads, kv_heads)]
    table = np.array([[3, 0, 2]])
    whole = Device(kv_heads, head_dim, group, page, 4, np.array([0, n]), np.array([n]), table)
    whole.append(k, v, np.float16)
    at_once = whole.attend(q, heads)
    for i in range(n):
        d = Device(kv_heads, head_dim, group, page, 4, np.array([0, 1]), np.array([i + 1]), table)
        if i:
            d.cache.copy_(cache)
        d.append(k[i:i + 1], v[i:i + 1], np.float16)
        cache = d.cache
        one = d.attend(q[i:i + 1], heads)
        whole.host.set_token(table[0][i // page], i % page, k[i], v[i])
        exact, largest, score = attention(q[i:i + 1], whole.host, table, np.array([i + 1]), np.array([0, 1]), head_dim**-0.5, True, 0)
        check_attention(one, exact, largest, score)
        check_attention(at_once[i:i + 1], exact, largest, score)
    held = np.nonzero(cache.cpu().numpy() != whole.cache.cpu().numpy())[0]
    assert held.size == 0
