"""The ops over the cache of 4-bit codes at the edges of what they are given."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

import mldhip as M
from kv4math import attention
from test_gpu_kv4 import SHAPES, Device, batch, check_attention, stream

torch = pytest.importorskip("torch")


def guarded(size, dtype, room=4096):
    """(a buffer of `size` elements, what is in front of it and behind it, all sevens)"""
    whole = torch.full((size + 2 * room,), 7, dtype=dtype, device="cuda")
    return whole[room:room + size], (whole[:room], whole[room + size:])


@pytest.mark.parametrize("head_dim", [64, 128, 256])
def test_starts_of_any_values_stay_in_bounds(head_dim):
    """Not a batch that means anything: whatever is written, what is in front of the buffers and behind them stays."""
    low, high = -2**31, 2**31 - 1
    starts = np.array([0, 60, low, 60, high, 5, low, 7, low + 5, high, 60, -7, 90])
    lengths = np.array([60, 0, high, 60, low, 60, 30, 60, high, 1, 60, 60])
    s, tokens = len(lengths), 60
    d = Device(2, head_dim, 32, 16, 4 * s + 2, starts, lengths, np.arange(4 * s).reshape(s, 4), tokens=tokens)
    d.fill(np.random.default_rng(1))
    cache, around_cache = guarded(d.cache.numel(), torch.uint8)
    cache.copy_(d.cache)
    src = [torch.zeros((h * head_dim // 4, tokens, 4), dtype=torch.float16, device="cuda") for h in (4, 2, 2)]

    def launched(op, srcs, dsts, around):
        op.bind(srcs + d.where, dsts)
        op.set_shape(1, 1, tokens)
        op.launch(stream())
        torch.cuda.synchronize()
        for edges in around:
            assert all((x == 7).all() for x in edges)

    for most in (1, 60):
        print("append", head_dim, most, flush=True)
        launched(M.kv4_append_create(d.desc, M.FLOAT16, tokens, most), src[1:], [cache], [around_cache])
        (k, around_k), (v, around_v) = [guarded(src[1].numel(), torch.float16) for _ in range(2)]
        print("read", head_dim, most, flush=True)
        launched(M.kv4_read_create(d.desc, M.FLOAT16, tokens, most), [cache], [k, v], [around_k, around_v])
    for many in (0, 1, -1):
        for parts in (1, 5):
            with M.tuning(kv4_many=many, kv4_parts=parts):
                op = M.kv4_attention_create(d.desc, 4, max_tokens=tokens, max_new_tokens=60)
            out, around = guarded(src[0].numel(), torch.float16)
            print("attend", head_dim, many, parts, flush=True)
            launched(op, [src[0], cache], [out], [around])


@pytest.mark.parametrize("kv_heads,head_dim,group,page", SHAPES)
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_read_of_many_tiles_for_a_wave(kv_heads, head_dim, group, page, dtype):
    """Launches sized for a few rows of a sequence: each wave reads many tiles, one after the other, through the same LDS."""
    rng = np.random.default_rng(head_dim + group + page + 2)
    counts, lengths = [333, 1, 150], [333, 40, 170]
    starts, lengths, table, pages = batch(rng, counts, lengths, page)
    d = Device(kv_heads, head_dim, group, page, pages, starts, lengths, table)
    d.fill(rng)
    values = d.host.values()
    for got, y in zip(d.read(dtype, most=9), values):
        for s, n in enumerate(counts):
            at = np.arange(lengths[s] - n, lengths[s])
            assert np.array_equal(got[starts[s]:starts[s + 1]].astype(np.float64), y[table[s][at // page], :, at % page])


# ---- groups of keys with a channel far from zero ------------------------------------------------------------------------------------

@pytest.mark.parametrize("kv_heads,head_dim,group,page", SHAPES)
@pytest.mark.parametrize("many,parts", [(0, 1), (0, 2), (1, 1)])
def test_attention_scores_are_sums_of_the_few_products_that_there_are(kv_heads, head_dim, group, page, many, parts):
    """Every group of a key has one channel at 100, which the queries do not look at, two a step of its scale from zero and all others at zero,
    while the queries' mean is far from zero: the score is the sum of two products for each group, and nothing else may be seen of the rest."""
    rng = np.random.default_rng(head_dim + group)
    counts, lengths = [3, 1, 40], [5, 2, 40]
    starts, lengths, table, pages = batch(rng, counts, lengths, page)
    d = Device(kv_heads, head_dim, group, page, pages, starts, lengths, table)
    groups = head_dim // group
    shape = (pages, kv_heads, page)
    k = np.zeros((*shape, groups, group))
    k[..., 0] = 100.0
    step = 6.6875  # (the least half of 7 significant bits whose 15-fold is 100)
    for _ in range(2):
        at = rng.integers(1, group, (*shape, groups))
        np.put_along_axis(k, at[..., None], rng.choice([0.0, step], (*shape, groups))[..., None], -1)
    v = rng.standard_normal((*shape, head_dim))
    d.host.set_all(k.reshape(*shape, head_dim), v)
    d.cache.copy_(torch.from_numpy(d.host.bytes))
    q = (8 + 8 * rng.standard_normal((d.tokens, kv_heads * 3, groups, group))).astype(np.float16)
    q[..., 0] = 0
    q = q.reshape(d.tokens, kv_heads * 3, head_dim)
    with M.tuning(kv4_many=many, kv4_parts=parts):
        got = d.attend(q, kv_heads * 3, scale=1 / 128)
    exact, largest, score = attention(q, d.host, table, lengths, starts, 1 / 128, True, 0)
    # 2 * groups products at most that are not zero, an fp32 sum of them (2^-23 each, whichever way it rounds); the exponent's own error and the
    # multiply-add in front of it, 2^-20 for scores of up to 8 or so; probabilities and outputs rounded to halfs, 2^-11 each, of what is averaged
    assert score.max() < 32
    tol = (2.0**-11 + 2 * (2 * groups * 2.0**-23 * score + 2.0**-20)) * largest + 2.0**-11 * np.abs(exact) + 2.0**-24
    err = np.abs(got.astype(np.float64) - exact)
    assert (err <= tol).all(), (err / tol).max()


@pytest.mark.parametrize("head_dim,group", [(64, 64), (128, 128), (128, 32), (256, 128)])
@pytest.mark.parametrize("away,mean", [(50.0, 5.0), (100.0, 3.0)])
def test_attention_of_keys_with_a_channel_far_away(head_dim, group, away, mean):
    """A key channel of 50 and 100, where queries are small, and queries with a mean elsewhere: outputs are as near the exact ones as the roundings of
    the probabilities and of the outputs let them be, in both kernels."""
    rng = np.random.default_rng(head_dim + group + int(away))
    counts, lengths, page, kv_heads, share = [2, 1], [500, 301], 64, 2, 4
    starts, lengths, table, pages = batch(rng, counts, lengths, page)
    d = Device(kv_heads, head_dim, group, page, pages, starts, lengths, table)
    shape = (pages, kv_heads, page, head_dim)
    k = rng.standard_normal(shape)
    k[..., 7] += away
    d.host.set_all(k, rng.standard_normal(shape))
    d.cache.copy_(torch.from_numpy(d.host.bytes))
    q = mean + mean * rng.standard_normal((d.tokens, kv_heads * share, head_dim))
    q[..., 7] = 0.05 * rng.standard_normal(q.shape[:-1])
    q = q.astype(np.float16)
    exact, _, _ = attention(q, d.host, table, lengths, starts, head_dim**-0.5, True, 0)
    for many in (0, 1):
        with M.tuning(kv4_many=many):
            got = d.attend(q, kv_heads * share)
        off = np.sqrt(((got - exact)**2).mean() / (exact**2).mean())
        # a half rounds by 2^-11 at most, 2^-11 / sqrt(3) in the mean of squares, the probabilities and the outputs once each: 4.0e-4
        print("off", many, off, flush=True)
        assert off <= 2.0**-11, (many, off)


# ---- rows of queries that are not finite ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("head_dim,group,page", [(64, 32, 16), (128, 64, 32), (256, 128, 64)])
@pytest.mark.parametrize("many,parts", [(0, 1), (0, 3), (0, 12), (1, 1), (1, 2), (1, 12)])
@pytest.mark.parametrize("odd", [np.nan, np.inf, -np.inf])
def test_attention_of_odd_rows_is_nan_or_nothing(head_dim, group, page, many, parts, odd):
    """An infinity or a NaN in a row of queries: NaN where the row sees a position (also if all its scores are -inf), 0 where it sees none, and no
    difference in any other row."""
    rng = np.random.default_rng(head_dim + parts)
    # sequence 0: the first 40 rows have positions below 0; 1: no page that is the cache's; 2: the first two pages are not, the window leaves some
    # rows only these; 3: two rows of a sequence of nothing; 4: ordinary
    counts, lengths, window = [60, 50, 40, 2, 33], [20, 50, 2 * page + 8, 0, 1500], 24
    starts, lengths, table, pages = batch(rng, counts, lengths, page)
    table[1, :], table[2, :2] = -1, pages + 5
    d = Device(2, head_dim, group, page, pages, starts, lengths, table)
    d.host.set_all(*(np.abs(rng.standard_normal((pages, 2, page, head_dim))) + 1 for _ in range(2)))  # (keys above 0: scores of one sign)
    d.cache.copy_(torch.from_numpy(d.host.bytes))
    q = rng.standard_normal((d.tokens, 6, head_dim)).astype(np.float16)
    odd_rows = rng.random((d.tokens, 6)) < 0.4
    with_odd = q.copy()
    at = rng.integers(0, head_dim, q.shape[:2])
    np.put_along_axis(with_odd, at[..., None], np.where(odd_rows, odd, np.take_along_axis(q, at[..., None], -1)[..., 0])[..., None].astype(np.float16), -1)
    _, largest, _ = attention(q, d.host, table, lengths, starts, head_dim**-0.5, True, window)
    sees = np.broadcast_to(largest[..., 0] > 0, odd_rows.shape)
    assert (odd_rows & sees).sum() > 50 and (odd_rows & ~sees).sum() > 50
    with M.tuning(kv4_many=many, kv4_parts=parts):
        got, rest = d.attend(with_odd, 6, window=window), d.attend(q, 6, window=window)
    assert np.isnan(got[odd_rows & sees]).all()
    assert (got[odd_rows & ~sees] == 0).all() and (rest[~sees] == 0).all()
    assert np.array_equal(got[~odd_rows], rest[~odd_rows])


@pytest.mark.parametrize("many,parts", [(0, 1), (0, 5), (1, 1), (1, 4)])
@pytest.mark.parametrize("page_there", [0, 63, 64, 130, 162, None])
def test_attention_of_odd_rows_over_a_table_with_one_page(many, parts, page_there):
    """Of 163 pages one is there, or none."""
    rng = np.random.default_rng(7)
    counts, lengths = [40, 1], [2600, 2600]
    starts, lengths, table, pages = batch(rng, counts, lengths, 16)
    for row in table:
        row[np.arange(len(row)) != (-1 if page_there is None else page_there)] = -3
    d = Device(1, 64, 32, 16, pages, starts, lengths, table)
    d.fill(rng)
    q = rng.standard_normal((d.tokens, 4, 64)).astype(np.float16)
    odd_rows = rng.random((d.tokens, 4)) < 0.4
    q[odd_rows, 5] = np.nan
    with M.tuning(kv4_many=many, kv4_parts=parts):
        got = d.attend(q, 4)
    exact, largest, score = attention(np.where(odd_rows[..., None], 0, q), d.host, table, lengths, starts, 64**-0.5, True, 0)
    sees = (largest[..., 0] > 0) & (np.zeros((1, 4)) == 0)
    assert sees.any() == (page_there is not None)
    assert np.isnan(got[odd_rows & sees]).all() and (got[~sees] == 0).all()
    ordinary = ~odd_rows & sees
    check_attention(got[ordinary], exact[ordinary], largest[ordinary], score[ordinary])
