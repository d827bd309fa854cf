"""The ops over the cache of 4-bit codes at the edges of what they are given."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

import mldhip as M
from test_gpu_kv4 import SHAPES, Device, batch, stream

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
