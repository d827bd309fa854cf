"""Argument checks and object lists of the ops between the q / k / v projections and the o projection.  No kernel is launched here."""
import numpy as np
import pytest

import mldhip as M
from kv4math import SCALES, Cache, kept, quantized


def refused(code, fn, *a, **k):
    with pytest.raises(M.MldhipError) as e:
        fn(*a, **k)
    assert e.value.code == code, e.value
    return e.value.message


GOOD = dict(kv_heads=2, head_dim=128, group_size=32, page_size=64, pages=10, sequences=3, pages_per_sequence=4)


def cache(**other):
    return M.kv4_cache_desc(**dict(GOOD, **other))


def test_object_order():
    op = M.qk_norm_rope_create(M.FLOAT16, 8, 2, 128, norm=True, max_tokens=4)
    assert op.src_names == ["src_q", "src_k", "positions", "q_norm_weight", "k_norm_weight"] and op.dst_names == ["dst_q", "dst_k"]
    assert M.qk_norm_rope_create(M.FLOAT32, 8, 2, 128).src_names == ["src_q", "src_k", "positions"]
    op = M.kv4_append_create(cache(), M.FLOAT16, 8)
    assert op.src_names == ["src_k", "src_v", "page_table", "lengths", "starts"] and op.dst_names == ["cache"]
    op = M.kv4_read_create(cache(), M.FLOAT32, 8)
    assert op.src_names == ["cache", "page_table", "lengths", "starts"] and op.dst_names == ["dst_k", "dst_v"]
    op = M.kv4_attention_create(cache(), 8, max_tokens=8)
    assert op.src_names == ["src_q", "cache", "page_table", "lengths", "starts"] and op.dst_names == ["dst_tensor"]


@pytest.mark.parametrize("head_dim,group,page", [(64, 32, 16), (64, 64, 1024), (128, 32, 64), (128, 128, 16), (256, 64, 128)])
def test_cache_bytes(head_dim, group, page):
    c = cache(head_dim=head_dim, group_size=group, page_size=page)
    assert M.kv4_cache_bytes(c) == Cache(2, head_dim, group, page, 10).bytes.size
    big = cache(head_dim=head_dim, group_size=group, page_size=page, pages=1 << 20, kv_heads=64)
    assert M.kv4_cache_bytes(big) == (64 << 20) * page * (head_dim + 4 * head_dim // group)  # (past 32 bits)


def creators():
    return [lambda c: M.kv4_cache_bytes(c), lambda c: M.kv4_append_create(c, M.FLOAT16, 4), lambda c: M.kv4_read_create(c, M.FLOAT16, 4),
            lambda c: M.kv4_attention_create(c, c.kv_heads * 4, scale=1.0, max_tokens=4)]


@pytest.mark.parametrize("create", creators())
def test_cache_descriptions_that_are_refused(create):
    create(cache())
    for name in ("kv_heads", "pages", "sequences", "pages_per_sequence"):
        refused(M.INVALID_ARGUMENT, create, cache(**{name: 0}))
        refused(M.INVALID_ARGUMENT, create, cache(**{name: -3}))
    for head_dim in (0, 32, 96, 192, 512):
        refused(M.UNIMPLEMENTED, create, cache(head_dim=head_dim))
    for group in (0, 16, 48, 256):
        refused(M.INVALID_ARGUMENT, create, cache(group_size=group))
    refused(M.INVALID_ARGUMENT, create, cache(head_dim=64, group_size=128))
    for page in (0, 8, 24, 48, 2048, -16):
        refused(M.INVALID_ARGUMENT, create, cache(page_size=page))
    refused(M.OUT_OF_RANGE, create, cache(sequences=65536))
    refused(M.OUT_OF_RANGE, create, cache(kv_heads=32768))
    refused(M.OUT_OF_RANGE, create, cache(page_size=1024, pages_per_sequence=(1 << 20) + 1))


def test_other_arguments_that_are_refused():
    for create in (M.kv4_append_create, M.kv4_read_create):
        refused(M.INVALID_ARGUMENT, create, cache(), M.INT8, 4)
        refused(M.INVALID_ARGUMENT, create, cache(), M.FLOAT16, 0)
        refused(M.INVALID_ARGUMENT, create, cache(), M.FLOAT16, 4, 0)
    make = lambda heads=8, **k: M.kv4_attention_create(cache(), heads, **dict(dict(max_tokens=4), **k))
    make()
    for heads in (0, -8, 7):
        refused(M.INVALID_ARGUMENT, make, heads)
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        refused(M.INVALID_ARGUMENT, make, scale=scale)
    refused(M.INVALID_ARGUMENT, make, window=-1)
    refused(M.INVALID_ARGUMENT, make, window=(1 << 30) + 1)
    refused(M.INVALID_ARGUMENT, make, causal=2)
    refused(M.INVALID_ARGUMENT, make, max_tokens=0)
    refused(M.INVALID_ARGUMENT, make, max_new_tokens=0)
    refused(M.OUT_OF_RANGE, make, max_tokens=(1 << 27) + 1)
    rope = lambda **k: M.qk_norm_rope_create(**dict(dict(src_type=M.FLOAT16, heads=4, kv_heads=2, head_dim=64, rotary_dim=64, norm=True), **k))
    rope()
    for bad in (dict(src_type=M.INT8), dict(heads=0), dict(kv_heads=0), dict(head_dim=0), dict(head_dim=60), dict(rotary_dim=-8), dict(rotary_dim=12),
                dict(rotary_dim=72), dict(eps=-1.0), dict(eps=float("nan")), dict(weight_offset=float("inf")), dict(base=0.0), dict(base=float("nan")),
                dict(interleaved=2), dict(max_tokens=0), dict(frequencies=np.full(32, np.inf))):
        refused(M.INVALID_ARGUMENT, rope, **bad)
    refused(M.UNIMPLEMENTED, rope, head_dim=264, rotary_dim=8)
    refused(M.OUT_OF_RANGE, rope, heads=65535)
    with pytest.raises(ValueError):
        rope(frequencies=np.ones(31))


def test_bindings_and_shapes():
    op = M.kv4_attention_create(cache(), 8, max_tokens=4, max_new_tokens=2)
    assert "src_q" in refused(M.FAILED_PRECONDITION, op.launch)
    refused(M.OUT_OF_RANGE, op.set_shape, 1, 1, 5)
    op.set_shape(1, 1, 3)
    sizes = [8 * 128 * 3 * 2, M.kv4_cache_bytes(cache()), 3 * 4 * 4, 3 * 4, 4 * 4]
    for i, n in enumerate(sizes):
        op.set_src_raw(i, 4096, n)
    op.set_dst_raw(0, 4096, sizes[0])
    for i, n in enumerate(sizes):
        op.set_src_raw(i, 4096, n - 1)
        assert op.src_names[i] in refused(M.INVALID_ARGUMENT, op.launch)
        op.set_src_raw(i, 4096, n)
    op.set_dst_raw(0, 4096, sizes[0] - 1)
    assert "dst_tensor" in refused(M.INVALID_ARGUMENT, op.launch)
    refused(M.INVALID_ARGUMENT, op.set_src_raw, 1, 4100, 1 << 20)  # not 16-byte aligned
    for op, srcs, dsts in (
            (M.kv4_append_create(cache(), M.FLOAT32, 4), [2 * 128 * 4 * 4] * 2 + sizes[2:], [sizes[1]]),
            (M.kv4_read_create(cache(), M.FLOAT16, 4), sizes[1:], [2 * 128 * 4 * 2] * 2),
            (M.qk_norm_rope_create(M.FLOAT16, 8, 2, 128, norm=True, max_tokens=4), [8 * 128 * 8, 2 * 128 * 8, 16, 256, 256], [8 * 128 * 8, 2 * 128 * 8])):
        op.set_shape(1, 1, 4)
        for i, n in enumerate(srcs):
            op.set_src_raw(i, 4096, n)
        for i, n in enumerate(dsts):
            op.set_dst_raw(i, 4096, n)
        for i, n in enumerate(srcs):
            op.set_src_raw(i, 4096, n - 1)
            assert op.src_names[i] in refused(M.INVALID_ARGUMENT, op.launch)
            op.set_src_raw(i, 4096, n)
        for i, n in enumerate(dsts):
            op.set_dst_raw(i, 4096, n - 1)
            assert op.dst_names[i] in refused(M.INVALID_ARGUMENT, op.launch)
            op.set_dst_raw(i, 4096, n)


def test_cost():
    op = M.kv4_append_create(cache(), M.FLOAT16, 4)
    op.set_shape(1, 1, 4)
    assert op.cost() == (2 * 4 * 256 * 2 + (3 * 4 + 3 + 4) * 4 + 4 * 2 * (128 + 16), 20 * 4 * 256)
    op = M.kv4_attention_create(cache(), 8, max_tokens=4)
    op.set_shape(1, 1, 4)
    held = 3 * 4 * 64
    assert op.cost() == (2 * 4 * 8 * 128 * 2 + (3 * 4 + 3 + 4) * 4 + held * 2 * (128 + 16), 4 * 4 * 8 * 128 * 4 * 64)


def test_the_arithmetic_that_the_gpu_tests_check_against():
    """Properties of the cache's definition: values are halfs, at most half a step off (a whole one at the ends), idempotent."""
    rng = np.random.default_rng(0)
    x = rng.standard_normal((200, 128)) * 10.0 ** rng.uniform(-4, 3, (200, 1)) + rng.standard_normal((200, 1))
    codes, scale, zero = quantized(x, 32)
    assert codes.min() >= 0 and codes.max() <= 15 and zero.min() >= 0 and zero.max() <= 15
    assert np.isin(scale, SCALES).all() and np.array_equal(SCALES.astype(np.float16).astype(np.float64), SCALES)
    assert not (SCALES.astype(np.float16).view(np.uint16) & 15).any()
    y = kept(x, 32)
    assert np.array_equal(y.astype(np.float16).astype(np.float64), y)
    assert (np.abs(x - y).reshape(200, 4, 32) <= scale[..., None] * 1.0001).all()
    inner = (codes > 0) & (codes < 15)
    assert (np.abs(x - y)[inner] <= 0.5 * np.repeat(scale, 32, -1)[inner] * 1.0001).all()
    widest = kept(np.array([[1e9, -1e9] + [0.0] * 30]), 32)
    assert np.isfinite(widest.astype(np.float16)).all() and abs(widest[0, 0] - 57344) < 8000
    assert not kept(np.full((1, 32), np.nan), 32).any()


def test_sizes_past_what_a_launch_can_count_are_refused():
    for create in creators():
        refused(M.OUT_OF_RANGE, create, cache(head_dim=256, group_size=32, page_size=1024, pages=(1 << 31) - 1, kv_heads=32767))  # 2^64 and more
        refused(M.OUT_OF_RANGE, create, cache(page_size=1024, pages=1 << 28, kv_heads=128))
    most = 1 << 24
    for create in (M.kv4_append_create, M.kv4_read_create):
        create(cache(), M.FLOAT16, most)
        refused(M.OUT_OF_RANGE, create, cache(), M.FLOAT16, most + 1)
    refused(M.OUT_OF_RANGE, M.kv4_attention_create, cache(), 2, max_tokens=most + 1)
    refused(M.INVALID_ARGUMENT, M.kv4_attention_create, cache(), 2, scale=3e38)
    M.qk_norm_rope_create(M.FLOAT16, 8, 2, 128, max_tokens=most)
    refused(M.OUT_OF_RANGE, M.qk_norm_rope_create, M.FLOAT16, 8, 2, 128, max_tokens=most + 1)


def test_attention_into_its_own_queries_is_refused():
    op = M.kv4_attention_create(cache(), 8, max_tokens=4)
    op.set_shape(1, 1, 4)
    for i, n in enumerate([8 * 128 * 4 * 2, M.kv4_cache_bytes(cache()), 3 * 4 * 4, 3 * 4, 4 * 4]):
        op.set_src_raw(i, 4096 * (i + 1), n)
    op.set_dst_raw(0, 4096, 8 * 128 * 4 * 2)
    assert "src_q" in refused(M.INVALID_ARGUMENT, op.launch)


def test_results_into_one_buffer_are_refused():
    def launch(op, srcs, dsts):
        op.set_shape(1, 1, 4)
        for i, p in enumerate(srcs):
            op.set_src_raw(i, p, 1 << 30)
        for i, p in enumerate(dsts):
            op.set_dst_raw(i, p, 1 << 30)
        return refused(M.INVALID_ARGUMENT, op.launch)

    rope = M.qk_norm_rope_create(M.FLOAT16, 2, 2, 128, max_tokens=4)
    assert "src_k" in launch(rope, [4096, 8192, 12288], [8192, 16384])
    assert "src_q" in launch(rope, [4096, 8192, 12288], [16384, 4096])
    assert "one buffer" in launch(rope, [4096, 8192, 12288], [16384, 16384])
    assert "one buffer" in launch(M.kv4_read_create(cache(), M.FLOAT16, 4), [4096, 8192, 12288, 16384], [20480, 20480])
