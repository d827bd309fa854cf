"""Norms and rotation, append and attention one behind the other, each checked row by row against 64-bit arithmetic on what it was given: nothing that
one op rounds is taken for an error of the next one, so that the bounds are those of one op."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from kv4math import attention, norm_rope, unslices
from test_gpu_kv4 import check_attention, check_rope, decode_step, rope_tolerance, stream

torch = pytest.importorskip("torch")

SHAPES = [dict(), dict(kv_heads=1, share=8, head_dim=256, group=128, page=64, counts=(1, 3, 0, 1, 7), lengths=(1, 90, 5, 700, 64)),
          dict(kv_heads=4, share=1, head_dim=64, group=32, page=32, counts=(1, 1, 90, 2), lengths=(333, 2, 150, 65)),
          dict(kv_heads=2, share=3, head_dim=128, group=64, page=16, counts=(60, 1, 17), lengths=(60, 1000, 47))]


def check_each(d, host, cache_before, positions, weights, tensors, out, table, starts):
    """host: the step's inputs; tensors: its q, k and v as the step left them."""
    head_dim = d.desc.head_dim
    q, k, v = [unslices(x.cpu().numpy(), head_dim) for x in tensors]
    for x, y, w in zip((q, k), host[:2], weights):
        check_rope(x, norm_rope(y, positions, head_dim, False, weight=w, offset=1.0), rope_tolerance(np.float16, weights), head_dim, False)
    assert np.array_equal(v, host[2])
    d.host.bytes[:] = cache_before
    for s in range(len(d.lengths)):
        for i in range(starts[s], starts[s + 1]):
            d.host.set_token(table[s][positions[i] // d.desc.page_size], positions[i] % d.desc.page_size, k[i], v[i])
    assert np.array_equal(d.cache.cpu().numpy(), d.host.bytes)
    exact, largest, score = attention(q, d.host, table, d.lengths, starts, head_dim**-0.5, True, 0)
    check_attention(unslices(out.cpu().numpy(), head_dim), exact, largest, score)
    return exact, largest, score


def inputs(rng, host, scale):
    return [(x * scale + 0.1 * rng.standard_normal(x.shape)).astype(np.float16) for x in host]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("captured", [False, True])
def test_every_row_of_a_step(shape, captured):
    """Steps with other inputs, eager on another stream than the current one, or replayed from one graph."""
    rng = np.random.default_rng(50 + len(shape))
    d, host, positions, weights, tensors, out, ops, table, starts = decode_step(rng, **shape)
    before = d.host.bytes.copy()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()

    def run(s):
        for op in ops:
            op.launch(s)

    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            run(side.cuda_stream)
    for scale in (1.0, 0.5, 2.0):
        now = inputs(rng, host, scale)
        for x, y in zip(tensors, now):
            x.copy_(torch.from_numpy(y.reshape(y.shape[0], -1, 4).transpose(1, 0, 2).copy()))
        d.cache.copy_(torch.from_numpy(before))
        out.fill_(3.0)
        torch.cuda.synchronize()
        print("step", shape, captured, scale, flush=True)
        if captured:
            graph.replay()
        else:
            run(side.cuda_stream)
        torch.cuda.synchronize()
        check_each(d, now, before, positions, weights, tensors, out, table, starts)


def test_the_bounds_of_a_step_tell_a_position_more_from_one_less():
    """The oracle's own mistakes are seen: a row's last position left out, another head's keys."""
    rng = np.random.default_rng(60)
    d, host, positions, weights, tensors, out, ops, table, starts = decode_step(rng)
    for op in ops:
        op.launch(stream())
    torch.cuda.synchronize()
    exact, largest, score = check_each(d, host, d.host.bytes.copy(), positions, weights, tensors, out, table, starts)
    got = unslices(out.cpu().numpy(), d.desc.head_dim)
    q = unslices(tensors[0].cpu().numpy(), d.desc.head_dim)
    for lengths, rows in ((np.maximum(np.asarray(d.lengths) - 1, 1), q), (d.lengths, np.roll(q, 1, 1))):
        wrong, _, _ = attention(rows, d.host, table, lengths, starts, d.desc.head_dim**-0.5, True, 0)
        with pytest.raises(AssertionError):
            check_attention(got, wrong, largest, score)
