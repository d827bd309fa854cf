"""The attention of a decoder layer through the C-ABI, from its input to the o projection's output: prompts, chunks and single tokens of a
ragged batch, captured and replayed, each op against 64-bit arithmetic on what it was given."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

import workloads as W
from decoder_stack import AttentionBlock
from kv4math import Cache, attention, norm_rope, unslices
from test_gpu_fc import check_fp, textbook
from test_gpu_kv4 import check_attention, check_rope, rope_tolerance


def step(block, rng, table, lengths, counts, launch, host):
    """One step of the batch: the rows go in, each op's output is checked against its inputs."""
    import torch
    starts = np.concatenate([[0], np.cumsum(counts)])
    rows = int(starts[-1])
    x = W.round_to(rng.standard_normal((block.tokens, block.cases[0]["k"])), np.float16)
    block.x.copy_(torch.from_numpy(W.to_slices(x).astype(np.float16)))
    block.out.fill_(7.0)
    launch()
    torch.cuda.synchronize()
    fc = lambda i, act: textbook(dict(block.cases[i], m=len(act), act=act))
    # q and k are turned where they are: their projections are checked through the op's formula, at the tolerance of both
    cached = block.cache.cpu().numpy()
    v = block.v.cpu().numpy()
    check_fp(W.from_slices(v.astype(np.float32), v.shape[0] * 4)[:rows], fc(2, x[:rows]), dict(block.cases[2], m=rows), "v")
    positions = block.positions.cpu().numpy()[:rows]
    d = block.head_dim
    for i, (got, heads) in enumerate(((block.q, block.heads), (block.k, block.kv_heads))):
        ref = norm_rope(fc(i, x[:rows]).reshape(rows, heads, d), positions, d, False, weight=block.norms[i].cpu().numpy())
        err = np.abs(unslices(got.cpu().numpy(), d)[:rows].astype(np.float64) - ref)
        # a projection is within 2e-2 of its rms (check_fp); the norm makes rms 1, the weights up to 1.5, a rotation mixes two channels
        assert err.max() <= 2e-2 * 1.5 * 2 * np.sqrt(2), err.max()
    k = unslices(block.k.cpu().numpy(), d)
    for s in range(len(lengths)):
        for i in range(starts[s], starts[s + 1]):
            p = positions[i]
            host.set_token(table[s][p // block.desc.page_size], p % block.desc.page_size, k[i], unslices(v, d)[i])
    assert np.array_equal(cached, host.bytes)
    q = unslices(block.q.cpu().numpy(), d)
    exact, largest, score = attention(q, host, table, lengths, starts, d**-0.5, True, 0)
    attended = unslices(block.attended.cpu().numpy(), d)
    check_attention(attended[:rows], exact[:rows], largest[:rows], score[:rows])
    act = attended.reshape(block.tokens, -1).astype(np.float32)
    got = W.from_slices(block.out.cpu().numpy().astype(np.float32), block.cases[3]["n"])
    check_fp(got, fc(3, act), dict(block.cases[3], m=block.tokens), "o")


def test_a_batch_from_prompts_to_single_tokens():
    """A prompt beside a chunk of another, then tokens one by one in a captured graph whose lengths advance between replays."""
    import torch
    rng = np.random.default_rng(3)
    block = AttentionBlock(sequences=2, max_tokens=48, pages=9, pages_per_sequence=4, page_size=16)
    block.cache.random_(generator=torch.Generator(device="cuda").manual_seed(1))
    host = Cache(block.kv_heads, block.head_dim, block.desc.group_size, block.desc.page_size, block.desc.pages)
    host.bytes[:] = block.cache.cpu().numpy().reshape(host.bytes.shape)
    table = np.array([[7, 0, 3, 5], [2, 8, 1, 4]], np.int32)
    lengths = np.array([19, 21])
    block.set_batch(table, lengths, [0, 19, 40])
    step(block, rng, table, lengths, [19, 21], block.launch, host)
    lengths = lengths + [1, 17]
    block.set_batch(table, lengths, [0, 1, 18], tokens=20)  # (two rows of no sequence)
    step(block, rng, table, lengths, [1, 17], block.launch, host)
    lengths = lengths + 1
    block.set_batch(table, lengths, [0, 1, 2])
    step(block, rng, table, lengths, [1, 1], block.launch, host)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        block.launch()
    for _ in range(4):
        lengths = lengths + 1
        block.set_batch(table, lengths, [0, 1, 2])
        step(block, rng, table, lengths, [1, 1], graph.replay, host)
