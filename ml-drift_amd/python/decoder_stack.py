"""The FullyConnected sequence of a decoder stack (Gemma-2B-like: hidden 2048, MQA k/v 256,
gated MLP 16384, int4 group-32 weights, fp16 tensors), as the reference's model builder emits
it per layer (samples/llm/gemma3_model_builder.cc:1115-1128): q, k, v, o, gate, up, down.

DecoderStack reproduces the FCs only (no attention, norm or activation): every FC reads a synthetic
N(0,1) activation tensor of its input width and writes its own output tensor, and the FCs run
in the graph's order on one stream, i.e. with the dependencies of the real layer.  Every FC of
every layer has weights and scales of its own (seed layer * 7 + index), so a decode step streams
the whole stack's 1.1 GB through HBM.  (What a GEMV or GEMM costs does not depend on the values of
its activations, so the synthetic inputs time like the fed-forward ones; the chain with the values
flowing through it is a parity test.)

AttentionBlock is the attention of such a layer with the values flowing through it: q / k / v, the norms of the
heads and the rotation, the new keys and values into a paged cache of 4-bit codes, attention over it, o.

Nothing here computes a result on the host.
"""
import numpy as np

import mldhip as M
import workloads as W


class DecoderStack:
    def __init__(self, layers=W.C5_LAYERS, max_tokens=128, seed=5, layer_shapes=None, device="cuda", keep_host=True,
                 decode_layout=False):
        import torch
        self.torch = torch
        self.layers = layers
        self.max_tokens = max_tokens
        self.shapes = list(layer_shapes or W.C5_LAYER)
        self.device = device
        # host-side cases: every FC of every layer has weights and scales of its own, seed
        # layer * 7 + index; the FCs of one input width share one synthetic N(0,1) activation tensor
        self.inputs = {}
        rng = np.random.default_rng(seed)
        for _, k, _ in self.shapes:
            if k not in self.inputs:
                self.inputs[k] = W.round_to(rng.standard_normal((max_tokens, k)), np.float16)
        self.keep_host = keep_host
        self.layer_cases = []
        self.tokens = None
        self.src = {}
        self.nodes = []  # (layer, case index, op, out tensor, weights, scales)
        self._weights = []
        for layer in range(layers):
            cases = []
            for idx, (name, k, n) in enumerate(self.shapes):
                case = W.make_fc_case(seed=layer * 7 + idx, m=1, k=k, n=n, weight_bits=4, tensor_dtype=np.float16,
                                      groups=k // 32)
                case["name"] = name
                case["m"] = max_tokens
                case["act"] = self.inputs[k]
                # decode_layout: the weights as a decode graph's ops ask for them (the prefill graph keeps
                # its own packed copy)
                desc, w = W.pack_fc_weights(case, decode_layout=decode_layout)
                sc = M.scale_to_tensor(case["scale"], M.FLOAT16).view(np.float16)
                w_dev = torch.from_numpy(w).to(device)
                s_dev = torch.from_numpy(sc).to(device)
                out = torch.zeros((W.div_up(n, 4), max_tokens, 4), dtype=torch.float16, device=device)
                op = M.fc_create(M.PRECISION_F32_F16, M.FLOAT16, M.FLOAT16, n, k, desc,
                                 scale_shape=(n, case["groups"]), max_tokens=max_tokens)
                self._weights.append((w_dev, s_dev))
                self.nodes.append((layer, idx, op, out, w_dev, s_dev))
                if not keep_host:  # the bench needs the shapes only
                    case = dict(case, w=None, scale=None)
                cases.append(case)
            self.layer_cases.append(cases)
        self.cases = self.layer_cases[0]
        self.set_tokens(1)

    def weight_bytes(self):
        """Packed weights + scales of the whole stack (the bytes a decode step must stream)."""
        return sum(w.numel() * w.element_size() + s.numel() * s.element_size() for w, s in self._weights)

    def flops(self, tokens):
        return self.layers * sum(2.0 * tokens * c["k"] * c["n"] for c in self.cases)

    def set_tokens(self, tokens):
        """Re-binds every FC for `tokens` tokens (the first `tokens` rows of the synthetic input)."""
        assert 1 <= tokens <= self.max_tokens
        torch = self.torch
        self.tokens = tokens
        self.src = {k: torch.from_numpy(W.to_slices(a[:tokens]).astype(np.float16)).to(self.device)
                    for k, a in self.inputs.items()}
        self.outs = []
        for layer, idx, op, out, w_dev, s_dev in self.nodes:
            case = self.cases[idx]
            view = out.view(-1)[: W.div_up(case["n"], 4) * tokens * 4].view(W.div_up(case["n"], 4), tokens, 4)
            op.bind([self.src[case["k"]], w_dev, s_dev], [view])
            op.set_shape(1, 1, tokens)
            self.outs.append(view)

    def launch(self, stream=None, fused=True):
        """One pass over the stack in node order.  With `fused`, the FCs of a layer that read the
        same tensor (q/k/v; gate/up) go out as one launch where the library can serve them
        together (decode), singly otherwise."""
        s = self.torch.cuda.current_stream().cuda_stream if stream is None else stream
        if not fused:
            for _, _, op, _, _, _ in self.nodes:
                op.launch(s)
            return
        names = [c["name"] for c in self.cases]
        per_layer = len(self.cases)
        groups = [[names.index(n) for n in grp] for grp in self.PARALLEL if all(n in names for n in grp)]
        for layer in range(self.layers):
            idx = 0
            while idx < per_layer:
                grp = next((g for g in groups if g[0] == idx and g == list(range(idx, idx + len(g)))), None)
                if grp is not None:
                    ops = [self.nodes[layer * per_layer + i][2] for i in grp]
                    try:
                        M.fc_launch_fused(ops, s)
                        idx += len(grp)
                        continue
                    except M.MldhipError as e:
                        if e.code != M.FAILED_PRECONDITION:
                            raise
                self.nodes[layer * per_layer + idx][2].launch(s)
                idx += 1

    # FCs of a layer that read the same tensor and do not depend on each other
    PARALLEL = (("q", "k", "v"), ("gate", "up"))

    def capture(self, parallel=False):
        """Captures one pass over the stack into a graph and returns it (replay with .replay()).
        With `parallel`, the FCs of a layer that are independent in the real graph (q/k/v; gate/up)
        are captured as parallel branches, each on its own stream of default priority; the
        dependent ones (o after q/k/v, down after gate/up, next layer after down) stay ordered.
        (On MI355X the fork/join of the branches costs more than the overlap gains: 1093 us
        against 873 us for a decode step, hence the default.)"""
        torch = self.torch
        self.launch(fused=False)  # warm-up
        torch.cuda.synchronize()
        main = torch.cuda.Stream()
        side = [torch.cuda.Stream(), torch.cuda.Stream()]
        names = [c["name"] for c in self.cases]
        group_of = {}
        for grp in self.PARALLEL:
            if parallel and all(n in names for n in grp):
                for n in grp:
                    group_of[n] = grp
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=main):
            per_layer = len(self.cases)
            for layer in range(self.layers):
                idx = 0
                while idx < per_layer:
                    name = names[idx]
                    grp = group_of.get(name)
                    if grp is None or name != grp[0]:
                        self.nodes[layer * per_layer + idx][2].launch(main.cuda_stream)
                        idx += 1
                        continue
                    fork = main.record_event()
                    members = [names.index(n) for n in grp]
                    self.nodes[layer * per_layer + members[0]][2].launch(main.cuda_stream)
                    for st, mi in zip(side, members[1:]):
                        st.wait_event(fork)
                        self.nodes[layer * per_layer + mi][2].launch(st.cuda_stream)
                        main.wait_event(st.record_event())
                    idx = max(members) + 1
        self._graph_streams = (main, side)
        return graph

    def result(self, layer, idx):
        self.torch.cuda.synchronize()
        pos = layer * len(self.cases) + idx
        return W.from_slices(self.outs[pos].cpu().numpy().astype(np.float32), self.cases[idx]["n"])

    def case(self, idx, tokens=None, layer=0):
        """The host-side case of FC `idx` of `layer` restricted to the current token count."""
        t = self.tokens if tokens is None else tokens
        c = dict(self.layer_cases[layer][idx])
        c["m"] = t
        c["act"] = c["act"][:t]
        return c

    def kernel_names(self):
        return [op.kernel_name for _, _, op, _, _, _ in self.nodes]


class AttentionBlock:
    """q / k / v -> norms and rotation -> cache -> attention -> o, on one stream (q / k / v as one launch where they can be) over ragged batches of
    `sequences` sequences: prompts, chunks of prompts and single tokens alike.  set_batch() says which rows are whose and rebinds; launch() neither
    allocates nor synchronises and may be captured, and page_table, lengths, starts and positions may be rewritten between replays.
    The cache has `pages` pages, of which the caller gives each sequence its own in page_table."""

    def __init__(self, heads=8, kv_heads=1, head_dim=256, hidden=2048, sequences=1, max_tokens=128, max_new_tokens=None, pages=64,
                 pages_per_sequence=None, page_size=64, group_size=32, window=0, base=10000.0, seed=5, device="cuda"):
        import torch
        self.torch = torch
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        self.max_tokens = max_tokens
        most_new = max_tokens if max_new_tokens is None else max_new_tokens
        self.desc = M.kv4_cache_desc(kv_heads, head_dim, group_size, page_size, pages, sequences, pages_per_sequence or pages)
        self.cache = torch.zeros(M.kv4_cache_bytes(self.desc), dtype=torch.uint8, device=device)
        ints = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=device)
        self.page_table, self.lengths = ints(sequences, self.desc.pages_per_sequence), ints(sequences)
        self.starts, self.positions = ints(sequences + 1), ints(max_tokens)
        rng = np.random.default_rng(seed)
        self.norms = [torch.from_numpy(rng.uniform(0.5, 1.5, head_dim).astype(np.float16)).to(device) for _ in range(2)]
        width = heads * head_dim
        self.cases, self.fc, self._weights, self._buffers = [], [], [], {}
        for i, (name, k, n) in enumerate([("q", hidden, width), ("k", hidden, kv_heads * head_dim), ("v", hidden, kv_heads * head_dim),
                                          ("o", width, hidden)]):
            case = W.make_fc_case(seed=seed * 7 + i, m=1, k=k, n=n, weight_bits=4, tensor_dtype=np.float16, groups=k // 32)
            case["name"] = name
            desc, w = W.pack_fc_weights(case)
            sc = M.scale_to_tensor(case["scale"], M.FLOAT16).view(np.float16)
            self._weights.append((torch.from_numpy(w).to(device), torch.from_numpy(sc).to(device)))
            self.fc.append(M.fc_create(M.PRECISION_F32_F16, M.FLOAT16, M.FLOAT16, n, k, desc, scale_shape=(n, case["groups"]),
                                       max_tokens=max_tokens))
            self.cases.append(case)
        for name, channels in [("x", hidden), ("q", width), ("k", kv_heads * head_dim), ("v", kv_heads * head_dim), ("attended", width),
                               ("out", hidden)]:
            self._buffers[name] = torch.zeros(channels * max_tokens, dtype=torch.float16, device=device)
        self.rope = M.qk_norm_rope_create(M.FLOAT16, heads, kv_heads, head_dim, base=base, norm=True, max_tokens=max_tokens)
        self.append = M.kv4_append_create(self.desc, M.FLOAT16, max_tokens, most_new)
        self.attend = M.kv4_attention_create(self.desc, heads, window=window, max_tokens=max_tokens, max_new_tokens=most_new)

    def set_batch(self, page_table, lengths, starts, tokens=None):
        """page_table [sequences][pages_per_sequence], lengths and starts as the ops over the cache take them (lengths count the new
        tokens).  tokens: rows of the tensors, starts[-1] unless given (padded batches)."""
        torch = self.torch
        page_table, lengths, starts = [np.asarray(a, np.int32) for a in (page_table, lengths, starts)]
        if page_table.ndim == 1 and len(self.page_table) == 1:
            page_table = page_table[None]  # (of one sequence)
        for name, a, to in (("page_table", page_table, self.page_table), ("lengths", lengths, self.lengths), ("starts", starts, self.starts)):
            if a.shape != tuple(to.shape):
                raise ValueError("%s: %s where the block has %s" % (name, a.shape, tuple(to.shape)))
        tokens = int(starts[-1]) if tokens is None else tokens
        if not 1 <= tokens <= self.max_tokens:
            raise ValueError("%d rows where the block was made for 1 .. %d" % (tokens, self.max_tokens))
        if starts[0] < 0 or starts[-1] > tokens or (np.diff(starts) < 0).any():
            raise ValueError("starts must not decrease, and lie within the %d rows" % tokens)
        positions = np.zeros(self.max_tokens, np.int32)
        for s, length in enumerate(lengths):
            positions[starts[s]:starts[s + 1]] = np.arange(length - (starts[s + 1] - starts[s]), length)
        for to, values in ((self.page_table, page_table), (self.lengths, lengths), (self.starts, starts), (self.positions, positions)):
            to.copy_(torch.from_numpy(np.ascontiguousarray(values, np.int32)))
        self.tokens = tokens
        view = lambda name: self._buffers[name][:self._buffers[name].numel() // self.max_tokens * tokens].view(-1, tokens, 4)
        self.x, self.q, self.k, self.v, self.attended, self.out = [view(n) for n in ("x", "q", "k", "v", "attended", "out")]
        where = [self.page_table, self.lengths, self.starts]
        for op, src, dst, weights in zip(self.fc, (self.x, self.x, self.x, self.attended), (self.q, self.k, self.v, self.out), self._weights):
            op.bind([src, *weights], [dst])
        self.rope.bind([self.q, self.k, self.positions, *self.norms], [self.q, self.k])
        self.append.bind([self.k, self.v, *where], [self.cache])
        self.attend.bind([self.q, self.cache, *where], [self.attended])
        for op in (*self.fc, self.rope, self.append, self.attend):
            op.set_shape(1, 1, tokens)

    def launch(self, stream=None):
        s = self.torch.cuda.current_stream().cuda_stream if stream is None else stream
        try:
            M.fc_launch_fused(self.fc[:3], s)
        except M.MldhipError as e:
            if e.code != M.FAILED_PRECONDITION:
                raise
            for op in self.fc[:3]:
                op.launch(s)
        for op in (self.rope, self.append, self.attend, self.fc[3]):
            op.launch(s)
