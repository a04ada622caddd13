"""A drafted step as a serving program runs it, over one pool of pages for two layers: prompts in, then step after step the last tokens
and trees of drafts stored and attended to, verified, and the accepted rows kept; against the same kept on the host in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import mxfp4
from tests.drafts import masked_attention64, quantise64, random_parents, seen_rows, turned64, verify64
from tests.serving import assert_within, attention64, cumulative, i32
from texelator_amd import layers

pytestmark = pytest.mark.gpu
LAYERS, HEADS, KV_HEADS, PAGE, VOCAB = 2, 10, 2, 16, 700


class Server:
    """What the program keeps on the device, and every sequence's cached values [2, positions, kv_heads, dim] of each layer on the host."""

    def __init__(self, rows, dim, dtype, chain=False, columns=24):
        self.rows, self.dim, self.dtype, self.scale, self.chain = rows, dim, dtype, dim ** -0.5, chain
        slots = len(rows)
        rng = np.random.default_rng(3)
        self.pools = layers.kv4_pages(slots * columns + 5, KV_HEADS, dim, PAGE, layers=LAYERS)
        self.pools.fill_(255)  # NaN wherever it is read unwritten
        self.table = i32(rng.permutation(slots * columns + 5)[:slots * columns]).view(slots, columns)
        self.lengths = torch.zeros(slots, dtype=torch.int32, device="cuda")
        self.count = [0] * slots  # positions decided
        self.cached = [[torch.zeros(2, 0, KV_HEADS, dim, dtype=torch.float64) for _ in rows] for _ in range(LAYERS)]
        frequency = 1e4 ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
        angles = torch.arange(columns * PAGE, dtype=torch.float64)[:, None] * frequency
        self.cos, self.sin = angles.cos().float().cuda(), angles.sin().float().cuda()
        self.g = torch.Generator().manual_seed(5)
        self.trees = [list(range(-1, n - 1)) if chain else random_parents(rng, n) for n in rows]
        self.depths = [[0] * n for n in rows]
        for tree, depth in zip(self.trees, self.depths):
            for i, p in enumerate(tree):
                depth[i] = depth[p] + 1 if p >= 0 else 0
        self.cu = cumulative(rows)
        self.parents = None if chain else i32([p for tree in self.trees for p in tree])
        total = sum(rows)
        self.depth = i32([d for depth in self.depths for d in depth])
        self.sequence = torch.repeat_interleave(torch.arange(slots, device="cuda"), i32(rows).long())
        # The step's own buffers: inputs of every layer, the model's logits, drafts and random numbers.
        self.q = [torch.zeros(total, HEADS, dim, dtype=dtype, device="cuda") for _ in range(LAYERS)]
        self.kv = [torch.zeros(total, 2, KV_HEADS, dim, dtype=dtype, device="cuda") for _ in range(LAYERS)]
        self.out = [torch.zeros(total, HEADS, dim, dtype=dtype, device="cuda") for _ in range(LAYERS)]
        self.turned = [torch.zeros(total, HEADS, dim, dtype=dtype, device="cuda") for _ in range(LAYERS)]
        self.logits = torch.zeros(total, VOCAB, dtype=torch.bfloat16, device="cuda")
        self.draft_logits = torch.zeros_like(self.logits) if chain else None
        self.ids = torch.zeros(total, dtype=torch.int64, device="cuda")
        self.uniforms = torch.zeros(total, device="cuda")
        self.temperature = torch.tensor([(0.8, 0.0, 1.2)[i % 3] for i in range(slots)], device="cuda")
        self.result = (torch.zeros(slots, dtype=torch.int32, device="cuda"), torch.zeros(total, dtype=torch.int32, device="cuda"),
                       torch.zeros(total, dtype=torch.int64, device="cuda"))
        self.kept = torch.zeros(slots, dtype=torch.int32, device="cuda")

    def stored(self, k, v, positions):
        """float64 [2, tokens, kv_heads, dim]: what the cache holds of these rows."""
        turned = turned64(k.cpu(), self.cos[positions].cpu(), self.sin[positions].cpu(), False)
        return torch.from_numpy(mxfp4.dequantize(*quantise64(torch.stack([turned, v.cpu().double()]).numpy())))

    def prompt(self, new):
        cu, places = cumulative(new), [p for n in new for p in range(n)]
        self.lengths.copy_(i32(new))
        for layer in range(LAYERS):
            q, k, v = (torch.randn(sum(new), h, self.dim, generator=self.g).to(self.dtype).cuda() for h in (HEADS, KV_HEADS, KV_HEADS))
            turned = torch.empty_like(k)
            q = layers.kv4_append_rope(q, k, v, self.cos, self.sin, self.pools[layer], self.table, self.lengths, cu=cu, k_out=turned)
            out = layers.packed_attention(q, turned, v, cu, self.scale)
            values = self.stored(k, v, places)
            for s, n in enumerate(new):
                rows = slice(sum(new[:s]), sum(new[:s]) + n)
                for h in range(HEADS):
                    kv = h // (HEADS // KV_HEADS)
                    assert_within(out[rows, h], *attention64(q[rows, h], turned[rows, kv], v[rows, kv], self.scale, 0))
                self.cached[layer][s] = values[:, rows]
        self.count = list(new)
        self.lengths += i32(self.rows)

    def fill(self):
        """Another step's inputs: drafts that mostly agree with the target."""
        def fresh(t, x):
            t.copy_(x.to(t.dtype))

        for layer in range(LAYERS):
            fresh(self.q[layer], torch.randn(self.q[layer].shape, generator=self.g))
            fresh(self.kv[layer], torch.randn(self.kv[layer].shape, generator=self.g))
        target = 2 * torch.randn(self.logits.shape, generator=self.g)
        target.scatter_add_(1, torch.randint(0, VOCAB, (len(target), 3), generator=self.g), torch.full((len(target), 3), 12.0))
        draft = (target + 0.7 * torch.randn(target.shape, generator=self.g)).bfloat16()
        ids, at = torch.zeros(len(target), dtype=torch.int64), 0
        for tree in self.trees:
            tried = {}
            for i, parent in enumerate(tree):
                rank = tried.get(parent, 0)
                tried[parent] = rank + 1
                row = draft[at + max(parent, 0)].float()
                ids[at + i] = torch.multinomial(torch.softmax(row, 0), 1, generator=self.g)[0] if self.chain else row.topk(rank + 1).indices[-1]
            at += len(tree)
        fresh(self.logits, target)
        fresh(self.ids, ids)
        fresh(self.uniforms, torch.rand(len(target), generator=self.g))
        if self.chain:
            fresh(self.draft_logits, draft)

    def step(self):
        """All on the device: nothing of it waits for the host."""
        places = (self.lengths - (self.cu[1:] - self.cu[:-1]))[self.sequence] + self.depth
        for layer in range(LAYERS):
            layers.kv4_append_rope(self.q[layer], self.kv[layer][:, 0], self.kv[layer][:, 1], self.cos, self.sin, self.pools[layer], self.table,
                                   self.lengths, cu=self.cu, positions=places.int(), out=self.turned[layer])
            layers.kv4_tree_attention(self.turned[layer], self.pools[layer], self.table, self.lengths, self.cu, self.scale,
                                      parents=self.parents, out=self.out[layer])
        layers.verify_drafts(self.logits, self.ids, self.uniforms, self.cu, parents=self.parents, draft_logits=self.draft_logits,
                             temperature=self.temperature, out=self.result)
        layers.kv4_keep_path(self.pools, self.table, self.lengths, self.cu, self.result[1], self.result[0], self.dim, out=self.kept)
        self.lengths.copy_(self.kept + (self.cu[1:] - self.cu[:-1]))

    def check(self):
        """After a step: its outputs, its choice, and the lengths; then the host's copy of the cache follows."""
        want = verify64(self.logits.cpu(), self.ids.cpu(), self.uniforms.cpu(), self.trees, self.temperature.tolist(),
                        None if self.draft_logits is None else self.draft_logits.cpu())
        assert [t.tolist() for t in self.result] == [list(w) for w in want]
        places = [c + d for c, depth in zip(self.count, self.depths) for d in depth]
        for layer in range(LAYERS):
            rows = self.stored(self.kv[layer][:, 0], self.kv[layer][:, 1], places)
            at = 0
            for s, (n, tree) in enumerate(zip(self.rows, self.trees)):
                values = torch.cat([self.cached[layer][s], rows[:, at:at + n]], dim=1)
                hidden = torch.cat([torch.zeros(n, self.count[s], dtype=torch.bool), torch.from_numpy(~seen_rows(tree, n))], dim=1).cuda()
                for h in range(HEADS if n else 0):
                    k, v = values[:, :, h // (HEADS // KV_HEADS)].cuda()
                    assert_within(self.out[layer][at:at + n, h], *masked_attention64(self.turned[layer][at:at + n, h], k, v, self.scale, hidden))
                steps = [r for r in want[1][at:at + n] if r >= 0]
                self.cached[layer][s] = torch.cat([self.cached[layer][s], rows[:, [at + r for r in steps]]], dim=1)
                at += n
        self.count = [c + a + 1 for c, a in zip(self.count, want[0])]
        assert self.kept.tolist() == self.count and self.lengths.tolist() == [c + n for c, n in zip(self.count, self.rows)]
        return want[0]

    def check_cache(self):
        """Every decided position of every layer as the cache reads it."""
        for layer in range(LAYERS):
            k, v = layers.kv4_read(self.pools[layer], self.table, self.kept, self.dim, cu=cumulative(self.count), tokens=sum(self.count), dtype=self.dtype)
            want = torch.cat(self.cached[layer], dim=1).to(self.dtype)
            assert torch.equal(torch.stack([k, v]).cpu(), want)


@pytest.mark.parametrize("rows,dim,dtype,chain", [([6, 1, 11, 0], 128, torch.bfloat16, False), ([4, 9, 2], 64, torch.float16, True)])
def test_step_after_step(ext, rows, dim, dtype, chain):
    server = Server(rows, dim, dtype, chain)
    server.prompt([37, 5, 90, 16][:len(rows)])
    accepted = 0
    for _ in range(6):
        server.fill()
        server.step()
        accepted += sum(max(a, 0) for a in server.check())
    server.check_cache()
    assert accepted > 0


@pytest.mark.parametrize("rows,dim,dtype,chain", [([6, 1, 11, 0], 128, torch.bfloat16, False), ([4, 9, 2], 64, torch.float16, True)])
def test_a_captured_step_serves_the_lengths_of_each_replay(ext, rows, dim, dtype, chain):
    """The whole step captured once: lengths, paths and caches go from replay to replay on the device, with eager work between."""
    server = Server(rows, dim, dtype, chain)
    server.prompt([37, 5, 90, 16][:len(rows)])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        server.fill()
        before, pools = server.lengths.clone(), server.pools.clone()
        server.step()  # the warm-up
        stream.synchronize()
        server.lengths.copy_(before)
        server.pools.copy_(pools)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            server.step()
        for turn in range(8):
            if turn:
                server.fill()
            graph.replay()
            stream.synchronize()
            server.check()
        server.check_cache()


def test_two_graphs_share_workspaces(ext):
    """Attention and verification of two kinds of batch captured into two graphs with the same workspaces, replayed in turn on one
    stream."""
    servers = [Server([6, 1, 11, 0], 128, torch.bfloat16), Server([4, 9, 2], 128, torch.bfloat16, chain=True)]
    for server in servers:
        server.prompt([300, 5, 90, 16][:len(server.rows)])
    sizes = [(layers.kv4_tree_attention_workspace_bytes(s.pools[0], s.table, sum(s.rows), HEADS, s.dim),
              layers.verify_drafts_workspace_bytes(s.logits, len(s.rows), sampled=s.chain)) for s in servers]
    spaces = [torch.full((max(size[i] for size in sizes) + 16,), 255, dtype=torch.uint8, device="cuda") for i in range(2)]

    def run(server):
        for layer in range(LAYERS):
            layers.kv4_tree_attention(server.q[layer], server.pools[layer], server.table, server.lengths, server.cu, server.scale,
                                      parents=server.parents, out=server.out[layer], workspace=spaces[0])
        layers.verify_drafts(server.logits, server.ids, server.uniforms, server.cu, parents=server.parents, draft_logits=server.draft_logits,
                             temperature=server.temperature, out=server.result, workspace=spaces[1])

    stream, graphs = torch.cuda.Stream(), []
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for server in servers:
            run(server)
            stream.synchronize()
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=stream):
                run(server)
        for turn in range(6):
            for server, graph in zip(servers, graphs):
                server.fill()
                for layer in range(LAYERS):
                    layers.kv4_append_rope(server.q[layer], server.kv[layer][:, 0], server.kv[layer][:, 1], server.cos, server.sin,
                                           server.pools[layer], server.table, server.lengths, cu=server.cu, out=server.turned[layer])
                graph.replay()
            stream.synchronize()
            for server in servers:
                got = [t.clone() for t in (*server.out, *server.result)]
                for layer in range(LAYERS):
                    want = layers.kv4_tree_attention(server.q[layer], server.pools[layer], server.table, server.lengths, server.cu,
                                                     server.scale, parents=server.parents)
                    assert torch.equal(got[layer], want), turn
                want = layers.verify_drafts(server.logits, server.ids, server.uniforms, server.cu, parents=server.parents,
                                            draft_logits=server.draft_logits, temperature=server.temperature)
                assert all(torch.equal(a, b) for a, b in zip(got[LAYERS:], want)), turn
