"""GPU: plan, cache write, attention and token scores together, as a server runs them: several steps of a ragged batch through
PagedKvCache -- prompts in chunks, single tokens, idle and finished requests, padded rows -- eager on a stream of its own or as
one captured graph that is replayed with other lengths.  After each step every array is compared with a plain 64-bit run of the
same steps; the tolerances are those of the operators' own tests (attention: test_gpu_kv_cache.py, scores:
test_gpu_token_logprobs.py)."""
import numpy as np
import pytest

import kv_oracle
from pyc_b200 import abi
from pyc_b200.kv_cache import PagedKvCache
from test_gpu_token_logprobs import _check as check_scores

pytestmark = pytest.mark.gpu
VOCAB, TOP, LAYERS = 777, 5, 2


class Server:
    """The device side of a step (static buffers, so that it can be captured) and the same step on the host."""

    def __init__(self, backend, dtype, requests, num_blocks, bs, width, max_tokens, group, kv_heads, dim, max_query, seed):
        import torch
        self.torch, self.backend = torch, backend
        self.c = PagedKvCache(torch, requests, num_blocks, bs, width, max_tokens, group * kv_heads, kv_heads, dim, dtype, layers=LAYERS, max_query=max_query)
        self.rng = np.random.default_rng(seed)
        H = group * kv_heads
        self.qkv = torch.zeros((LAYERS, max_tokens, (H + 2 * kv_heads) * dim), dtype=dtype, device="cuda")          # one projection's output
        self.out = torch.zeros((LAYERS, max_tokens, H, dim), dtype=dtype, device="cuda")
        self.lse = torch.zeros((LAYERS, max_tokens, H), device="cuda")
        self.head = torch.from_numpy(self.rng.standard_normal((H * dim, VOCAB))).cuda().to(dtype)
        self.logits = torch.zeros((max_tokens, VOCAB), dtype=dtype, device="cuda")
        self.tokens = torch.zeros(max_tokens, dtype=torch.int32, device="cuda")
        self.lp, self.ent, self.z = (torch.zeros(max_tokens, device="cuda") for _ in range(3))
        self.ids, self.top = torch.zeros((max_tokens, TOP), dtype=torch.int32, device="cuda"), torch.zeros((max_tokens, TOP), device="cuda")
        # host
        self.context, self.table = [0] * requests, np.full((requests, width), -1, np.int32)
        self.free, self.count = np.arange(num_blocks, dtype=np.int32), num_blocks
        self.codes = np.zeros((LAYERS, 2, num_blocks, kv_heads, bs, dim), np.uint8)
        self.scale = np.ones((LAYERS, 2, num_blocks, kv_heads), np.float32)

    def device_step(self):
        c, H = self.c, self.c.heads
        c.plan()
        for layer in range(LAYERS):
            q, k, v = self.qkv[layer].split((H * c.head_dim, c.kv_heads * c.head_dim, c.kv_heads * c.head_dim), dim=1)
            c.write(layer, k, v)
            c.attend(layer, q, out=self.out[layer], lse=self.lse[layer])
        self.torch.matmul(self.out[LAYERS - 1].flatten(1), self.head, out=self.logits)
        kind = abi.DTYPE_BF16 if c.dtype == self.torch.bfloat16 else abi.DTYPE_F16
        self.backend.token_logprobs(kind, c.max_tokens, VOCAB, self.logits.data_ptr(), self.tokens.data_ptr(), self.lp.data_ptr(),
                                    entropy=self.ent.data_ptr(), lse=self.z.data_ptr(), top_k=TOP, top_ids=self.ids.data_ptr(),
                                    top_logprobs=self.top.data_ptr(), stream=self.torch.cuda.current_stream().cuda_stream)
        c.advance()

    def feed(self, new):
        """Inputs of the next step; rows behind its tokens hold NaN in q, k and v."""
        torch, c = self.torch, self.c
        n = sum(new)
        x = self.rng.standard_normal(tuple(self.qkv.shape)) * np.exp2(self.rng.integers(-1, 2, (LAYERS, c.max_tokens, 1)))
        x[:, n:] = np.nan
        self.qkv.copy_(torch.from_numpy(x).to(c.dtype))
        self.tokens.copy_(torch.from_numpy(np.where(np.arange(c.max_tokens) < n, self.rng.integers(0, VOCAB, c.max_tokens), -1).astype(np.int32)))
        self.out.fill_(7.0)
        self.lse.fill_(7.0)
        c.new_lens.copy_(torch.tensor(new, dtype=torch.int32))

    def check(self, new):
        c, H, D = self.c, self.c.heads, self.c.head_dim
        host = lambda t: t.detach().cpu().numpy()
        want = kv_oracle.plan(self.context, new, self.free, self.count, self.table, c.block_size, c.num_blocks, c.max_tokens)
        assert want is not None
        self.count = want["free_count"]
        for name in ("query_start", "seq_lens", "slot_map", "positions", "token_request"):
            assert np.array_equal(host(getattr(c, name)), want[name]), name
        assert int(c.free_count) == self.count and np.array_equal(host(c.block_table), self.table)
        assert np.array_equal(host(c.context_lens), want["seq_lens"])
        n = sum(new)
        for layer in range(LAYERS):
            x = self.qkv[layer].double().cpu().numpy()
            q, k, v = np.split(x, [H * D, (H + c.kv_heads) * D], axis=1)
            for which, (y, codes, scale) in enumerate(((k, c.k_cache, c.k_scale), (v, c.v_cache, c.v_scale))):
                kv_oracle.write(y.reshape(len(y), c.kv_heads, D), want["slot_map"], self.codes[layer, which], self.scale[layer, which])
                assert np.array_equal(host(scale[layer]), self.scale[layer, which]) and np.array_equal(host(codes[layer]), self.codes[layer, which])
            o, z, mag = kv_oracle.attend(q.reshape(len(q), H, D), self.codes[layer, 0], self.codes[layer, 1], self.scale[layer, 0], self.scale[layer, 1],
                                         self.table, want["query_start"], want["seq_lens"], D ** -0.5, True, H // c.kv_heads)
            got, gz = self.out[layer].double().cpu().numpy(), self.lse[layer].double().cpu().numpy()
            assert (got[n:] == 7.0).all() and (gz[n:] == 7.0).all()
            eps = 2.0 ** -8 if c.dtype == self.torch.bfloat16 else 2.0 ** -11
            largest = 448 * self.scale[layer, 1].max()
            tol = eps * np.abs(o[:n]) + (2.0 ** -11 + 2.0 ** -18) * mag[:n] + max(want["seq_lens"]) * 2.0 ** -25 * largest
            assert n == 0 or (np.abs(got[:n] - o[:n]) <= tol).all()
            assert n == 0 or np.abs(gz[:n] - z[:n]).max() <= 2.0 ** -15
        check_scores(self.logits.double().cpu().numpy(), [host(self.lp).astype(float), host(self.ent).astype(float), host(self.z).astype(float),
                                                          host(self.ids), host(self.top).astype(float)], host(self.tokens), TOP)
        self.context = [int(x) for x in want["seq_lens"]]
        assert self.backend.device_status() == 0

    def release(self, finished):
        self.c.release(finished)
        for r, f in enumerate(finished):
            if f:
                n = -(-self.context[r] // self.c.block_size)
                self.free[self.count:self.count + n] = self.table[r, :n]
                self.table[r, :n] = -1
                self.count, self.context[r] = self.count + n, 0
        self.torch.cuda.synchronize()
        assert int(self.c.free_count) == self.count
        assert np.array_equal(self.c.free_blocks.cpu().numpy()[:self.count], self.free[:self.count])


# new tokens of each step; a step may be followed by requests that finish
STEPS = [([37, 1, 0, 5], None), ([1, 1, 70, 1], None), ([1, 1, 1, 1], [0, 1, 0, 0]), ([1, 40, 1, 0], None), ([0, 0, 0, 0], [1, 0, 1, 0]), ([64, 1, 1, 1], None),
         ([1, 1, 17, 1], None)]


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("kind, bs, group, kv_heads, dim", [("bfloat16", 16, 4, 2, 128), ("float16", 32, 1, 3, 64), ("bfloat16", 64, 8, 1, 64), ("float16", 128, 3, 2, 128)])
def test_steps_of_a_server(backend, captured, kind, bs, group, kv_heads, dim):
    import torch
    s = Server(backend, getattr(torch, kind), 4, 24, bs, 12 if bs == 16 else 4, 80, group, kv_heads, dim, 80, seed=bs + group)
    stream = torch.cuda.Stream()
    graph = None
    if captured:
        s.feed([0, 0, 0, 0])
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            s.device_step()                                           # outside the capture first: an empty step
        torch.cuda.synchronize()
        s.check([0, 0, 0, 0])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            s.device_step()
    for new, finished in STEPS:
        s.feed(new)
        torch.cuda.synchronize()
        if graph is not None:
            graph.replay()
        else:
            with torch.cuda.stream(stream):
                s.device_step()
        torch.cuda.synchronize()
        assert s.c.status()[0] == sum(new)
        s.check(new)
        if finished:
            s.release(finished)


def test_a_step_that_the_pool_cannot_hold_changes_nothing(backend):
    import torch
    s = Server(backend, torch.bfloat16, 2, 5, 16, 8, 80, 2, 1, 64, 80, seed=3)
    s.feed([40, 20])
    s.device_step()
    s.check([40, 20])
    s.feed([1, 13])                                                   # one block too many
    before = [t.clone() for t in (s.c.k_cache, s.c.v_cache, s.c.k_scale, s.c.block_table, s.c.free_count, s.c.context_lens)]
    s.device_step()
    with pytest.raises(backend.BackendError, match="too few free blocks .1 missing"):
        s.c.status()
    for a, b in zip(before, (s.c.k_cache, s.c.v_cache, s.c.k_scale, s.c.block_table, s.c.free_count, s.c.context_lens)):
        assert torch.equal(a, b)
    assert (s.out == 7.0).all() and (s.lse == 7.0).all()
    s.release([1, 0])
    s.feed([2, 13])
    s.device_step()
    s.check([2, 13])


def test_queries_without_a_row_are_left_out(backend):
    """A step of 30 and 20 tokens whose queries stop at row 33: those of the rows that are there are unchanged, bit for bit."""
    import torch
    s = Server(backend, torch.bfloat16, 2, 8, 16, 4, 64, 4, 1, 64, 64, seed=4)
    s.feed([30, 20])
    s.device_step()
    s.check([30, 20])
    q = s.qkv[0][:33, :4 * 64].contiguous()
    for most in (None, 64, 30):
        out = s.c.attend(0, q, max_query=most)
        torch.cuda.synchronize()
        assert torch.equal(out, s.out[0][:33])
    assert backend.device_status() == 0


@pytest.mark.parametrize("new", [1, 3, 40])
def test_two_attentions_at_once_with_a_workspace_each(backend, new):
    """Two caches attended from two streams without waiting for one another give what each gives alone, bit for bit."""
    import torch
    servers = [Server(backend, torch.bfloat16, 4, 64, 32, 16, 200, 4, 2, 128, 100, seed=5 + i) for i in range(2)]
    for s in servers:
        for n in (50, 45, 49, new):
            s.feed([n] * 4)
            s.device_step()
    torch.cuda.synchronize()
    q = [s.qkv[0][:4 * new, :8 * 128] for s in servers]
    alone = []
    for s, x in zip(servers, q):
        alone.append(s.c.attend(0, x))
        torch.cuda.synchronize()
    outs = [[torch.empty_like(a) for _ in range(20)] for a in alone]
    streams = [torch.cuda.Stream() for _ in servers]
    torch.cuda.synchronize()
    for i in range(20):
        for j, s in enumerate(servers):
            with torch.cuda.stream(streams[j]):
                s.c.attend(0, q[j], out=outs[j][i])
    torch.cuda.synchronize()
    for a, some in zip(alone, outs):
        for o in some:
            assert torch.equal(o, a)
    assert backend.device_status() == 0


def test_two_graphs_share_a_workspace(backend):
    """A captured step of single tokens and one of chunks on the same cache, replayed in turn, give what eager calls give."""
    import torch
    s = Server(backend, torch.float16, 3, 64, 16, 20, 300, 4, 2, 128, 150, seed=9)
    for new in ([140, 90, 60], [1, 1, 1]):
        s.feed(new)
        s.device_step()
    q = s.qkv[1][:3, :8 * 128].contiguous()
    eager, eager_all = s.c.attend(1, q, max_query=1), s.c.attend(1, q)
    torch.cuda.synchronize()
    assert torch.equal(eager, eager_all)                              # with and without room for chunks
    graphs, outs = [], [torch.zeros_like(eager) for _ in range(2)]
    for out, most in zip(outs, (1, None)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s.c.attend(1, q, out=out, max_query=most)
        graphs.append(g)
    for _ in range(5):
        for g, out in zip(graphs, outs):
            out.zero_()
            g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], eager) and torch.equal(outs[1], eager)
    assert backend.device_status() == 0
