"""Host side of the 8-bit paged key/value cache: the pool, the tables and one serving step's calls.

    cache = PagedKvCache(torch, requests=64, num_blocks=8192, block_size=16, max_blocks=512, max_tokens=4096,
                         heads=32, kv_heads=8, head_dim=128, dtype=torch.bfloat16, layers=32)
    cache.plan(new_lens)                       # block tables and slots of this step's tokens
    for layer in range(32):
        cache.write(layer, k, v)               # quantise the step's keys and values into their slots
        o = cache.attend(layer, q)             # every request's queries over its own tokens
    cache.advance()                            # the step's tokens become context
    cache.release(finished)                    # finished requests give their blocks back

Everything that a step decides is decided on the device (lengths, tables, free list), nothing synchronises, and the arrays
never move: plan .. advance can be captured as one CUDA graph and replayed after new_lens has been filled again.  Steps follow
one another: all of a cache's calls go to one stream (or to streams that wait for one another), for they share its tables and
its workspace, and between a plan and its advance the tables belong to that step.  max_query (the constructor's, or attend's
for one call) bounds the new tokens of a request; rows of a request beyond it are left undone, and a tight bound spares
launches.  The compute
is the C-ABI library (include/pyc_b200.h); torch holds the buffers.  PyC has no cache and no ragged batch.
"""
from . import abi, backend

RESULT_ERRORS = {1: "a negative length", 2: "a request longer than its table row", 4: "more new tokens than max_tokens",
                 8: "too few free blocks", 16: "a block id outside the pool"}


class PagedKvCache:
    def __init__(self, torch, requests, num_blocks, block_size, max_blocks, max_tokens, heads, kv_heads, head_dim, dtype, layers=1,
                 max_query=None, device=None):
        self.torch = torch
        self.device = torch.device(device if device is not None else "cuda")
        if self.device.index is None and self.device.type == "cuda":
            self.device = torch.device("cuda", torch.cuda.current_device())
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"dtype {dtype}: queries, keys and values are bfloat16 or float16")
        if block_size not in (16, 32, 64, 128) or head_dim not in (64, 128):
            raise ValueError(f"block_size {block_size} must be 16, 32, 64 or 128 and head_dim {head_dim} 64 or 128")
        if heads % kv_heads:
            raise ValueError(f"{heads} heads do not split over {kv_heads} key heads")
        self.dtype, self._kind = dtype, abi.DTYPE_BF16 if dtype == torch.bfloat16 else abi.DTYPE_F16
        self.requests, self.num_blocks, self.block_size, self.max_blocks = requests, num_blocks, block_size, max_blocks
        self.max_tokens, self.max_query = max_tokens, min(max_query or max_tokens, max_tokens)
        self.heads, self.kv_heads, self.head_dim, self.layers = heads, kv_heads, head_dim, layers
        self._planned = False                                       # between plan and advance

        def ints(*shape, fill=0, kind=torch.int32):
            return torch.full(shape, fill, dtype=kind, device=self.device)

        pool = (layers, num_blocks, kv_heads, block_size, head_dim)
        self.k_cache = torch.zeros(pool, dtype=torch.uint8, device=self.device)
        self.v_cache = torch.zeros(pool, dtype=torch.uint8, device=self.device)
        self.k_scale = torch.ones(pool[:3], dtype=torch.float32, device=self.device)
        self.v_scale = torch.ones(pool[:3], dtype=torch.float32, device=self.device)
        self.free_blocks = torch.arange(num_blocks, dtype=torch.int32, device=self.device)
        self.free_count = ints(1, fill=num_blocks)
        self.block_table = ints(requests, max_blocks, fill=-1)
        self.context_lens, self.new_lens, self.seq_lens = ints(requests), ints(requests), ints(requests)
        self.query_start = ints(requests + 1)
        self.slot_map, self.positions = ints(max_tokens, fill=-1, kind=torch.int64), ints(max_tokens)
        self.token_request, self.result = ints(max_tokens, fill=-1), ints(4)
        self.workspace = torch.zeros(backend.paged_attention_workspace_bytes(requests, self.max_query, heads, kv_heads, head_dim),
                                     dtype=torch.uint8, device=self.device)

    def _stream(self):
        if self.device.index != self.torch.cuda.current_device():
            raise ValueError(f"the cache lives on {self.device}, the current device is cuda:{self.torch.cuda.current_device()}")
        return self.torch.cuda.current_stream().cuda_stream

    def _rows(self, name, x, width):
        """`x` as rows of `width` values: [tokens, heads, head_dim] or [tokens, heads * head_dim], any row stride."""
        if x.device != self.device or x.dtype != self.dtype:
            raise ValueError(f"{name}: {x.dtype} on {x.device}, the cache wants {self.dtype} on {self.device}")
        if x.dim() == 3 and tuple(x.shape[1:]) == (width // self.head_dim, self.head_dim):
            if x.stride(2) != 1 or (x.shape[1] > 1 and x.stride(1) != self.head_dim):
                raise ValueError(f"{name}: heads must lie next to one another (strides {x.stride()})")
        elif x.dim() != 2 or x.shape[1] != width or (width > 1 and x.stride(1) != 1):
            raise ValueError(f"{name}: shape {tuple(x.shape)} is not [tokens, {width // self.head_dim}, {self.head_dim}] or [tokens, {width}]")
        if not 1 <= x.shape[0] <= self.max_tokens:
            raise ValueError(f"{name}: {x.shape[0]} rows, max_tokens is {self.max_tokens}")
        if x.shape[0] > 1 and (x.stride(0) < width or x.stride(0) % 8):
            raise ValueError(f"{name}: rows {x.stride(0)} values apart, expected a multiple of 8 of at least {width}")
        return x.shape[0], (x.stride(0) if x.shape[0] > 1 else width)

    def plan(self, new_lens=None):
        """Tables and slots for a step that adds new_lens[r] tokens to request r (a device tensor, or a list; None: self.new_lens
        as it is).  Check `status()` after it wherever the pool may run out; a step that could not be planned has no tokens, and
        after `status()` has raised for it another one may be planned."""
        if self._planned:
            raise RuntimeError("plan: the step before has not been advanced (its blocks would be lost)")
        if new_lens is not None:
            x = self.torch.as_tensor(new_lens, dtype=self.torch.int32)
            if tuple(x.shape) != (self.requests,):
                raise ValueError(f"new_lens: shape {tuple(x.shape)}, expected ({self.requests},)")
            self.new_lens.copy_(x, non_blocking=True)
        backend.kv_plan(self.requests, self.block_size, self.max_blocks, self.max_tokens, self.num_blocks, self.context_lens.data_ptr(),
                        self.new_lens.data_ptr(), self.free_blocks.data_ptr(), self.free_count.data_ptr(), self.block_table.data_ptr(),
                        self.query_start.data_ptr(), self.seq_lens.data_ptr(), self.slot_map.data_ptr(), self.positions.data_ptr(),
                        self.token_request.data_ptr(), self.result.data_ptr(), stream=self._stream())
        self._planned = True

    def status(self):
        """(tokens, blocks taken) of the last plan; synchronises.  Raises when it could not be planned."""
        code, tokens, taken, missing = self.result.tolist()
        if code:
            if code & 15:
                self._planned = False                               # nothing was handed out
            what = ", ".join(text for bit, text in RESULT_ERRORS.items() if code & bit)
            raise backend.BackendError(f"kv plan: {what}" + (f" ({missing} missing)" if missing else ""))
        return tokens, taken

    def write(self, layer, k, v):
        """Quantise the step's keys and values (row t: token t of the plan; rows behind the last token are skipped)."""
        rows, ks = self._rows("k", k, self.kv_heads * self.head_dim)
        rows_v, vs = self._rows("v", v, self.kv_heads * self.head_dim)
        if rows != rows_v:
            raise ValueError(f"{rows} rows of keys, {rows_v} of values")
        backend.kv_write(self._kind, rows, self.kv_heads, self.head_dim, self.block_size, self.num_blocks, k.data_ptr(), v.data_ptr(),
                         self.slot_map.data_ptr(), self.k_cache[layer].data_ptr(), self.v_cache[layer].data_ptr(),
                         self.k_scale[layer].data_ptr(), self.v_scale[layer].data_ptr(), k_stride=ks, v_stride=vs, stream=self._stream())

    def attend(self, layer, q, out=None, lse=None, scale=None, causal=True, max_query=None):
        """Attention of the step's queries over the cache.  Rows of `out` behind the last token are left as they were (zero when
        it is made here); tokens of the step for which `q` has no row are left out."""
        most = self.max_query if max_query is None else max_query
        if not 1 <= most <= self.max_query:
            raise ValueError(f"max_query {most} is not in 1 .. {self.max_query}")
        rows, qs = self._rows("q", q, self.heads * self.head_dim)
        if out is None:
            out = self.torch.zeros((rows, self.heads, self.head_dim), dtype=self.dtype, device=self.device)
        out_rows, os_ = self._rows("out", out, self.heads * self.head_dim)
        if out_rows != rows:
            raise ValueError(f"{rows} rows of queries, {out_rows} of out")
        if lse is not None and (tuple(lse.shape) != (rows, self.heads) or lse.dtype != self.torch.float32 or not lse.is_contiguous() or
                                lse.device != self.device):
            raise ValueError(f"lse must be contiguous float32 [{rows}, {self.heads}] on {self.device}")
        backend.paged_attention(self._kind, self.requests, most, self.heads, self.kv_heads, self.head_dim, self.block_size,
                                self.num_blocks, self.max_blocks, q.data_ptr(), self.k_cache[layer].data_ptr(),
                                self.v_cache[layer].data_ptr(), self.k_scale[layer].data_ptr(), self.v_scale[layer].data_ptr(),
                                self.block_table.data_ptr(), self.query_start.data_ptr(), self.seq_lens.data_ptr(), out.data_ptr(),
                                scale if scale is not None else self.head_dim ** -0.5, causal, self.workspace.data_ptr(),
                                self.workspace.numel(), lse=lse.data_ptr() if lse is not None else None, q_stride=qs, out_stride=os_,
                                rows=rows, stream=self._stream())
        return out

    def advance(self):
        """The step's tokens become context of the next one."""
        self.context_lens.copy_(self.seq_lens)
        self._planned = False

    def release(self, finished):
        """Give back the blocks of the requests with finished[r] != 0 (a device tensor or a list); their length becomes 0.
        Between steps only: after advance, before the next plan."""
        if self._planned:
            raise RuntimeError("release: the planned step has not been advanced")
        x = self.torch.as_tensor(finished).to(device=self.device, dtype=self.torch.int32).contiguous()
        if tuple(x.shape) != (self.requests,):
            raise ValueError(f"finished: shape {tuple(x.shape)}, expected ({self.requests},)")
        backend.kv_release(self.requests, self.block_size, self.max_blocks, self.num_blocks, x.data_ptr(), self.context_lens.data_ptr(),
                           self.block_table.data_ptr(), self.free_blocks.data_ptr(), self.free_count.data_ptr(), stream=self._stream())
