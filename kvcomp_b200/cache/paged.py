"""PagedKVCache: the cache of a serving batch, whose requests have lengths of their own and come and go.  Beside KVCompCache, which compresses a
rectangular batch: here tokens stay fp16 or bf16, in pages that requests take from a common pool and give back.

    cache = PagedKVCache(requests, pages, layer_num, kv_heads, head_dim, frequencies=..., ...)
    plan = cache.begin(new, tokens)                        # once a step: new[b] tokens of request b, packed one request behind the other
    for layer in range(layer_num):
        q = cache.append(q, k, v, layer)                   # q, k rotated, k and v into their pages
        out = cache.attend(q, layer)                       # a decode step: one token per request, or none; row by row as the step is packed
    cache.release(done)                                    # the pages of finished requests go back

Everything is launched and nothing waited for or asked of the device: a step of at most one token per request can be captured into a CUDA graph and
replayed, with the lengths, the tables and the free list going on from replay to replay (new[b] may be 0 in any of them); nothing has to be called
before it.  append and attend go by the last begin, captured or not.  Layers may be attended on streams of their own: each keeps a workspace of 15
to 45 MB, and so does each graph.  Streams are ordered by the caller: begin and release change what the attention reads, and may run only behind all
of it (Stream.wait_stream).  (The prompt's own attention is the model's: its keys and values are in hand there.)  No gradient goes through a cache;
tensors that a call writes are known to autograd as changed."""
import math

import torch

from .. import _lib, ops
from .._lib import KvcError


class PagedKVCache:
    def __init__(self, requests, pages, layer_num, kv_heads, head_dim, page_size=64, max_tokens=None, dtype=torch.float16, device="cuda",
                 frequencies=None, layout="half", factor=1.0, window=0):
        """A pool of `pages` pages of `page_size` tokens for `requests` requests of up to max_tokens tokens each (all of the pool where it is not given).  head_dim: 64, 96, 128 or
        256, what the attention takes (ops.rotary_paged_store alone takes any).
        frequencies, layout, factor: the rotation (utils.rotary.frequencies; None: keys and queries come rotated).  window > 0: attention over the
        last `window` tokens."""
        if min(requests, pages, layer_num, kv_heads, head_dim, page_size) <= 0:
            raise KvcError("PagedKVCache: sizes must be positive")
        if head_dim not in ops.PAGED_HEADS:
            raise KvcError("PagedKVCache: heads of 64, 96, 128 or 256 channels, got %d" % head_dim)
        if dtype not in (torch.float16, torch.bfloat16):
            raise KvcError("PagedKVCache: fp16 or bf16, got %s" % dtype)
        device = torch.empty(0, device=device).device
        if device.type != "cuda":
            raise KvcError("PagedKVCache: kvcomp_b200 has no CPU path")
        self.requests, self.pages, self.layer_num, self.kv_heads, self.head_dim, self.page_size = requests, pages, layer_num, kv_heads, head_dim, page_size
        self.max_tokens = pages * page_size if max_tokens is None else max_tokens
        self.dtype, self.device, self.layout, self.factor, self.window = dtype, device, layout, float(factor), window
        self.frequencies = None if frequencies is None else frequencies.to(device=device, dtype=torch.float64)
        # (zeros: rows that no token was written to are never read, but a pool can be saved and compared)
        self.keys, self.values = (torch.zeros(layer_num, pages, page_size, kv_heads, head_dim, dtype=dtype, device=device) for _ in range(2))
        self.lengths = torch.zeros(requests, dtype=torch.int32, device=device)
        self.table = torch.full((requests, -(-self.max_tokens // page_size)), -1, dtype=torch.int32, device=device)
        self.free = torch.arange(pages, dtype=torch.int32, device=device)
        self.head = torch.zeros(1, dtype=torch.int32, device=device)
        self.status = ops.new_status(device)
        self.plan = None
        self._workspaces = {}

    def __getstate__(self):
        return {name: value for name, value in self.__dict__.items() if name != "_workspaces"}                           # (a copy makes its own)

    def __setstate__(self, state):
        self.__dict__.update(state, _workspaces={})
        self.__dict__.pop("_workspace", None)                        # (what it was once kept under)

    def begin(self, new, tokens):
        """A step that brings new[b] tokens (int32[requests], on the device) of each request, `tokens` rows in all.  Returns the plan (ops.PagePlan):
        slots, positions, the requests' first rows; taken[b] = -1 where request b was refused: its tokens have no slot and it keeps its length.  The
        cache's lengths, tables and free list are behind the step from here on."""
        plan = ops.PagePlan(self.lengths, self.head, *(torch.empty(n, dtype=torch.int32, device=self.device) for n in (self.requests + 1, self.requests, tokens, tokens)))
        self.plan = ops.page_plan(self.lengths, new, self.table, self.free, self.head, self.page_size, tokens, out=plan, status=self.status)
        return self.plan

    def append(self, query_states, key_states, value_states, layer_idx):
        """The step's rows of a layer: queries [tokens, Hq, D] (or None), keys and values [tokens, Hkv, D].  Keys go rotated into their pages, values as they are;
        returns the rotated queries."""
        if self.plan is None:
            raise KvcError("append before any begin")
        return ops.rotary_paged_store(query_states, key_states, value_states, self.plan.positions, self.plan.slots, self.frequencies, self.keys[layer_idx],
                                      self.values[layer_idx], layout=self.layout, factor=self.factor, status=self.status)

    def attend(self, query_states, layer_idx, scaling=None, return_lse=False, by_request=False):
        """The step's rows as append returns them, at most one of a request: [tokens, Hq, D] -> [tokens, Hq, D], each over the tokens that its request has.  Rows behind the last
        are 0 (a captured step has as many as there are requests, whatever they bring), and so are those of a request that brought more than one (reported: check).
        by_request, or as many rows as requests where the step had another number: row b is request b's, whatever it brought; 0 for one without tokens."""
        rows, starts = query_states.shape[0], None
        if not by_request and self.plan is not None and rows == self.plan.slots.shape[0]:
            if rows > self.requests:
                raise KvcError("attend: one token per request, got %d rows of %d requests" % (rows, self.requests))
            starts = self.plan.starts
        workspace = self._workspace(query_states.shape[1])
        return ops.paged_attn(query_states, self.keys[layer_idx], self.values[layer_idx], self.table, self.lengths,
                              1.0 / math.sqrt(self.head_dim) if scaling is None else scaling, window=self.window, return_lse=return_lse, workspace=workspace, status=self.status,
                              starts=starts)

    def _workspace(self, heads):
        """The attention's workspace, cleared, for the current stream: calls on streams of their own may run at once.  A capture has its own too, cleared by the
        graph where the capture's first call lies (a launch more for a graph): an eager call or another graph neither finds it uncleared nor in use."""
        stream, capture = _lib.torch_calls().stream_of(self.device.index)
        workspace = self._workspaces.get((heads, stream, capture))
        if workspace is None:
            if capture:                                              # captures on this stream before are over: their memory is their graphs'
                self._workspaces = {key: w for key, w in self._workspaces.items() if key[1] != stream or key[2] in (0, capture)}
            workspace = self._workspaces[heads, stream, capture] = ops.paged_attn_workspace(self.requests, heads, self.kv_heads, self.head_dim, self.device)
        return workspace

    def release(self, done):
        """The requests with done[b] (bool[requests], on the device) end: their pages go back, their lengths are 0."""
        ops.page_release(self.lengths, done, self.table, self.free, self.head, self.page_size, out=(self.lengths, self.head), status=self.status)

    def check(self):
        """The conditions reported since the last check (_lib.FLAG_*; FLAG_NO_PAGES: a request was refused).  Raises where a page or a length was bad.
        Synchronises; nothing else here does."""
        flags = int(self.status.item())
        self.status.zero_()
        return ops.check_flags(flags, what="PagedKVCache")

    def get_seq_length(self, request=0):
        """Tokens of a request (synchronises)."""
        return int(self.lengths[request].item())
