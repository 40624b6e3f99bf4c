"""PagedKVCache: the cache of a serving batch, whose requests have lengths of their own and come and go.  Beside KVCompCache, which compresses a
rectangular batch: here tokens stay fp16 or bf16, or have 8-bit codes and a scale for each row (codes="int8" or "e4m3"), in pages that requests take from a common pool and give back.

    cache = PagedKVCache(requests, pages, layer_num, kv_heads, head_dim, frequencies=..., ...)
    plan = cache.begin(new, tokens)                        # once a step: new[b] tokens of request b, packed one request behind the other
    for layer in range(layer_num):
        q = cache.append(q, k, v, layer)                   # q, k rotated, k and v into their pages
        out = cache.attend(q, layer)                       # a decode step: one token per request, or none; row by row as the step is packed
    cache.release(done)                                    # the pages of finished requests go back

A prompt in chunks attends with the rows that its cache holds so far (slots, rows).  Requests that continue a common prompt are said to follow the request that holds it (follow): its
tokens come before theirs, and attend reads them once for all.

Everything is launched and nothing waited for or asked of the device: a step of at most one token per request can be captured into a CUDA graph and
replayed, with the lengths, the tables and the free list going on from replay to replay (new[b] may be 0 in any of them); nothing has to be called
before it.  append and attend go by the last begin, captured or not.  Layers may be attended on streams of their own: each keeps a workspace of 15
to 45 MB (with followers 30 to 100), and so does each graph.  Streams are ordered by the caller: begin, follow and release change what the attention reads, and may run only behind all
of it (Stream.wait_stream).  (The prompt's own attention is the model's: its keys and values are in hand there.)  No gradient goes through a cache;
tensors that a call writes are known to autograd as changed."""
import math

import torch

from .. import _lib, ops
from .._lib import KvcError


CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


class PagedKVCache:
    codes = key_scales = value_scales = None                         # (of a cache that was pickled without)
    parents = shared = prefixes = None                               # whom requests follow, how many tokens of it, and ops.prefix_plan's answer

    def __init__(self, requests, pages, layer_num, kv_heads, head_dim, page_size=64, max_tokens=None, dtype=torch.float16, device="cuda",
                 frequencies=None, layout="half", factor=1.0, window=0, codes=None):
        """A pool of `pages` pages of `page_size` tokens for `requests` requests of up to max_tokens tokens each (all of the pool where it is not given).  head_dim: 64, 96, 128 or
        256, what the attention takes (ops.rotary_paged_store alone takes any).
        frequencies, layout, factor: the rotation (utils.rotary.frequencies; None: keys and queries come rotated).  window > 0: attention over the
        last `window` tokens.
        codes: None, or "int8" or "e4m3": tokens are held in 8 bits, with a scale in 32 for each token's row of a KV head (ops.rotary_paged_store); `dtype` is what queries, new rows and
        results have."""
        if min(requests, pages, layer_num, kv_heads, head_dim, page_size) <= 0:
            raise KvcError("PagedKVCache: sizes must be positive")
        if head_dim not in ops.PAGED_HEADS:
            raise KvcError("PagedKVCache: heads of 64, 96, 128 or 256 channels, got %d" % head_dim)
        if dtype not in (torch.float16, torch.bfloat16):
            raise KvcError("PagedKVCache: fp16 or bf16, got %s" % dtype)
        if codes is not None and codes not in CODES:
            raise KvcError("PagedKVCache: codes are None, 'int8' or 'e4m3', got %r" % (codes,))
        device = torch.empty(0, device=device).device
        if device.type != "cuda":
            raise KvcError("PagedKVCache: kvcomp_b200 has no CPU path")
        self.requests, self.pages, self.layer_num, self.kv_heads, self.head_dim, self.page_size = requests, pages, layer_num, kv_heads, head_dim, page_size
        self.max_tokens = pages * page_size if max_tokens is None else max_tokens
        self.dtype, self.device, self.layout, self.factor, self.window = dtype, device, layout, float(factor), window
        self.frequencies = None if frequencies is None else frequencies.to(device=device, dtype=torch.float64)
        # (zeros: rows that no token was written to are never read, but a pool can be saved and compared)
        self.codes = codes
        self.keys, self.values = (torch.zeros(layer_num, pages, page_size, kv_heads, head_dim, dtype=CODES.get(codes, dtype), device=device) for _ in range(2))
        self.key_scales, self.value_scales = (torch.zeros(layer_num, pages, kv_heads, page_size, device=device) if codes else None for _ in range(2))
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
        if self.prefixes is not None:
            ops.page_shift(plan.starts, self.shared, plan.positions)
        return self.plan

    def follow(self, parents, shared=None):
        """From here on request b's tokens come behind the first shared[b] tokens of request parents[b] (int32[requests] on the device; below 0: of none): their positions go on from there
        (begin), and attend covers both.  shared None: all tokens that the parent has now.  Requests that follow the same tokens are attended to together, and these are read once.  To be said
        before a follower's first tokens; for all requests at once, those that followed before included.  Who is followed brings no more tokens, stays until its followers have ended, and
        follows no one; a follower that ends (release) follows no one any more; a parent that is no request, or the request itself, is none (reported: check).  Steps that are captured behind
        the first call go by the last one, captured or not.  Heads of 64, 96 or 128 channels, no window, no codes.  Pays from some 260000 on of followers x shared tokens x KV heads; one
        follower alone costs more than the same tokens of its own."""
        if self.window or self.codes or self.head_dim not in ops.SHARED_HEADS:
            raise KvcError("PagedKVCache.follow: heads of 64, 96 or 128 channels, no window and no codes")
        if not isinstance(parents, torch.Tensor) or parents.dtype != torch.int32 or tuple(parents.shape) != (self.requests,) or parents.device != self.device:
            raise KvcError("parents must be int32[%d] on %s" % (self.requests, self.device))
        if shared is None:
            shared = self.lengths[parents.clamp(0, self.requests - 1).long()]
        elif not isinstance(shared, torch.Tensor) or shared.dtype != torch.int32 or tuple(shared.shape) != (self.requests,) or shared.device != self.device:
            raise KvcError("shared must be int32[%d] on %s" % (self.requests, self.device))
        if self.prefixes is None and _lib.torch_calls().stream_of(self.device.index)[1]:         # (the capture of the cache's own device)
            raise KvcError("PagedKVCache.follow: the first call makes what all steps go by, and must not be captured")
        # whom nobody can follow is followed by none, in the plan, in positions and in lengths alike, and is reported (check raises)
        valid = (parents >= 0) & (parents < self.requests) & (parents != torch.arange(self.requests, dtype=torch.int32, device=self.device)) & (shared >= 0)
        none = ((parents >= 0) & ~valid).any().int() * _lib.FLAG_BAD_LENGTH
        parents, shared = torch.where(valid, parents, -1), torch.where(valid, shared, 0)
        if self.prefixes is None:                                    # (a plan that cannot be made leaves the cache as it was)
            self.prefixes, self.parents, self.shared = ops.prefix_plan(parents, shared, status=self.status), parents, shared
        else:
            self.parents.copy_(parents)
            self.shared.copy_(shared)
            ops.prefix_plan(self.parents, self.shared, out=self.prefixes, status=self.status)
        self.status.bitwise_or_(none)

    def slots(self, tokens):
        """Where the tokens that requests have lie, request by request: (slots int32[tokens], starts int32[requests + 1]), for rows.  tokens: their number, as the host knows it; slots behind them
        are -1.  A prefix that a request follows is its parent's."""
        return ops.page_slots(self.table, self.lengths, self.page_size, tokens, status=self.status)

    def rows(self, layer_idx, slots):
        """Keys (rotated) and values of a layer's slots, [N, Hkv, D] each, as attend reads them.  For a prompt in chunks, behind append: begin, slots, and in each layer append, rows and the model's own
        attention."""
        return ops.paged_rows(self.keys[layer_idx], self.values[layer_idx], slots, dtype=self.dtype, status=self.status, **self._scales(layer_idx))

    def _scales(self, layer_idx):
        return dict(kscales=self.key_scales[layer_idx], vscales=self.value_scales[layer_idx]) if self.codes else {}

    def append(self, query_states, key_states, value_states, layer_idx):
        """The step's rows of a layer: queries [tokens, Hq, D] (or None), keys and values [tokens, Hkv, D].  Keys go rotated into their pages, values as they are;
        returns the rotated queries."""
        if self.plan is None:
            raise KvcError("append before any begin")
        return ops.rotary_paged_store(query_states, key_states, value_states, self.plan.positions, self.plan.slots, self.frequencies, self.keys[layer_idx],
                                      self.values[layer_idx], layout=self.layout, factor=self.factor, status=self.status, **self._scales(layer_idx))

    def attend(self, query_states, layer_idx, scaling=None, return_lse=False, by_request=False):
        """The step's rows as append returns them, at most one of a request: [tokens, Hq, D] -> [tokens, Hq, D], each over the tokens that its request has.  Rows behind the last
        are 0 (a captured step has as many as there are requests, whatever they bring), and so are those of a request that brought more than one (reported: check).
        by_request, or as many rows as requests where the step had another number: row b is request b's, whatever it brought; 0 for one without tokens."""
        rows, starts = query_states.shape[0], None
        if not by_request and self.plan is not None and rows == self.plan.slots.shape[0]:
            if rows > self.requests:
                raise KvcError("attend: one token per request, got %d rows of %d requests" % (rows, self.requests))
            starts = self.plan.starts
        scaling = 1.0 / math.sqrt(self.head_dim) if scaling is None else scaling
        if self.prefixes is not None:
            return ops.paged_attn_shared(query_states, self.keys[layer_idx], self.values[layer_idx], self.table, self.lengths, self.prefixes, scaling, return_lse=return_lse,
                                         workspace=self._workspace(query_states.shape[1], True), status=self.status, starts=starts)
        return ops.paged_attn(query_states, self.keys[layer_idx], self.values[layer_idx], self.table, self.lengths, scaling, window=self.window, return_lse=return_lse,
                              workspace=self._workspace(query_states.shape[1]), status=self.status, starts=starts, **self._scales(layer_idx))

    def _workspace(self, heads, prefixes=False):
        """The attention's workspace, cleared, for the current stream: calls on streams of their own may run at once.  A capture has its own too, cleared by the
        graph where the capture's first call lies (a launch more for a graph): an eager call or another graph neither finds it uncleared nor in use."""
        stream, capture = _lib.torch_calls().stream_of(self.device.index)
        key = (heads, stream, capture, prefixes)
        workspace = self._workspaces.get(key)
        if workspace is None:
            if capture:                                              # captures on this stream before are over: their memory is their graphs'
                self._workspaces = {key: w for key, w in self._workspaces.items() if key[1] != stream or key[2] in (0, capture)}
            make = ops.paged_attn_shared_workspace if prefixes else ops.paged_attn_workspace
            workspace = self._workspaces[key] = make(self.requests, heads, self.kv_heads, self.head_dim, self.device)
        return workspace

    def release(self, done):
        """The requests with done[b] (bool[requests], on the device) end: their pages go back, their lengths are 0."""
        ops.page_release(self.lengths, done, self.table, self.free, self.head, self.page_size, out=(self.lengths, self.head), status=self.status)
        if self.prefixes is not None:
            # those that ended follow no one; neither do those whose prefix has gone, which is reported (check raises)
            lost = (self.parents >= 0) & done[self.parents.clamp(min=0).long()]
            self.status.bitwise_or_((lost & ~done).any().int() * _lib.FLAG_BAD_LENGTH)
            self.parents.masked_fill_(lost | done, -1)
            self.shared.masked_fill_(lost | done, 0)
            ops.prefix_plan(self.parents, self.shared, out=self.prefixes, status=self.status)

    def check(self):
        """The conditions reported since the last check (_lib.FLAG_*; FLAG_NO_PAGES: a request was refused).  Raises where a page or a length was bad.
        Synchronises; nothing else here does."""
        flags = int(self.status.item())
        self.status.zero_()
        return ops.check_flags(flags, what="PagedKVCache")

    def get_seq_length(self, request=0):
        """Tokens of a request, those that it follows included (synchronises)."""
        return int(self.lengths[request].item()) + (0 if self.shared is None else int(self.shared[request].item()))
