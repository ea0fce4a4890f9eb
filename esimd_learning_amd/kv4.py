"""The 4-bit paged key/value cache of a stack of decoder layers.

    kv = KV4Cache(layers, num_blocks, n_kv, head_dim, requests, tokens, max_len)
    each step:
      kv.advance(q_lens)                    esimd_kv_block_tables: room, slots and
                                            positions of the step's new tokens, by
                                            rows as cu_q says
      per layer i: kv.layers[i].attend(q, k, v, out)
                                            esimd_kv4_cache_write, then
                                            esimd_kv4_attention over old and new
                                            tokens

``forward`` and ``capture_forward`` (layer.py) call them with ``kv=``.  All
layers share the block tables; each has a cache of its own.  The state lives
on the device and is updated in place, so a step is launches alone and a
captured one continues from where the last replay stopped: a decode loop
replays ONE graph and never copies lengths or tables to the host.
"""

import torch


class KV4Layer:
    """One layer's cache.  ``scale`` of the scores (None: head_dim ** -0.5) and
    ``window`` (0: every earlier token) can be set by layer."""

    def __init__(self, owner, cache):
        self.owner, self.cache = owner, cache
        self.scale, self.window = None, 0

    def write(self, k, v):
        """Quantise the step's rows k, v into their slots."""
        self.owner.ops.esimd_kv4_cache_write(k, v, self.cache, self.owner.slot_mapping)

    def attend(self, q, k, v, out):
        """Store the step's k and v rows; out = causal attention of q over the cache.

        Rows behind the step's last token are padding: not stored, and left as
        they were in out.  So are a refused request's rows where they stay
        (``fixed_rows`` of advance), but for out, which holds nothing of use."""
        o = self.owner
        self.write(k, v)
        o.ops.esimd_kv4_attention(q, self.cache, o.block_tables, o.lens, o.cu_q, out,
                                  o.head_dim ** -0.5 if self.scale is None else self.scale,
                                  o.max_q_len, o.max_kv_len, self.window)

    def read(self, slots, dtype=torch.float16):
        """(k, v), [len(slots), n_kv, head_dim], as the cache holds them."""
        o = self.owner
        k = torch.empty(slots.numel(), o.n_kv, o.head_dim, dtype=dtype, device=self.cache.device)
        v = torch.empty_like(k)
        o.ops.esimd_kv4_cache_read(self.cache, slots, k, v)
        return k, v


class KV4Cache:
    """num_blocks blocks of block_size tokens for each of ``layers`` layers,
    shared by up to ``requests`` requests of at most max_len tokens; a step
    brings up to ``tokens`` new ones, of all requests together."""

    def __init__(self, layers, num_blocks, n_kv, head_dim, requests, tokens, max_len, block_size=32, device="cuda:0"):
        from . import ops as _load_ops
        self.ops = _load_ops()
        self.n_kv, self.head_dim, self.block_size, self.requests, self.tokens = n_kv, head_dim, block_size, requests, tokens
        i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=device)  # noqa: E731
        self.layers = [KV4Layer(self, self.ops.kv4_cache(num_blocks, n_kv, block_size, head_dim, device))
                       for _ in range(layers)]
        self.free_ring, self.ring_state = self.ops.kv_free_ring(num_blocks, device)
        self.block_tables = i32(requests, -(-max_len // block_size))
        self.lens = i32(requests)                     # cached tokens, the last step's included
        self.keep_all = torch.full((requests,), 2 ** 31 - 1, dtype=torch.int32, device=device)
        self.cu_q, self.status = i32(requests + 1), i32(requests)
        self.slot_mapping = torch.full((tokens,), -1, dtype=torch.int64, device=device)
        self.positions = torch.zeros(tokens, dtype=torch.int64, device=device)
        self.max_q_len = self.max_kv_len = 0

    def advance(self, q_lens, keep_lens=None, max_q_len=0, max_kv_len=0, fixed_rows=False):
        """Begin a step: q_lens [requests] int32 new tokens of each request, whose
        rows stand one request after another; positions, slots, tables and lens
        follow.

        A request that gets no room has no token in the step.  Its rows are closed
        up: request r's are cu_q[r] .. cu_q[r + 1] - 1, known after the call.  With
        ``fixed_rows`` they stay, as padding, and everyone's rows are where q_lens
        puts them: for a caller that lays out its rows without reading status or
        cu_q back, as around a captured step.

        keep_lens [requests] int32: how many of its cached tokens each request
        keeps (None, or beyond its length: all) -- fewer after rejected drafts, 0
        for one that ended.  status [requests] says afterwards which request got
        no room (see esimd_kv_block_tables).  max_q_len and max_kv_len, bounds of
        the step's new and cached tokens of one request (0: not known), let the
        attention choose its kernels without looking; wrong ones cost only time."""
        self.ops.esimd_kv_block_tables(self.lens, self.keep_all if keep_lens is None else keep_lens, q_lens,
                                       self.block_size, self.free_ring, self.ring_state, self.block_tables, self.lens,
                                       self.ring_state, self.cu_q, self.slot_mapping, self.positions, self.status,
                                       fixed_rows)
        self.max_q_len, self.max_kv_len = max_q_len, max_kv_len

    def slots(self, request, start, count):
        """int64 [count]: the slots of tokens start .. start + count - 1 of a request."""
        p = torch.arange(start, start + count, device=self.lens.device)
        return self.block_tables[request].long()[p // self.block_size] * self.block_size + p % self.block_size
