"""Performance cases of the 4-bit key/value cache: bookkeeping, writes, reads and attention on one GPU.

Four kinds of work, as a serving program calls them once a step and layer:

* ``tables``  from the requests' lengths: blocks taken from and returned to the free ring, block
              tables, slots and positions of the step's tokens;
* ``write``   quantise the step's k and v rows into the cache at their slots, and read back what
              the cache now holds for them;
* ``read``    cached rows by slot, as 16-bit values (a prefix that is handed on);
* ``attn``    attention of the step's query rows over the cached keys and values: one token a
              request, drafted tokens, prompt chunks, and batches of both.

The cache is uint8 ``[num_blocks, n_kv, block_size, head_dim + 8]``; one (block, head) holds, in
this order, the K codes ``[bs, hd / 2]`` (low nibble first), the V codes ``[bs / 4, hd / 4, 4, 2]``
(for each run of four values, four tokens side by side), then the K and the V parameters ``[bs]``
(bf16 step s, bf16 centre m) each.  A value is ``m + s (c - 7.5)``.

Heads and head sizes are those of the benchmark configurations (16 x 256, 32 / 8 x 128) and
generic ones.  Lengths are spread evenly in their logarithm between two bounds, the same ones for
every seed; values are N(0, 1), q twice that, so that a softmax has a few heavy keys.
"""

import math

import torch

own = False

DEV = "cuda"
IO = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _tables(r, lo, hi, q, bs, roll=0, new=0, io="fp16"):
    """r running requests of lo..hi cached tokens, up to q new tokens each, up to roll of the
    cached ones dropped; the last `new` requests start over (nothing kept)."""
    return {"kind": "tables", "r": r, "lo": lo, "hi": hi, "q": q, "bs": bs, "roll": roll, "new": new}


def _write(t, nk, hd, bs, io="fp16", run=0, pad=0):
    """t rows, `pad` more behind them that have no slot; slots in runs of `run` tokens of a request
    (0: every row another request's)."""
    return {"kind": "write", "t": t, "nk": nk, "hd": hd, "bs": bs, "io": io, "run": run, "pad": pad}


def _read(t, nk, hd, bs, io="fp16", run=0):
    return {"kind": "read", "t": t, "nk": nk, "hd": hd, "bs": bs, "io": io, "run": run, "pad": 0}


def _attn(r, lo, hi, q, nq, nk, hd, bs, io="fp16", window=0, chunks=0, chunk_q=0):
    """r requests of lo..hi cached tokens, the step's among them: q query tokens each, but
    chunk_q for the last `chunks` of them."""
    return {"kind": "attn", "r": r, "lo": lo, "hi": hi, "q": q, "nq": nq, "nk": nk, "hd": hd, "bs": bs, "io": io,
            "window": window, "chunks": chunks, "chunk_q": chunk_q}


def listed():
    return [
        # a decode step's bookkeeping for a few requests: launch latency
        dict(_tables(8, 100, 4000, 1, 16), name="tables_r8"),
        # a busy server: drafted tokens verified, some dropped again, prompts of new requests
        dict(_tables(256, 50, 16000, 37, 32, roll=5, new=12), name="tables_r256"),
        # k and v of a decode step, eight requests: launch latency
        dict(_write(8, 8, 128, 16, io="bf16"), name="write_t8"),
        # k and v of a prompt chunk, padded to the captured size
        dict(_write(8000, 8, 128, 32, run=1999, pad=192), name="write_t8000"),
        # a short prefix handed on, in bf16
        dict(_read(777, 16, 256, 16, io="bf16", run=259), name="read_t777"),
        # a long prefix handed on
        dict(_read(32768, 8, 128, 64, run=32768), name="read_t32768"),
        # one chat request being decoded, fp16
        dict(_attn(1, 700, 700, 1, 32, 8, 128, 16), name="attn_r1_700"),
        # one long document being decoded
        dict(_attn(1, 131071, 131071, 1, 32, 8, 128, 64, io="bf16"), name="attn_r1_131071"),
        # a decode batch of ragged requests (the benchmark's QKV layout)
        dict(_attn(64, 300, 16000, 1, 32, 8, 128, 32, io="bf16"), name="attn_r64_ragged"),
        # drafted tokens verified in the decoder layer's 16 heads of 256, sliding window
        dict(_attn(16, 900, 6000, 5, 16, 16, 256, 16, window=4096), name="attn_r16_draft"),
        # prompt chunks behind cached prefixes (the largest)
        dict(_attn(4, 1900, 4100, 1, 32, 8, 128, 32, chunks=4, chunk_q=1900), name="attn_prefill"),
        # a mixed step: decodes beside a prompt chunk
        dict(_attn(13, 250, 5000, 1, 16, 4, 64, 16, io="bf16", chunks=1, chunk_q=1000), name="attn_mixed"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choices(["tables", "write", "read", "attn"], [15, 15, 10, 60])[0]
    io, bs = rng.choice(["fp16", "bf16"]), rng.choice([16, 32, 64, 128])
    if kind == "tables":
        r, lo = _log_int(rng, 1, 512), _log_int(rng, 1, 500)
        return _tables(r, lo, _log_int(rng, lo, 16000), _log_int(rng, 1, 64), bs, roll=rng.choice([0, 3, 7]),
                       new=rng.randrange(1 + r // 8))
    hd = rng.choice([64, 128, 128, 256])
    nq = rng.choice([8, 16, 28, 32])
    nk = rng.choice([v for v in (1, 2, 4, 8, nq) if nq % v == 0])
    if kind != "attn":
        t = _log_int(rng, 1, 32768 if kind == "read" else 8192)
        while t * nk * hd > 2 ** 25:
            t = max(1, t // 2)
        run = rng.choice([0, 1 + t // 3, t])
        return _read(t, nk, hd, bs, io=io, run=run) if kind == "read" else \
            _write(t, nk, hd, bs, io=io, run=run, pad=rng.choice([0, 0, 1 + t // 50]))
    window = rng.choice([0, 0, 0, 1024, 4096])
    mode = rng.choice(["decode", "decode", "draft", "prefill", "mixed"])
    lo = _log_int(rng, 16, 4000)
    if mode in ("decode", "draft"):
        r, q = _log_int(rng, 1, 128), 1 if mode == "decode" else rng.randint(2, 8)
        hi = _log_int(rng, lo, 16000 if r > 4 else 131072)
        while r * hi * nk * (hd + 8) > 9e8 or r * hi * nq * q > 3e8:
            hi = max(lo, hi // 2) if hi > lo else hi
            r = max(1, r // 2)
        return _attn(r, lo, hi, q, nq, nk, hd, bs, io=io, window=window)
    r = rng.randint(1, 4) if mode == "prefill" else rng.randint(2, 16)
    chunk = _log_int(rng, 60, 1900)
    lo = max(lo, chunk if mode == "prefill" else 1)
    hi = max(lo, chunk, _log_int(rng, lo, 6000))
    while r * nq * chunk * hi * hd > 4 * 32 * 1900 * 3000 * 128 and r > 2:
        r -= 1
    while r * nq * chunk * hi * hd > 4 * 32 * 1900 * 3000 * 128:
        chunk, hi = max(1, chunk // 2), max(lo, hi // 2, chunk // 2)
        lo = min(lo, hi)
    return _attn(r, lo, hi, 1, nq, nk, hd, bs, io=io, window=window, chunks=r if mode == "prefill" else 1, chunk_q=chunk)


# ---- what a case holds, whatever its seed ------------------------------------

def _spread(n, lo, hi, least=1):
    """n lengths of lo..hi, even in their logarithm, in a mixed order, the longest last."""
    at = [math.fmod(0.5 + 0.6180339887498949 * i, 1.0) for i in range(n - 1)] + [1.0]
    return [max(least, int(round(lo * (hi / lo) ** f))) for f in at]


def _attn_lens(case):
    r, c = case["r"], case["chunks"]
    q = [case["chunk_q"] if i >= r - c else case["q"] for i in range(r)]
    return [max(n, m) for n, m in zip(_spread(r, case["lo"], case["hi"]), q)], q


def _table_lens(case):
    r, new = case["r"], case["new"]
    lens = _spread(r, case["lo"], case["hi"])
    q = [1 + (7 * i) % case["q"] for i in range(r)]
    keep = [0 if i >= r - new else max(0, n - (5 * i) % (case["roll"] + 1)) for i, n in enumerate(lens)]
    q = [case["q"] * 40 + 3 * i if i >= r - new else n for i, n in enumerate(q)]
    return lens, keep, q


def _blocks(n, bs):
    return -(-n // bs)


def _seen(case):
    """(query, key) pairs of one head, and the keys that a request's rows see together."""
    pairs, keys = 0, 0
    for n, q in zip(*_attn_lens(case)):
        w = case["window"] or n
        pairs += sum(min(w, n - q + 1 + i) for i in range(q))
        keys += min(n, w + q - 1)
    return pairs, keys


def work(case):
    if case["kind"] == "tables":
        lens, keep, q = _table_lens(case)
        moved = sum(abs(_blocks(n, case["bs"]) - _blocks(k + m, case["bs"])) for n, k, m in zip(lens, keep, q))
        return {"bytes": 24 * case["r"] + 8 * moved + 16 * sum(q), "flops": 0}
    nk, hd = case["nk"], case["hd"]
    if case["kind"] == "attn":
        pairs, keys = _seen(case)
        rows = sum(_attn_lens(case)[1])
        return {"bytes": keys * nk * (hd + 8) + 4 * rows * case["nq"] * hd, "flops": 4 * hd * case["nq"] * pairs}
    row = nk * (4 * hd + hd + 8) + 8
    if case["kind"] == "read":
        return {"bytes": case["t"] * row, "flops": 0}
    # the rows in, the cache's bytes written, and the same bytes and rows of the reading back
    return {"bytes": 2 * case["t"] * row, "flops": 0}


# ---- the cache, in plain torch -------------------------------------------------

def _quantise(x):
    """fp32 rows [..., hd] -> codes (uint8), step and centre (bf16 values in fp32)."""
    lo, hi = x.amin(-1), x.amax(-1)
    ok = torch.isfinite(lo) & torch.isfinite(hi)
    m = (0.5 * lo + 0.5 * hi).bfloat16().float()
    s = (torch.maximum(hi - m, m - lo) / 7.5).bfloat16().float()
    s = torch.where(ok & (s >= 2.0 ** -100), s, torch.zeros_like(s))
    m = torch.where(ok, m, torch.full_like(m, math.nan))
    by = torch.where(s > 0, s, torch.ones_like(s))
    c = ((x - m[..., None]) / by[..., None] + 7.5).round().clamp(0, 15)
    return torch.where((s > 0)[..., None], c, torch.full_like(c, 8.0)).to(torch.uint8), s, m


def _nibbles(c):
    return c[..., 0::2] | (c[..., 1::2] << 4)


def _codes(b):
    return torch.stack([b & 15, b >> 4], dim=-1).flatten(-2)


def _params(s, m):
    return torch.stack([s.bfloat16(), m.bfloat16()], dim=-1).view(torch.uint8)


def _parts(cache, hd):
    """Views of the cache: K codes [nb, nk, bs, hd/2], V codes [nb, nk, bs/4, hd/4, 4, 2], K and V parameters [nb, nk, bs, 4]."""
    nb, nk, bs = cache.shape[:3]
    flat, half = cache.view(nb, nk, bs * (hd + 8)), bs * hd // 2
    return (flat[..., :half].view(nb, nk, bs, hd // 2), flat[..., half:2 * half].view(nb, nk, bs // 4, hd // 4, 4, 2),
            flat[..., 2 * half:2 * half + 4 * bs].view(nb, nk, bs, 4), flat[..., 2 * half + 4 * bs:].view(nb, nk, bs, 4))


def _values(codes, par):
    p = par.contiguous().view(torch.bfloat16).float()
    return p[..., 1:] + p[..., :1] * (codes.float() - 7.5)


def _plain_write(k, v, cache, slots):
    hd, bs = k.shape[-1], cache.shape[2]
    # rows without a slot store row 0's bytes once more
    src = torch.where(slots >= 0, torch.arange(slots.numel(), device=slots.device), 0)
    blk, off = slots[src] // bs, slots[src] % bs
    kc, vc, kp, vp = _parts(cache, hd)
    for x, par in ((k, kp), (v, vp)):
        c, s, m = _quantise(x[src].float())
        b = _nibbles(c)
        par[blk, :, off] = _params(s, m)
        if x is k:
            kc[blk, :, off] = b
        else:
            vc[blk, :, off // 4, :, off % 4] = b.view(*b.shape[:-1], hd // 4, 2)


def _plain_read(cache, slots, hd, dtype):
    bs = cache.shape[2]
    blk, off, ok = slots.clamp(min=0) // bs, slots.clamp(min=0) % bs, (slots >= 0)[:, None, None]
    kc, vc, kp, vp = _parts(cache, hd)
    k = _values(_codes(kc[blk, :, off]), kp[blk, :, off])
    v = _values(_codes(vc[blk, :, off // 4, :, off % 4].flatten(-2)), vp[blk, :, off])
    return torch.where(ok, k, 0).to(dtype), torch.where(ok, v, 0).to(dtype)


def _unpack(cache, tables, hd):
    """fp32 K and V [R, nk, L, hd] of the blocks of each request."""
    kc, vc, kp, vp = (x[tables.clamp(min=0).long()] for x in _parts(cache, hd))   # [R, n, nk, ...]
    k = _values(_codes(kc), kp)
    v = _values(_codes(vc.permute(0, 1, 2, 3, 5, 4, 6).flatten(-2).flatten(3, 4)), vp)
    return tuple(x.transpose(1, 2).flatten(2, 3) for x in (k, v))


def _plain_attn(s):
    q, out, (nq, nk, hd) = s["q"], s["out"], s["heads"]
    r, most = s["kv_lens"].numel(), s["max_q"]
    k, v = _unpack(s["cache"], s["tables"], hd)
    n = k.shape[2]
    # rows padded to [R, most]: row i of request r is its i-th query token
    at = s["cu_q"][:-1, None].long() + torch.arange(most, device=q.device)
    real = at < s["cu_q"][1:, None]
    at = at.clamp(max=q.shape[0] - 1)
    x = q[at].float().view(r, most, nk, nq // nk, hd).permute(0, 2, 1, 3, 4).reshape(r, nk, -1, hd).contiguous()
    pos = (s["kv_lens"] - (s["cu_q"][1:] - s["cu_q"][:-1]))[:, None] + torch.arange(most, device=q.device)
    key = torch.arange(n, device=q.device)
    seen = key <= pos[..., None]
    if s["window"]:
        seen &= key > pos[..., None] - s["window"]
    score = torch.matmul(x, k.transpose(-1, -2).contiguous()).mul_(s["scale"]).view(r, nk, most, nq // nk, n)
    score.masked_fill_(~seen[:, None, :, None], -math.inf)
    score -= score.amax(-1, keepdim=True).clamp(min=-1e30)
    score.exp_()
    den = score.sum(-1)
    o = torch.matmul(score.view(r, nk, -1, n), v)
    o = o.view(r, nk, most, nq // nk, hd) / den.clamp(min=1e-30)[..., None]
    o = o.permute(0, 2, 1, 3, 4).reshape(r, most, nq, hd).to(out.dtype)
    # rows past a request's last token store its last one again
    last = (s["cu_q"][1:] - s["cu_q"][:-1] - 1).long()
    o = torch.where(real[..., None, None], o, o[torch.arange(r, device=q.device), last][:, None])
    out[torch.where(real, at, (s["cu_q"][1:, None] - 1).long())] = o
    return out


def _plain_tables(s):
    lens, bs, tables, ring = s["kv_lens"].long(), s["bs"], s["tables"], s["ring"]
    cap, t_max, width = ring.numel(), s["slots"].numel(), tables.shape[1]
    head, free = s["ring_state"][0].long(), s["ring_state"][1].long()
    keep, q = torch.minimum(s["keep"].long(), lens).clamp(min=0), s["q_lens"].long().clamp(min=0)
    have = (lens + bs - 1) // bs
    want = (keep + q + bs - 1) // bs
    fits = want <= width
    need = torch.where(fits, (want - have).clamp(min=0), 0)
    q = torch.where(fits, q, 0)
    short, wide = (need > 0) & (need.cumsum(0) > free), (q > 0) & (q.cumsum(0) > t_max)
    go = fits & ~short & ~wide
    need, q = torch.where(go, need, 0), torch.where(go, q, 0)
    want = torch.where(go, want, (keep + bs - 1) // bs)
    gone = (have - want).clamp(min=0)
    to = q.cumsum(0)
    s["cu_q"][1:] = to
    s["kv_lens_out"].copy_(keep + q)
    s["status"].copy_(torch.where(~fits, 2, torch.where(short, 1, torch.where(wide, 3, 0))))
    col = torch.arange(width, device=lens.device)
    mine = tables.long()
    # returned blocks to the ring's tail, then taken ones from its head
    i = gone.cumsum(0)[:, None] - gone[:, None] + col - want[:, None]
    given = (col >= want[:, None]) & (col < have[:, None])
    new_ring = torch.cat([ring, ring.new_zeros(1)])
    new_ring[torch.where(given, (head + free + i) % cap, cap)] = tables
    i = need.cumsum(0)[:, None] - need[:, None] + col - have[:, None]
    taken = (col >= have[:, None]) & (col < (have + need)[:, None])
    mine = torch.where(taken, ring[(head + i.clamp(min=0)) % cap].long(), mine)
    ring.copy_(new_ring[:cap])
    tables.copy_(mine)
    s["ring_state_out"].copy_(torch.stack([(head + need.sum()) % cap, free - need.sum() + gone.sum()]))
    t = torch.arange(t_max, device=lens.device)
    r = torch.searchsorted(to, t, right=True).clamp(max=lens.numel() - 1)
    real = t < to[-1]
    pos = torch.where(real, keep[r] + t - (to - q)[r], 0)
    s["positions"].copy_(pos)
    s["slots"].copy_(torch.where(real, mine[r, (pos // bs).clamp(max=width - 1)] * bs + pos % bs, -1))


# ---- inputs --------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _filled(blocks, nk, hd, bs, g):
    """A cache whose blocks hold N(0, 1) keys and values, quantised."""
    cache = torch.empty(blocks, nk, bs, hd + 8, dtype=torch.uint8, device=DEV)
    step = max(1, 2 ** 26 // (nk * bs * hd))
    for i in range(0, blocks, step):
        part = cache[i:i + step]
        kc, vc, kp, vp = _parts(part, hd)
        for codes, par in ((kc, kp), (vc, vp)):
            c, s, m = _quantise(torch.randn(part.shape[0], nk, bs, hd, device=DEV, generator=g))
            b = _nibbles(c)
            par.copy_(_params(s, m))
            codes.copy_(b if codes is kc else b.view(-1, nk, bs // 4, 4, hd // 4, 2).transpose(3, 4))
    return cache


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEV)


def _block_tables(lens, bs, width, order):
    t = torch.full((len(lens), width), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(lens):
        t[i, :_blocks(n, bs)] = order[at:at + _blocks(n, bs)]
        at += _blocks(n, bs)
    return t.to(DEV), at


def prepare(case, seed):
    g = _generator(seed)
    bs = case["bs"]
    if case["kind"] == "tables":
        lens, keep, q = _table_lens(case)
        width = max(_blocks(max(n, k + m), bs) for n, k, m in zip(lens, keep, q)) + 3
        used = sum(_blocks(n, bs) for n in lens)
        blocks = used + sum(_blocks(k + m, bs) for k, m in zip(keep, q)) + 5
        order = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed)).int()
        tables, at = _block_tables(lens, bs, width, order)
        ring, head = torch.zeros(blocks, dtype=torch.int32), blocks - 3
        ring[(head + torch.arange(blocks - at)) % blocks] = order[at:]
        t_max = sum(q) + 7
        empty = lambda n, dtype=torch.int32: torch.zeros(n, dtype=dtype, device=DEV)  # noqa: E731
        return {"kind": "tables", "bs": bs, "tables": tables, "ring": ring.to(DEV), "kv_lens": _ints(lens), "keep": _ints(keep),
                "q_lens": _ints(q), "ring_state": _ints([head, blocks - at]), "ring_state_out": empty(2),
                "kv_lens_out": empty(case["r"]), "cu_q": empty(case["r"] + 1), "status": empty(case["r"]),
                "slots": empty(t_max, torch.int64), "positions": empty(t_max, torch.int64)}
    nk, hd, dtype = case["nk"], case["hd"], IO[case["io"]]
    if case["kind"] in ("write", "read"):
        t, run = case["t"], case["run"] or 1
        # runs of tokens, each in blocks of its own from a token inside the first on
        per = _blocks(run, bs) + 1
        blocks = _blocks(t, run) * per
        order = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed))
        i = torch.arange(t)
        pos = i % run + (5 * (i // run)) % bs
        slots = order[(i // run) * per + pos // bs] * bs + pos % bs
        slots = torch.cat([slots, torch.full((case["pad"],), -1)]).to(DEV)
        state = {"kind": case["kind"], "slots": slots, "cache": _filled(blocks, nk, hd, bs, g), "hd": hd, "dtype": dtype}
        rows = t + case["pad"]
        if case["kind"] == "write":
            # k and v as a fused projection leaves them: columns of one row
            kv = torch.randn(rows, 2 * nk, hd, device=DEV, generator=g).to(dtype)
            state["k"], state["v"] = kv[:, :nk], kv[:, nk:]
        state["out"] = tuple(torch.empty(rows, nk, hd, dtype=dtype, device=DEV) for _ in range(2))
        return state
    lens, q = _attn_lens(case)
    nq, t = case["nq"], sum(q)
    blocks = sum(_blocks(n, bs) for n in lens) + 4
    order = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed)).int()
    tables, _ = _block_tables(lens, bs, _blocks(max(lens), bs), order)
    cu = [0]
    for n in q:
        cu.append(cu[-1] + n)
    rows = 2 * torch.randn(t, nq, hd, device=DEV, generator=g)
    return {"kind": "attn", "cache": _filled(blocks, nk, hd, bs, g), "tables": tables, "kv_lens": _ints(lens), "cu_q": _ints(cu),
            "q": rows.to(dtype), "out": torch.zeros(t, nq, hd, dtype=dtype, device=DEV), "heads": (nq, nk, hd),
            "scale": hd ** -0.5, "max_q": max(q), "max_kv": max(lens), "window": case["window"]}


# ---- one pass ------------------------------------------------------------------

def _ops():
    import esimd_learning_amd
    return esimd_learning_amd.ops()


def run(state):
    s = state
    if s["kind"] == "tables":
        if own:
            _ops().esimd_kv_block_tables(s["kv_lens"], s["keep"], s["q_lens"], s["bs"], s["ring"], s["ring_state"],
                                         s["tables"], s["kv_lens_out"], s["ring_state_out"], s["cu_q"], s["slots"],
                                         s["positions"], s["status"])
        else:
            _plain_tables(s)
        return {n: s[n] for n in ("tables", "ring", "ring_state_out", "kv_lens_out", "cu_q", "slots", "positions", "status")}
    if s["kind"] == "attn":
        if own:
            _ops().esimd_kv4_attention(s["q"], s["cache"], s["tables"], s["kv_lens"], s["cu_q"], s["out"], s["scale"],
                                       s["max_q"], s["max_kv"], s["window"])
            return s["out"]
        return _plain_attn(s)
    if s["kind"] == "write":
        if own:
            _ops().esimd_kv4_cache_write(s["k"], s["v"], s["cache"], s["slots"])
        else:
            _plain_write(s["k"], s["v"], s["cache"], s["slots"])
    if own:
        _ops().esimd_kv4_cache_read(s["cache"], s["slots"], *s["out"])
        return s["out"]
    return _plain_read(s["cache"], s["slots"], s["hd"], s["dtype"])


# ---- the definitions in 64 bits --------------------------------------------------

def _exact_rows(raw, at, hd, bs, value):
    """Rows `at` (block, token) of the cache's bytes [nb, nk, bs (hd + 8)], in 64 bits: [len, nk, hd]."""
    blk, tok = at
    d = torch.arange(hd, device=raw.device)
    byte = (bs * hd // 2 + ((tok[:, None] // 4) * (hd // 4) + d // 4) * 8 + (tok[:, None] % 4) * 2 + (d % 4) // 2) if value \
        else tok[:, None] * (hd // 2) + d // 2
    code = torch.gather(raw[blk], 2, byte[:, None].expand(-1, raw.shape[1], -1)).long() >> (4 * (d % 2)) & 15
    base = bs * hd + (4 * bs if value else 0)
    par = torch.stack([raw[blk, :, base + 4 * tok + i] for i in range(4)], dim=-1).contiguous().view(torch.bfloat16).double()
    return par[..., 1:] + par[..., :1] * (code.double() - 7.5)


def _exact_quantised(x):
    """What the cache holds for the rows x: the parameters are bf16 by definition, the code is the nearest step."""
    x = x.double()
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    m = ((lo + hi) / 2).float().bfloat16().double()
    s = (torch.maximum(hi - m, m - lo) / 7.5).float().bfloat16().double()
    return m + s * (((x - m) / s + 7.5).round().clamp(0, 15) - 7.5)


def exact(case, seed):
    if case["kind"] == "tables":
        return None
    s = prepare(case, seed)
    hd, bs = case["hd"], case["bs"]
    if case["kind"] == "write":
        real = (s["slots"] >= 0)[:, None, None]
        return tuple(torch.where(real, _exact_quantised(x), 0) for x in (s["k"], s["v"]))
    raw = s["cache"].flatten(2)
    if case["kind"] == "read":
        return tuple(_exact_rows(raw, (s["slots"] // bs, s["slots"] % bs), hd, bs, value) for value in (False, True))
    lens, q = _attn_lens(case)
    nq, nk = case["nq"], case["nk"]
    out, at = torch.zeros(sum(q), nq, hd, dtype=torch.float64, device=DEV), 0
    for i, (n, m) in enumerate(zip(lens, q)):
        j = torch.arange(n, device=DEV)
        where = (s["tables"][i, j // bs].long(), j % bs)
        k, v = (_exact_rows(raw, where, hd, bs, value) for value in (False, True))
        p = torch.arange(n - m, n, device=DEV)[:, None]
        bad = (j > p) | (j <= p - case["window"]) if case["window"] else j > p
        for h in range(nq):
            kv = h * nk // nq
            w = (s["q"][at:at + m, h].double() @ k[:, kv].t()) * s["scale"]
            out[at:at + m, h] = torch.softmax(w.masked_fill(bad, -math.inf), -1) @ v[:, kv]
        at += m
    return out
