"""Oracle of the 4-bit key/value cache's operators, on the CPU.

Quantisation follows the format's definition in fp32, one rounding an operation;
values and attention are computed in fp64; tables by plain loops.
"""

import math

import torch


def quantise(x):
    """Rows [..., hd] -> (codes uint8, step, centre), the last two bf16 values in fp32."""
    x = x.float()
    lo, hi = x.amin(-1), x.amax(-1)
    ok = torch.isfinite(x).all(-1)
    m = (0.5 * lo + 0.5 * hi).bfloat16().float()
    s = (torch.maximum(hi - m, m - lo) / 7.5).bfloat16().float()
    s = torch.where(ok & (s >= 2.0 ** -100), s, torch.zeros_like(s))
    m = torch.where(ok, m, torch.full_like(m, math.nan))
    by = torch.where(s > 0, s, torch.ones_like(s))
    c = torch.nan_to_num(((x - m[..., None]) / by[..., None] + 7.5).round()).clamp(0, 15)
    return torch.where((s > 0)[..., None], c, torch.full_like(c, 8.0)).to(torch.uint8), s, m


def values(c, s, m):
    """fp64 values of codes."""
    return m.double()[..., None] + s.double()[..., None] * (c.double() - 7.5)


def empty(blocks, n_kv, bs, hd, fill=0xFF):
    """A cache of bytes `fill` (0xFF: every parameter a NaN)."""
    return torch.full((blocks, n_kv, bs, hd + 8), fill, dtype=torch.uint8)


def put(cache, slot, k, v):
    """Store one token's rows k, v [n_kv, hd] in a CPU cache, byte by byte."""
    nb, nk, bs, w = cache.shape
    hd = w - 8
    blk, tok = slot // bs, slot % bs
    for h in range(nk):
        raw = cache[blk, h].view(-1)
        for part, x in ((0, k[h]), (1, v[h])):
            c, s, m = quantise(x)
            c = c.int()
            par = torch.stack([s, m]).bfloat16()
            par = torch.where(par.isnan(), torch.tensor(0x7FC0, dtype=torch.int16).view(torch.bfloat16), par).view(torch.uint8)
            raw[bs * hd + part * 4 * bs + 4 * tok: bs * hd + part * 4 * bs + 4 * tok + 4] = par
            by = (c[0::2] | (c[1::2] << 4)).to(torch.uint8)
            if part == 0:
                raw[tok * hd // 2: (tok + 1) * hd // 2] = by
            else:
                words = raw[bs * hd // 2: bs * hd].view(bs // 4, hd // 4, 4, 2)
                words[tok // 4, :, tok % 4] = by.view(hd // 4, 2)


def get(cache, slot):
    """fp64 k, v [n_kv, hd] of a slot of a CPU cache."""
    nb, nk, bs, w = cache.shape
    hd = w - 8
    blk, tok = slot // bs, slot % bs
    flat = cache[blk].view(nk, -1)
    par = [flat[:, bs * hd + p * 4 * bs + 4 * tok: bs * hd + p * 4 * bs + 4 * tok + 4].contiguous().view(torch.bfloat16)
           for p in (0, 1)]
    kb = flat[:, tok * hd // 2: (tok + 1) * hd // 2]
    vb = flat[:, bs * hd // 2: bs * hd].view(nk, bs // 4, hd // 4, 4, 2)[:, tok // 4, :, tok % 4].reshape(nk, hd // 2)
    out = []
    for b, p in ((kb, par[0]), (vb, par[1])):
        c = torch.stack([b & 15, b >> 4], -1).flatten(-2)
        out.append(values(c, p[:, 0], p[:, 1]))
    return out


def attention(q, keys, vals, scale, window=0, weigh=()):
    """One request: q [n, n_q, hd], the last n tokens of keys / vals [len, n_kv, hd] -> fp64 [n, n_q, hd].

    With ``weigh``, a list of tensors [len, n_kv, d], returns (out, [sum_j p_j x_j of each])."""
    n, nq, hd = q.shape
    L, nk = keys.shape[0], keys.shape[1]
    p = torch.arange(L - n, L)[:, None]
    j = torch.arange(L)
    seen = (j <= p) & ((j > p - window) if window else (j >= 0))
    outs = [torch.zeros(n, nq, x.shape[-1], dtype=torch.float64) for x in (vals, *weigh)]
    for h in range(nq):
        g = h // (nq // nk)
        w = (q[:, h].double() @ keys[:, g].double().t()) * scale
        w = w.masked_fill(~seen, -math.inf)
        w = torch.exp(w - w.amax(-1, keepdim=True).clamp(min=-1e300)) if L else w
        w = w / w.sum(-1, keepdim=True).clamp(min=1e-300)
        for o, x in zip(outs, (vals, *weigh)):
            o[:, h] = w @ x[:, g].double()
    return (outs[0], outs[1:]) if weigh else outs[0]


def block_tables(kv_lens, keep_lens, q_lens, bs, ring, state, tables, T, fixed_rows=False):
    """One step on Python lists; tables is a list of rows, changed like ring in place.  Returns (kv_lens_out,
    ring_state_out, cu_q, slots, positions, status).  fixed_rows: refused requests keep their rows, as padding."""
    cap, width = len(ring), len(tables[0]) if tables else 0
    head, count = state
    taken = given = wish = rows = 0
    cu, lens, slots, pos, status = [0], [], [], [], []
    tail = head + count
    for r, (n, keep, q) in enumerate(zip(kv_lens, keep_lens, q_lens)):
        n = min(max(n, 0), width * bs)
        keep, q = min(max(keep, 0), n), max(q, 0)
        have, want, st, wished = -(-n // bs), -(-(keep + q) // bs), 0, q
        if want > width:
            st = 2
            rows += q if fixed_rows else 0
        else:
            need = max(0, want - have)
            wish += need
            rows += q
            if need and wish > count:
                st = 1
            elif q and rows > T:
                st = 3
        if st:
            q, want = 0, -(-keep // bs)
        for i in range(have, want):
            tables[r][i] = ring[(head + taken) % cap]
            taken += 1
        for i in range(want, have):
            ring[(tail + given) % cap] = tables[r][i]
            given += 1
        for p in range(keep, keep + q):
            pos.append(p)
            slots.append(tables[r][p // bs] * bs + p % bs)
        end = min(cu[-1] + wished, T) if fixed_rows else cu[-1] + q
        pos += [0] * (end - len(pos))
        slots += [-1] * (end - len(slots))
        cu.append(end)
        lens.append(keep + q)
        status.append(st)
    slots += [-1] * (T - len(slots))
    pos += [0] * (T - len(pos))
    return lens, [(head + taken) % cap, count - taken + given], cu, slots, pos, status
