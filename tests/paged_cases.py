"""Inputs and error bounds of the paged-cache GPU tests."""
import numpy as np
import torch

from oracle import ref

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # half a step, relative


def f64(t):
    return t.detach().cpu().double().numpy()


def cache(g, dt, Hk, T, D, lens, own, spare=3, junk=float("nan"), width=1):
    """One layer's key / value [Hk, P, T, D] whose pages stand in a random order, every row that holds no token `junk`; the table
    int32 [B, W]."""
    each = [-(-(n + own) // T) for n in lens]
    P = sum(each) + spare
    order = torch.randperm(P, generator=g)
    table = torch.full((len(lens), max(each) + width), -1, dtype=torch.int32)
    kv = torch.full((2, Hk, P, T, D), junk).to(dt)
    at = 0
    for b, (n, e) in enumerate(zip(lens, each)):
        pages = order[at:at + e]
        table[b, :e] = pages
        at += e
        t = torch.arange(n + own)
        kv[0][:, pages[t // T], t % T] = (torch.randn(Hk, n + own, D, generator=g) * 1.5).to(dt)
        kv[1][:, pages[t // T], t % T] = torch.randn(Hk, n + own, D, generator=g).to(dt)
    return kv[0], kv[1], table


def tree_masks(g, B, S):
    """Ancestor masks of random trees (row 0 the root), int64 [B, S]."""
    mask = torch.zeros(B, S, dtype=torch.int64)
    for b in range(B):
        m = [1]
        for r in range(1, S):
            m.append(m[int(torch.randint(0, r, (1,), generator=g))] | (1 << r))
        mask[b] = torch.tensor([x - (1 << 64) if x >= 1 << 63 else x for x in m])
    return mask


def bound(dt, want, spread, mass, heft, tokens, D):
    """How far an output may lie from float64, element by element (u = half a step of the type):
    u |out|: its own rounding; u spread: every weight rounded to the type, numerator and normaliser alike, moves
    sum w (v - out) by at most u sum w |v - out| (a second-order term below 2 u of it);
    2 e spread: a weight's relative error e = (the score's D products and sums in fp32, each within 2^-23 of the partial sums'
    magnitude `heft`) + (the exponent's argument and exp2: 2^-23 times the argument's size, at most 2 heft, plus 2^-22);
    fp32 sums over the tokens, rescales and joins: (32 within an MFMA, one each per 32 tokens and rescale, 600 of joins) 2^-24
    sum w |v|; fp16 weights under 2^-28 of the largest: 2^-39 of it each."""
    u = UNIT[dt]
    e = ((D + 4) * 2.0 ** -23 + 3 * 2.0 ** -23) * heft[..., None] + 2.0 ** -22
    sums = (tokens / 16 + 32 + 600) * 2.0 ** -24
    tiny = tokens * 2.0 ** -38 if dt == torch.float16 else 0.0
    err = (u * (1 + 4 * u) + 2 * e) * spread + (sums + tiny) * mass
    return u * (np.abs(want) + err) + err + 2.0 ** -24 * (dt == torch.float16)


def check(got, dt, q, key, value, table, lens, mask, scale, keep=None, rows=slice(None)):
    want, spread, mass, heft = ref.paged_attention(f64(q), f64(key), f64(value), table.numpy(), lens, None if mask is None else mask.numpy(),
                                                   scale, keep)
    tokens = max(lens) + q.shape[1]
    err, lim = np.abs(f64(got) - want), bound(dt, want, spread, mass, heft, tokens, q.shape[3])
    err, lim = err[:, rows], lim[:, rows]
    bad = ~(err <= lim)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist(), float(np.nanmax(err / np.maximum(lim, 1e-30))))
    return float(np.nanmax(err / np.maximum(lim, 1e-30)))


def views():
    """Strides of rows of 100 places [sequences, kv heads] apart from one another, of a second view of the buffer, and how many
    places ahead that begins."""
    for ob, oh in ((200, 100), (500, 210), (100, 300), (150, 460)):
        for pb, ph in ((ob, oh), (0, 0), (100, 0), (oh, ob), (1000, 7)):
            for d in (-2001, -901, -250, -101, -100, -99, -1, 1, 50, 99, 100, 101, 199, 250, 320, 410, 499, 700, 1200):
                yield ob, oh, pb, ph, d


def rows_meet(B, Hk, N, d, pb, ph, ob, oh):
    """Whether a row of the view at d meets one of the view at 0, place by place."""
    written = {b * ob + h * oh + t for b in range(B) for h in range(Hk) for t in range(N)}
    return any(d + b * pb + h * ph + t in written for b in range(B) for h in range(Hk) for t in range(N))
