"""A server's step over bounded caches, as cases to be measured: drafted tokens verified against the target's probabilities
(verify_drafts), attention over the pages within a sliding window and a few first tokens (attn_window), the attention weight
every cached token has drawn, summed up (attn_mass), and sequences thinned to the tokens of most weight (page_evict).

The cache is page_fork's and page_commit's: kv [layers, 2, kv_heads, pages, T, D] (keys, values), a sequence's pages in table
[sequences, W] (-1: none), its committed tokens in length, the references to a page in refs (0: free), and every full page's
mean key in ksum [layers, kv_heads, pages, D]. Where `own` is false, run() computes the operators from elementary torch operations
in 32 bits (verification in 64: a drawn token goes by the borders of long sums) and rounds once; where it is true it calls
mdx._C.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

DEV = "cuda"
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
HEADS = ((32, 8, 128), (16, 4, 256), (16, 8, 64), (32, 4, 128))  # q heads, kv heads, head_dim of the configurations and tests


# ---- the cases -------------------------------------------------------------------------------------
def listed():
    return [
        # three drafted tokens of one sequence over a small vocabulary: the smallest verification
        dict(name="verify_1x4", kind="verify", seqs=1, rows=4, vocab=32768, form="chain", heat=0.8, dt="bf16"),
        # drafted trees of 8 rows in 16 sequences, drafts without probabilities, as the hybrid stack drafts
        dict(name="verify_tree", kind="verify", seqs=16, rows=8, vocab=151936, form="tree", heat=0.7, dt="bf16"),
        # a serving batch: 32 sequences with six drafted tokens each, drawn from the draft's distributions
        dict(name="verify_32x7", kind="verify", seqs=32, rows=7, vocab=151936, form="chain", heat=1.0, dt="bf16"),
        # one token of one sequence in a window of 512: the smallest attention, head_dim 64, fp16
        dict(name="window_1", kind="window", heads=16, kv_heads=8, dim=64, page=16, seqs=1, rows=1, lo=4000, hi=4000, window=512, sinks=4, tree=False, dt="fp16"),
        # a serving batch: single tokens of 64 sequences, short ones and ones far past the window
        dict(name="window_64", kind="window", heads=32, kv_heads=8, dim=128, page=64, seqs=64, rows=1, lo=100, hi=32767, window=4096, sinks=4, tree=False, dt="bf16"),
        # drafted trees of 8 rows in 16 sequences, head_dim 256, short pages
        dict(name="window_tree_d256", kind="window", heads=16, kv_heads=4, dim=256, page=16, seqs=16, rows=8, lo=500, hi=16001, window=2000, sinks=16, tree=True, dt="bf16"),
        # 2048 rows of a long prompt
        dict(name="window_prompt_2k", kind="window", heads=32, kv_heads=8, dim=128, page=64, seqs=1, rows=2048, lo=30000, hi=30000, window=4096, sinks=4, tree=False, dt="bf16"),
        # the weights that single tokens of 32 sequences give
        dict(name="mass_32", kind="mass", heads=32, kv_heads=8, dim=128, page=64, seqs=32, rows=1, lo=500, hi=8191, window=0, sinks=0, tree=False, dt="bf16"),
        # the accepted rows of drafted trees of 8 rows in 8 sequences, head_dim 256, within a window
        dict(name="mass_tree_d256", kind="mass", heads=16, kv_heads=4, dim=256, page=32, seqs=8, rows=8, lo=1000, hi=6001, window=4000, sinks=4, tree=True, dt="bf16"),
        # 1000 rows of a prompt behind 4000 tokens
        dict(name="mass_prompt_1k", kind="mass", heads=32, kv_heads=8, dim=128, page=64, seqs=1, rows=1000, lo=4000, hi=4000, window=0, sinks=0, tree=False, dt="bf16"),
        # one layer of one sequence thinned to an eighth: the smallest eviction
        dict(name="evict_1", kind="evict", layers=1, kv_heads=8, dim=64, page=16, seqs=1, ctx=2001, keep=180, sinks=4, recent=64, room=8, dt="fp16"),
        # four sequences of 16 thousand tokens thinned to an eighth, all attention layers
        dict(name="evict_4x16k", kind="evict", layers=8, kv_heads=8, dim=128, page=64, seqs=4, ctx=16100, keep=1500, sinks=4, recent=544, room=8, dt="bf16"),
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(("verify", "window", "window", "mass", "mass", "evict"))
    heads, kv_heads, dim = rng.choice(HEADS)
    page = rng.choice((16, 32, 64, 128))
    dt = rng.choice(("bf16", "bf16", "fp16"))
    if kind == "verify":
        seqs, dt = log_int(1, 32), rng.choice(("bf16", "bf16", "fp16", "fp32"))
        most = (112 if dt == "fp32" else 224) // seqs
        return dict(kind=kind, seqs=seqs, rows=rng.randint(2, max(2, min(16, most))), vocab=log_int(4096, 151936), form=rng.choice(("chain", "chain", "tree")),
                    heat=round(rng.uniform(0.5, 1.2), 2), dt=dt)
    case = dict(kind=kind, kv_heads=kv_heads, dim=dim, page=page, dt=dt)
    if kind == "evict":
        ctx = log_int(100, 16000)
        keep = max(1, int(ctx * rng.uniform(0.05, 0.3)))
        return dict(case, layers=rng.choice((1, 2, 4)), seqs=rng.randint(1, 4), ctx=ctx, keep=keep, sinks=rng.randint(0, 8), recent=rng.randint(0, max(1, ctx // 8)), room=rng.randint(1, 64))
    form = rng.choice(("decode", "verify", "prompt"))
    seqs = 1 if form == "prompt" else log_int(1, 32)
    rows = 1 if form == "decode" else rng.randint(2, 16) if form == "verify" else log_int(65, 1000)
    hi = log_int(16, 4000 if form == "prompt" else 8000 if kind == "mass" else 30000)
    window = log_int(1, 4096) if kind == "window" or rng.random() < 0.5 else 0
    return dict(case, heads=heads, seqs=seqs, rows=rows, lo=rng.randint(0, hi), hi=hi, window=window, sinks=rng.choice((0, 1, 4, 16, 70)) if window else 0, tree=form == "verify")


# ---- inputs ----------------------------------------------------------------------------------------
def _lengths(case):
    """The sequences' committed tokens: spread over [lo, hi] (ctx: a little around it), the longest first."""
    n = case["seqs"]
    if "ctx" in case:
        return [max(0, case["ctx"] - (17 * i) % 61 * (i > 0)) for i in range(n)]
    return [case["hi"] - int((case["hi"] - case["lo"]) * (i * 0.6180339887498949 % 1.0)) for i in range(n)]


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _pages_of(seed, pages_each, spare, width):
    """A page table with `pages_each` pages per sequence in a random order of the pool, and the references."""
    order = torch.randperm(sum(pages_each) + spare, generator=_gen(seed), device=DEV).to(torch.int32)
    table = torch.full((len(pages_each), width), -1, dtype=torch.int32, device=DEV)
    refs = torch.zeros(order.numel(), dtype=torch.int32, device=DEV)
    at = 0
    for i, n in enumerate(pages_each):
        table[i, :n] = order[at:at + n]
        at += n
    refs[order[:at].long()] = 1
    return table, refs


def _random_kv(gen, layers, kv_heads, pages, page, dim, dt):
    """Keys of 1.5 about a mean of their own in every page (as the keys of a passage have), values of 1."""
    kv = torch.empty(layers, 2, kv_heads, pages, page, dim, dtype=dt, device=DEV)
    for i in range(layers):
        kv[i].normal_(generator=gen)
        kv[i, 0].mul_(1.5).add_(torch.randn(kv_heads, pages, 1, dim, generator=gen, device=DEV).to(dt))
    return kv


def _tree_masks(parent):
    """Ancestor bit masks int64 [seqs, rows] of the trees parent [seqs, rows]."""
    seqs, rows = parent.shape
    bit = torch.ones(rows, dtype=torch.int64, device=DEV) << torch.arange(rows, device=DEV)
    mask = torch.zeros(seqs, rows, dtype=torch.int64, device=DEV)
    mask[:, 0] = 1
    for r in range(1, rows):
        mask[:, r] = mask.gather(1, parent[:, r:r + 1].long())[:, 0] | bit[r]
    return mask


def _prepare_verify(case, gen, dt):
    """The target's and the draft's logits over a common part (a good draft differs little), a few likely tokens among many
    unlikely ones; drafted tokens drawn from the draft's distributions, a tree's children the draft's best."""
    n, rows, vocab = case["seqs"], case["rows"], case["vocab"]
    base = torch.randn(n, rows, vocab, generator=gen, device=DEV).mul_(1.6)
    for _ in range(6):
        at = torch.randint(0, vocab, (n, rows, 1), generator=gen, device=DEV)
        base.scatter_add_(2, at, 9.0 + 2.0 * torch.randn(n, rows, 1, generator=gen, device=DEV))
    s = dict(case=case, logits=torch.randn(n, rows, vocab, generator=gen, device=DEV).mul_(0.5).add_(base).to(dt), draft=None, parent=None)
    s["uniform"] = torch.rand(n, rows + 1, generator=gen, device=DEV, dtype=torch.float64)
    s["heat"] = torch.linspace(case["heat"], case["heat"] + 0.1, n, device=DEV)
    s["tokens"] = torch.zeros(n, rows, dtype=torch.int64, device=DEV)
    drafted = base[:, :rows - 1].add_(torch.randn(n, rows - 1, vocab, generator=gen, device=DEV).mul_(0.5))
    if case["form"] == "chain":
        s["draft"] = drafted.to(dt)
        noise = torch.empty(n, rows - 1, vocab, device=DEV).exponential_(generator=gen)
        s["tokens"][:, 1:] = (s["draft"].float() / s["heat"][:, None, None] - noise.log()).argmax(-1)
    else:
        # row 0 the root, every other row a child of an earlier one: its parent's next best token
        s["parent"] = (torch.rand(n, rows, generator=gen, device=DEV) ** 1.5 * torch.arange(rows, device=DEV)).to(torch.int32)
        best = drafted.topk(rows, -1).indices
        place = torch.stack([(s["parent"][:, 1:r] == s["parent"][:, r:r + 1]).sum(1) for r in range(1, rows)], 1)
        flat = s["parent"][:, 1:].long() * rows + place
        s["tokens"][:, 1:] = best.reshape(n, -1).gather(1, flat)
    return s


def _prepare_evict(case, seed, gen, dt):
    """The sequences in the first rows of the table, the thinned copies' places, empty before and after a pass, behind them; the
    weights drawn so far: a few large ones, many small, tokens that none has drawn."""
    lens, page, seqs = _lengths(case), case["page"], case["seqs"]
    width = (max(lens) + case["room"]) // page + 2
    most = case["keep"] + case["sinks"] + case["recent"]
    new = sum(-(-(min(n, most) + case["room"]) // page) for n in lens)
    s = dict(case=case)
    s["table"], s["refs"] = _pages_of(seed, [-(-n // page) for n in lens] + [0] * seqs, new + 3, width)
    s["length"] = torch.tensor(lens + [0] * seqs, dtype=torch.int32, device=DEV)
    s["kv"] = _random_kv(gen, case["layers"], case["kv_heads"], s["refs"].numel(), page, case["dim"], dt)
    s["ksum"] = s["kv"][:, 0].float().mean(-2).to(dt)
    mass = torch.randn(case["layers"], 2 * seqs, case["kv_heads"], width * page, generator=gen, device=DEV).mul_(2).exp_()
    s["mass"] = mass.mul_(torch.rand(mass.shape, generator=gen, device=DEV) > 0.05)
    s["src"] = torch.arange(seqs, dtype=torch.int32, device=DEV)
    s["dst"] = s["src"] + seqs
    s["none"] = torch.full_like(s["src"], -1)
    return s


def prepare(case, seed):
    gen, dt = _gen(seed), DT[case["dt"]]
    if case["kind"] == "verify":
        return _prepare_verify(case, gen, dt)
    if case["kind"] == "evict":
        return _prepare_evict(case, seed, gen, dt)
    lens, page = _lengths(case), case["page"]
    hk, dim, seqs, rows = case["kv_heads"], case["dim"], case["seqs"], case["rows"]
    s = dict(case=case, length=torch.tensor(lens, dtype=torch.int32, device=DEV))
    each = [-(-(n + rows) // page) for n in lens]
    s["table"], refs = _pages_of(seed, each, 3, max(each) + 1)
    s["kv"] = _random_kv(gen, 1, hk, refs.numel(), page, dim, dt)
    s["q"] = (torch.randn(seqs, rows, case["heads"], dim, generator=gen, device=DEV) * 1.5).to(dt)
    parent = (torch.rand(seqs, rows, generator=gen, device=DEV) * torch.arange(rows, device=DEV)).to(torch.int32)
    s["mask"] = _tree_masks(parent) if case["tree"] else None
    if case["kind"] == "mass":
        # the attention has run, and the accepted rows stand behind the committed tokens: every tree's deepest row's ancestors
        key, value = s["kv"][0, 0], s["kv"][0, 1]
        s["lse"] = _plain_window(s["q"], key, value, s["table"], s["length"], case["window"] or 1 << 30, case["sinks"], s["mask"], lens)[1]
        s["count"] = s["path"] = None
        if case["tree"]:
            r = torch.arange(rows, device=DEV)
            has = (s["mask"][:, :, None] >> r) & 1 == 1
            deep = has.sum(2).argmax(1)
            line = has[torch.arange(seqs, device=DEV), deep]
            s["count"] = line.sum(1).to(torch.int32)
            s["path"] = torch.where(line, r, rows).sort(1).values.to(torch.int32).contiguous()
            at = s["length"][:, None].long()
            a_page, a_row = _place(s["table"], at + s["path"].long().clamp(max=rows - 1), page)
            b_page, b_row = _place(s["table"], at + r[None], page)
            live = r[None] < s["count"][:, None]
            s["kv"][:, :, :, b_page[live], b_row[live]] = s["kv"][:, :, :, a_page[live], a_row[live]]
        places = s["table"].shape[1] * page
        s["prior"] = torch.empty(seqs, hk, places, device=DEV).exponential_(generator=gen)
        s["mass"] = torch.zeros(seqs, hk, places, device=DEV)
    return s


# ---- the operators in plain form -------------------------------------------------------------------
def _probabilities(logits, heat):
    z = logits.double() / heat.double()[:, None, None]
    e = torch.exp(z - z.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _draw(w, u):
    """The lowest index whose cumulative weight passes u of the whole (the last with a weight, if rounding leaves none)."""
    c = w.cumsum(-1)
    last = w.shape[-1] - 1 - (w > 0).flip(-1).to(torch.uint8).argmax(-1)
    return torch.minimum((c <= u[:, None] * c[:, -1:]).sum(-1), last)


def _plain_verify(logits, tokens, uniform, draft, parent, heat):
    n, rows, _ = logits.shape
    b = torch.arange(n, device=DEV)
    p = _probabilities(logits, heat)
    if parent is None:
        q = _probabilities(draft, heat)
        x = tokens[:, 1:, None]
        ok = uniform[:, :rows - 1] * q.gather(2, x)[..., 0] < p[:, :-1].gather(2, x)[..., 0]
        count = 1 + ok.long().cumprod(1).sum(1)
        r = torch.arange(rows, device=DEV)[None]
        path = torch.where(r < count[:, None], r, -1)
        w = p[b, count - 1]
        rest = (w - q[b, (count - 1).clamp(max=rows - 2)]).clamp(min=0)
        w = torch.where(((count < rows) & (rest.sum(1) > 0))[:, None], rest, w)
    else:
        cur, count, acc = torch.zeros_like(b), torch.ones_like(b), torch.zeros(n, dtype=torch.float64, device=DEV)
        path = torch.full((n, rows), -1, dtype=torch.int64, device=DEV)
        path[:, 0] = 0
        w = p[:, 0].clone()
        for c in range(1, rows):
            child, x = parent[:, c] == cur, tokens[:, c]
            acc = acc + torch.where(child, w[b, x], 0.0)
            taken = child & (uniform[b, cur] < acc)
            w[b, x] = torch.where(child, 0.0, w[b, x])
            path[b, count.clamp(max=rows - 1)] = torch.where(taken, c, path[b, count.clamp(max=rows - 1)])
            count = count + taken
            cur = torch.where(taken, c, cur)
            acc = torch.where(taken, 0.0, acc)
            w = torch.where(taken[:, None], p[:, c], w)
    return count.to(torch.int32), path.to(torch.int32), _draw(w, uniform[:, rows])


def _place(table, pos, page):
    """Pages and rows of the positions pos [n, r] of the n sequences."""
    return table.gather(1, (pos // page).clamp(max=table.shape[1] - 1)).long(), pos % page


def _attended(pos, length, rows, window, sinks, mask):
    """Which of the positions pos [n, t] each row attends, bool [n, rows, t]: of the committed tokens and the rows' own that it
    admits (in that order) the first `sinks` and the last `window`."""
    n, r = length[:, None, None].long(), torch.arange(rows, device=DEV)
    at = pos[:, None, :]
    if mask is None:
        seen = at <= n + r[:, None]
        return seen & ((at < sinks) | (at >= n + r[:, None] + 1 - window))
    bits = (mask[:, :, None] >> r) & 1
    before = bits.cumsum(2) - bits
    j = (at - n).clamp(0, rows - 1).expand(-1, rows, -1)
    index = torch.where(at < n, at, n + before.gather(2, j))
    seen = (at < n) | ((at < n + rows) & (bits.gather(2, j) == 1))
    return seen & ((index < sinks) | (index >= n + bits.sum(2, keepdim=True) - window))


def _scores(q, key, table, length, window, sinks, mask, lens):
    """Scores in 32 bits of every row over the tokens within reach of it: [kv_heads, n, rows * group, t], -inf where a row does
    not attend; the tokens' positions [n, t], pages and rows."""
    n, rows, heads, dim = q.shape
    hk, _, page, _ = key.shape
    first = [max(min(sinks, l + rows), l - window) for l in lens]
    width = max(l + rows - f for l, f in zip(lens, first))
    head = torch.arange(min(sinks, max(lens) + rows), device=DEV)[None].expand(n, -1)
    tail = torch.tensor(first, device=DEV)[:, None] + torch.arange(width, device=DEV)
    pos = torch.cat([head, tail], 1)
    at = (length[:, None].long() + rows - 1).clamp(min=0)
    live = torch.cat([head <= at, tail <= at], 1) & ~torch.cat([head >= torch.tensor(first, device=DEV)[:, None], tail < 0], 1)
    pages, row = _place(table, pos, page)
    pages = pages.clamp(min=0)
    k = key[:, pages, row].float()
    seen = live[:, None] & _attended(pos, length, rows, window, sinks, mask)
    seen = seen[:, :, None].expand(n, rows, heads // hk, -1).reshape(n, rows * (heads // hk), -1)
    qg = q.float().reshape(n, rows, hk, heads // hk, dim).permute(2, 0, 1, 3, 4).reshape(hk, n, -1, dim)
    z = qg @ k.transpose(-1, -2) * dim ** -0.5
    return z.masked_fill(~seen[None], -math.inf), pos, pages, row


def _plain_window(q, key, value, table, length, window, sinks, mask, lens):
    n, rows, heads, dim = q.shape
    hk = key.shape[0]
    z, _, pages, row = _scores(q, key, table, length, window, sinks, mask, lens)
    top = z.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    e = torch.exp(z - top)
    total = e.sum(-1, keepdim=True)
    o = (e @ value[:, pages, row].float()) / torch.where(total == 0, 1.0, total)
    shape = (hk, n, rows, heads // hk)
    out = o.reshape(*shape, dim).permute(1, 2, 0, 3, 4).reshape(n, rows, heads, dim).to(q.dtype)
    lse = (top + total.log()).reshape(shape).permute(1, 2, 0, 3).reshape(n, rows, heads)
    return out, lse


def _plain_mass(q, key, table, length, lse, prior, count, path, window, sinks, lens, out):
    n, rows, heads, _ = q.shape
    hk = key.shape[0]
    if path is not None:
        take = path.long().clamp(max=rows - 1)
        q = q.gather(1, take[:, :, None, None].expand_as(q))
        lse = lse.gather(1, take[:, :, None].expand_as(lse))
    z, pos, _, _ = _scores(q, key, table, length, window, sinks, None, lens)
    base = lse.reshape(n, rows, hk, heads // hk).permute(2, 0, 1, 3).reshape(hk, n, -1, 1)
    w = torch.exp(z - base).reshape(hk, n, rows, heads // hk, -1)
    if count is not None:
        w = w * (torch.arange(rows, device=DEV) < count[:, None])[None, :, :, None, None]
    w = w.sum((2, 3)).permute(1, 0, 2)  # [n, hk, t]
    places = torch.arange(out.shape[2], device=DEV)[None]
    ends = length.long() + (rows if count is None else count.long())
    total = torch.where((places < length[:, None])[:, None], prior, 0.0)
    inside = (pos < ends[:, None])[:, None] & (w > 0)
    at = pos.clamp(max=out.shape[2] - 1)[:, None].expand_as(w)
    total.scatter_add_(2, at, torch.where(inside, w, 0.0))
    out.copy_(torch.where((places < ends[:, None])[:, None], total, out))
    return out


def _give_pages(refs, want):
    """Pages for the true places of want [n, W], the lowest free ones in order: (page of each place, rows that got theirs).
    A row is served if it and all rows before it find enough pages."""
    free = (refs == 0).nonzero()[:, 0]
    ok = want.sum(1).cumsum(0) <= free.numel()
    want = want & ok[:, None]
    pages = torch.full(want.shape, -1, dtype=torch.int32, device=DEV)
    pages[want] = free[:int(want.sum())].to(torch.int32)
    return pages, ok


def _plain_evict(kv, ksum, table, length, refs, mass, dst, src, keep, sinks, recent, room, lens):
    layers, _, hk, _, page, dim = kv.shape
    most = keep + sinks + recent
    j = torch.arange(table.shape[1], device=DEV)[None]
    n = length[src.long()].long()
    m = n.clamp(max=most)
    pages, ok = _give_pages(refs, j < (-(-(m + room) // page))[:, None])
    kept = torch.full((src.numel(), layers, hk, most), -1, dtype=torch.int32, device=DEV)
    old = table[src.long()].clone()
    drawn = mass[:, src.long()].clone()
    for i, (a, b) in enumerate(zip(src.tolist(), dst.tolist())):
        t, c = torch.arange(lens[i], device=DEV), min(lens[i], most)
        worth = drawn[:, i, :, :lens[i]].clone()
        worth[:, :, (t < sinks) | (t >= lens[i] - recent)] = math.inf
        idx = worth.sort(dim=-1, descending=True, stable=True).indices[..., :c].sort(-1).values  # [layers, hk, c]
        kept[i, :, :, :c] = idx.to(torch.int32)
        from_page, from_row = old[i][idx // page].long(), idx % page
        k = torch.arange(c, device=DEV)
        to_page, to_row = pages[i][k // page].long(), k % page
        l, h = torch.arange(layers, device=DEV)[:, None, None], torch.arange(hk, device=DEV)[None, :, None]
        for part in (0, 1):
            kv[l, part, h, to_page, to_row] = kv[l, part, h, from_page, from_row]
        full = pages[i][:c // page].long()
        ksum[:, :, full] = kv[:, 0][:, :, full].float().mean(-2).to(ksum.dtype)
        mass[:, b, :, :c] = drawn[:, i].gather(-1, idx)
    gone = table[dst.long()]
    refs[gone[gone >= 0].long()] -= 1
    refs[pages[pages >= 0].long()] = 1
    table[dst.long()] = pages
    length[dst.long()] = m.to(torch.int32)
    return ok.to(torch.int32), kept


def _plain_drop(table, length, refs, dst):
    gone = table[dst.long()]
    refs[gone[gone >= 0].long()] -= 1
    table[dst.long()] = -1
    length[dst.long()] = 0
    return torch.ones_like(dst)


# ---- one pass ---------------------------------------------------------------------------------------
def _ops():
    at = os.path.join(os.getcwd(), "comfy-mono-decode-xpu_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    from mdx import _C
    return _C


def run(s):
    c = s["case"]
    if c["kind"] == "verify":
        if own:
            count, path, token = _ops().verify_drafts(s["logits"], s["tokens"], s["uniform"], draft=s["draft"], parent=s["parent"], temperature=s["heat"])
        else:
            count, path, token = _plain_verify(s["logits"], s["tokens"], s["uniform"], s["draft"], s["parent"], s["heat"])
        return dict(count=count, path=path, token=token)
    if c["kind"] == "evict":
        # the thinned copies are made and dropped again: the state is as before, and the copied rows stand in the pool
        a = (s["kv"], s["ksum"], s["table"], s["length"], s["refs"], s["mass"], s["dst"], s["src"], c["keep"], c["sinks"], c["recent"], c["room"])
        if own:
            made, kept = _ops().page_evict(*a)
            gone = _ops().page_fork(*a[:5], s["dst"], s["none"])
        else:
            made, kept = _plain_evict(*a, _lengths(c))
            gone = _plain_drop(s["table"], s["length"], s["refs"], s["dst"])
        return dict(kv=s["kv"].view(torch.int16), ksum=s["ksum"], mass=s["mass"], table=s["table"], length=s["length"], refs=s["refs"], kept=kept, made=made, gone=gone)
    key, value = s["kv"][0, 0], s["kv"][0, 1]
    lens = _lengths(c)  # what the program knows of its sequences
    window = c["window"] or 1 << 30
    if c["kind"] == "window":
        if own:
            out, lse = _ops().attn_window(s["q"], key, value, s["table"], s["length"], window, c["sinks"], mask=s["mask"])
        else:
            out, lse = _plain_window(s["q"], key, value, s["table"], s["length"], window, c["sinks"], s["mask"], lens)
        return dict(out=out, lse=lse)
    if own:
        return _ops().attn_mass(s["q"], key, s["table"], s["length"], s["lse"], prior=s["prior"], count=s["count"], path=s["path"], window=c["window"] or None,
                                sinks=c["sinks"], out=s["mass"])
    return _plain_mass(s["q"], key, s["table"], s["length"], s["lse"], s["prior"], s["count"], s["path"], window, c["sinks"], lens, s["mass"])


def work(case):
    if case["kind"] == "verify":
        # every logit of the target and the draft; 64-bit exponentials and sums of about 12 operations
        n, rows, vocab = case["seqs"], case["rows"], case["vocab"]
        read = n * vocab * (rows + (rows - 1) * (case["form"] == "chain"))
        return dict(bytes=read * DT[case["dt"]].itemsize + n * (rows * 20 + 12), flops=12 * read)
    lens, page, row = _lengths(case), case["page"], 2 * case["dim"]
    if case["kind"] == "evict":
        per = case["layers"] * case["kv_heads"]
        kept = sum(min(n, case["keep"] + case["sinks"] + case["recent"]) for n in lens)
        return dict(bytes=per * (4 * sum(lens) + kept * (4 * row + 8) + kept // page * row), flops=per * kept * case["dim"])
    rows, heads, hk, dim, sinks = case["rows"], case["heads"], case["kv_heads"], case["dim"], case["sinks"]
    window = case["window"] or 1 << 30
    pairs = tokens = 0
    for n in lens:
        tokens += min(n + rows, min(sinks, n) + min(n, window) + rows)
        # a tree's rows have about half of the rows as ancestors, as a chain's on average
        pairs += sum(min(n + r + 1, min(sinks, n) + window) for r in (range(rows) if not case["tree"] else [rows // 2] * rows))
    inout = case["seqs"] * rows * heads * (row * 2 + 4)
    if case["kind"] == "window":
        return dict(bytes=inout + tokens * hk * row * 2, flops=4 * pairs * heads * dim)
    share = 1.0 if not case["tree"] else 0.4  # (of a tree's rows, the accepted ones)
    return dict(bytes=int(inout * share) // 2 + tokens * hk * row + sum(n + rows for n in lens) * hk * 8, flops=int(2 * pairs * share) * heads * dim)


# ---- the definitions in 64 bits ---------------------------------------------------------------------
def _exact_verify(case, seed):
    """Sequence by sequence: the walk from the root, one distribution at a time, and the drawn token by a search."""
    s = prepare(case, seed)
    n, rows = case["seqs"], case["rows"]
    counts, paths, answers = [], [], []
    for b in range(n):
        heat = float(s["heat"][b])
        soft = lambda x: torch.softmax(x.double() / heat, 0)  # noqa: E731
        token, u = s["tokens"][b].tolist(), s["uniform"][b].tolist()
        parent = s["parent"][b].tolist() if s["parent"] is not None else [r - 1 for r in range(rows)]
        line, at = [0], 0
        while True:
            p = soft(s["logits"][b, at])
            children = [r for r in range(1, rows) if parent[r] == at]
            step = None
            if case["form"] == "chain":
                if children:
                    q = soft(s["draft"][b, at])
                    if u[at] * float(q[token[at + 1]]) < float(p[token[at + 1]]):
                        step = at + 1
                    else:
                        p = torch.relu(p - q)
            else:
                passed = 0.0
                for r in children:
                    passed += float(p[token[r]])
                    if u[at] < passed:
                        step = r
                        break
                    p[token[r]] = 0.0
            if step is None:
                break
            at = step
            line.append(at)
        sums = torch.cumsum(p, 0)
        answers.append(int(torch.searchsorted(sums, (u[rows] * sums[-1]).reshape(1), right=True)))
        counts.append(len(line))
        paths.append(line + [-1] * (rows - len(line)))
    return dict(count=torch.tensor(counts, dtype=torch.int32, device=DEV), path=torch.tensor(paths, dtype=torch.int32, device=DEV), token=torch.tensor(answers, device=DEV))


def exact(case, seed):
    """Attention and weights sequence by sequence and head by head in float64, over the tokens a row attends by their
    positions; mean keys row by row. Moved rows and bookkeeping are whole numbers: nothing to compute."""
    if case["kind"] == "verify":
        return _exact_verify(case, seed)
    s = prepare(case, seed)
    page, hk, lens = case["page"], case["kv_heads"], _lengths(case)
    if case["kind"] == "evict":
        # the lowest free pages are the copies', in the sequences' order
        ksum, free = s["ksum"].double(), [i for i, r in enumerate(s["refs"].tolist()) if r == 0]
        most = case["keep"] + case["sinks"] + case["recent"]
        for b, n in enumerate(lens):
            total = -(-(min(n, most) + case["room"]) // page)
            mine, free = free[:total], free[total:]
            pages = s["table"][b].long()
            for l in range(case["layers"]):
                for h in range(hk):
                    worth = s["mass"][l, b, h, :n].double()
                    order = torch.argsort(-worth, stable=True)
                    order = order[(order >= case["sinks"]) & (order < n - case["recent"])][:case["keep"]]
                    forced = torch.arange(n, device=DEV)
                    forced = forced[(forced < case["sinks"]) | (forced >= n - case["recent"])]
                    stay = torch.cat([forced, order]).unique() if n > most else torch.arange(n, device=DEV)
                    keys = s["kv"][l, 0, h, pages[stay // page], stay % page].double()
                    whole = stay.numel() // page
                    ksum[l, h, mine[:whole]] = keys[:whole * page].reshape(whole, page, case["dim"]).sum(1) / page
        return dict(kv=None, ksum=ksum, mass=None, table=None, length=None, refs=None, kept=None, made=None, gone=None)
    heads, dim, rows, sinks = case["heads"], case["dim"], case["rows"], case["sinks"]
    window, groups = case["window"] or 1 << 30, heads // hk
    out = torch.zeros(case["seqs"], rows, heads, dim, dtype=torch.float64, device=DEV)
    lse = torch.full((case["seqs"], rows, heads), -math.inf, dtype=torch.float64, device=DEV)
    mass = s["mass"].double() if case["kind"] == "mass" else None
    for b, n in enumerate(lens):
        t = torch.arange(n + rows, device=DEV)
        line = [list(range(r + 1)) for r in range(rows)]  # a row's own tokens, in order
        take, live = list(range(rows)), rows
        if case["kind"] == "mass" and s["path"] is not None:
            live = int(s["count"][b])
            take = s["path"][b].tolist()[:live]
        elif s["mask"] is not None:
            line = [[j for j in range(rows) if int(m) >> j & 1] for m in s["mask"][b].tolist()]
        allowed = torch.zeros(live, n + rows, dtype=torch.bool, device=DEV)
        for r in range(live):
            c = n + len(line[r])
            allowed[r, max(0, c - window):n] = True
            allowed[r, :min(sinks, n)] = True
            chosen = [n + j for i, j in enumerate(line[r]) if n + i < sinks or n + i >= c - window]
            allowed[r, chosen] = True
        pages = s["table"][b].long()[t // page]
        if mass is not None:
            mass[b, :, :n] = s["prior"][b, :, :n].double()
            mass[b, :, n:n + live] = 0
        for g in range(hk):
            k = s["kv"][0, 0, g, pages, t % page].double()
            v = s["kv"][0, 1, g, pages, t % page].double()
            for h in range(g * groups, (g + 1) * groups):
                z = (s["q"][b, take, h].double() @ k.T) / math.sqrt(dim)
                z = z.masked_fill(~allowed, -math.inf)
                if mass is not None:
                    mass[b, g, :n + live] += torch.exp(z - s["lse"][b, take, h].double()[:, None])[:, :n + live].sum(0)
                    continue
                lse[b, :, h] = torch.logsumexp(z, 1)
                out[b, :, h] = torch.softmax(z, 1).nan_to_num(0.0) @ v
    return mass if mass is not None else dict(out=out, lse=lse)
