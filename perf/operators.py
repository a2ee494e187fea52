"""The paged cache of several sequences and the attention that reads it, as cases to be measured: sequences forked, copied
and dropped (page_fork), a verified tree's rows committed (page_commit), attention of decode rows, drafted trees and prompt
rows over pages (attn_paged), and the same over the blocks of a long context that a cheap score selects (attn_blocks).

The cache: kv [layers, 2, kv_heads, pages, T, D] (keys, values), a sequence's pages in table [sequences, W] (-1: none), its
committed tokens in length, the references to a page in refs (0: free), and every full page's mean key in ksum
[layers, kv_heads, pages, D]. Where `own` is false, run() computes the operators from elementary torch operations in 32 bits
(block scores in 64: a selection goes by their order) and rounds once; where it is true it calls mdx._C.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

DEV = "cuda"
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
HEADS = ((32, 8, 128), (16, 4, 256), (16, 8, 64), (32, 4, 128))  # q heads, kv heads, head_dim of the configurations and tests


# ---- the cases -------------------------------------------------------------------------------------
def listed():
    return [
        # four sequences continue as one more each (sampling a second answer): full pages shared, four tails copied
        dict(name="fork_tails", kind="fork", layers=8, kv_heads=8, dim=128, page=64, seqs=4, ctx=700, share=True, room=8, dt="bf16"),
        # two prompts copied whole, to be edited apart: the largest move of pages
        dict(name="fork_copy_4k", kind="fork", layers=8, kv_heads=4, dim=256, page=128, seqs=2, ctx=4097, share=False, room=8, dt="bf16"),
        # the accepted rows of an 8-row verify in each of 32 sequences, all layers: rows closed up, pages that filled summed up
        dict(name="commit_tree", kind="commit", layers=8, kv_heads=8, dim=128, page=64, seqs=32, ctx=1000, rows=8, tree=True, dt="bf16"),
        # three prompts' rows become committed: the mean keys of all their pages
        dict(name="commit_prompts", kind="commit", layers=8, kv_heads=4, dim=256, page=32, seqs=3, ctx=37, rows=4001, tree=False, dt="bf16"),
        # one token of one sequence: the smallest call, head_dim 64, fp16
        dict(name="decode_1", kind="paged", heads=16, kv_heads=8, dim=64, page=16, seqs=1, rows=1, lo=513, hi=513, tree=False, dt="fp16"),
        # a tree of 16 drafted rows over one sequence, the hybrid stack's heads
        dict(name="verify_16x1", kind="paged", heads=32, kv_heads=8, dim=128, page=64, seqs=1, rows=16, lo=2048, hi=2048, tree=True, dt="bf16"),
        # a serving batch: single tokens of 64 sequences of unequal lengths
        dict(name="decode_64", kind="paged", heads=32, kv_heads=8, dim=128, page=64, seqs=64, rows=1, lo=100, hi=8191, tree=False, dt="bf16"),
        # trees of 8 drafted rows of 16 sequences, head_dim 256, short pages
        dict(name="verify_8x16_d256", kind="paged", heads=16, kv_heads=4, dim=256, page=16, seqs=16, rows=8, lo=1000, hi=8001, tree=True, dt="bf16"),
        # 2048 rows of a prompt behind a cached prefix
        dict(name="prompt_2k", kind="paged", heads=32, kv_heads=8, dim=128, page=64, seqs=1, rows=2048, lo=1000, hi=1000, tree=False, dt="bf16"),
        # one token of a sequence of 131000 tokens that attends 34 blocks of 64
        dict(name="blocks_1_128k", kind="blocks", heads=32, kv_heads=8, dim=128, page=64, seqs=1, rows=1, lo=131000, hi=131000, blocks=31, sink=1, local=2, tree=False, dt="bf16"),
        # single tokens of 16 sequences of up to 32 thousand tokens
        dict(name="blocks_16_32k", kind="blocks", heads=32, kv_heads=4, dim=128, page=32, seqs=16, rows=1, lo=3000, hi=32767, blocks=60, sink=1, local=3, tree=False, dt="bf16"),
        # trees of 8 drafted rows of 4 sequences, each row with a selection of its own, head_dim 256
        dict(name="blocks_8x4_d256", kind="blocks", heads=16, kv_heads=4, dim=256, page=64, seqs=4, rows=8, lo=9000, hi=16001, blocks=13, sink=1, local=2, tree=True, dt="bf16"),
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(("fork", "commit", "paged", "paged", "paged", "blocks", "blocks"))
    heads, kv_heads, dim = rng.choice(HEADS)
    page = rng.choice((16, 32, 64, 128))
    dt = rng.choice(("bf16", "bf16", "fp16"))
    case = dict(kind=kind, kv_heads=kv_heads, dim=dim, page=page, dt=dt)
    if kind == "fork":
        share = rng.random() < 0.6
        return dict(case, layers=rng.choice((1, 2, 4)), seqs=rng.randint(1, 12 if share else 3), ctx=log_int(1, 2500), share=share, room=rng.randint(1, 64))
    if kind == "commit":
        if rng.random() < 0.5:
            return dict(case, layers=rng.choice((2, 4, 8)), seqs=log_int(1, 32), ctx=log_int(1, 1000), rows=rng.randint(2, 16), tree=True)
        return dict(case, layers=rng.choice((2, 4)), seqs=rng.randint(1, 3), ctx=log_int(1, 300), rows=log_int(65, 2500), tree=False)
    if kind == "paged":
        form = rng.choice(("decode", "verify", "prompt"))
        seqs = 1 if form == "prompt" else log_int(1, 32)
        rows = 1 if form == "decode" else rng.randint(2, 16) if form == "verify" else log_int(65, 1000)
        hi = log_int(1, 2000 if form == "prompt" else 8000)
        return dict(case, heads=heads, seqs=seqs, rows=rows, lo=rng.randint(0, hi), hi=hi, tree=form == "verify")
    tree = rng.random() < 0.4
    hi = log_int(page, 16000)
    return dict(case, heads=heads, seqs=rng.randint(1, 4 if tree else 12), rows=rng.randint(2, 8) if tree else 1, lo=rng.randint(1, hi), hi=hi,
                blocks=log_int(1, 1024 // page), sink=rng.randint(0, 2), local=rng.randint(0, 3), tree=tree)


# ---- inputs ----------------------------------------------------------------------------------------
def _lengths(case):
    """The sequences' committed tokens: spread over [lo, hi] (ctx: a little around it), the longest first."""
    n = case["seqs"]
    if "ctx" in case:
        return [max(0, case["ctx"] - (17 * i) % 61 * (i > 0)) for i in range(n)]
    return [case["hi"] - int((case["hi"] - case["lo"]) * (i * 0.6180339887498949 % 1.0)) for i in range(n)]


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _pages_of(case, seed, pages_each, spare, width):
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


def _tree_masks(gen, seqs, rows):
    """Ancestor bit masks int64 [seqs, rows] of random trees: row 0 the root, every other row a child of an earlier one."""
    parent = (torch.rand(seqs, rows, generator=gen, device=DEV) * torch.arange(rows, device=DEV)).long()
    bit = torch.ones(rows, dtype=torch.int64, device=DEV) << torch.arange(rows, device=DEV)
    mask = torch.zeros(seqs, rows, dtype=torch.int64, device=DEV)
    mask[:, 0] = 1
    for r in range(1, rows):
        mask[:, r] = mask.gather(1, parent[:, r:r + 1])[:, 0] | bit[r]
    return mask


def prepare(case, seed):
    gen, dt = _gen(seed), DT[case["dt"]]
    lens, page = _lengths(case), case["page"]
    hk, dim, seqs = case["kv_heads"], case["dim"], case["seqs"]
    length = torch.tensor(lens, dtype=torch.int32, device=DEV)
    s = dict(case=case, length=length)
    if case["kind"] == "fork":
        # the second half of the table's rows are the copies' places, empty before and after a pass
        width = (max(lens) + case["room"]) // page + 2
        each = [-(-n // page) for n in lens] + [0] * seqs
        new = sum(-(-(n + case["room"]) // page) for n in lens)
        s["table"], s["refs"] = _pages_of(case, seed, each, new + 3, width)
        s["length"] = torch.cat([length, torch.zeros_like(length)])
        s["kv"] = _random_kv(gen, case["layers"], hk, s["refs"].numel(), page, dim, dt)
        s["ksum"] = s["kv"][:, 0].float().mean(-2).to(dt)
        s["src"] = torch.arange(seqs, dtype=torch.int32, device=DEV)
        s["dst"] = s["src"] + seqs
        s["none"] = torch.full_like(s["src"], -1)
    elif case["kind"] == "commit":
        rows = case["rows"]
        s["room"] = rows if case["tree"] else 1
        width = (max(lens) + rows + s["room"]) // page + 2
        each = [-(-(n + rows) // page) for n in lens]
        s["table"], s["refs"] = _pages_of(case, seed, each, 2 * seqs + 3, width)
        s["kv"] = _random_kv(gen, case["layers"], hk, s["refs"].numel(), page, dim, dt)
        s["ksum"] = torch.zeros(case["layers"], hk, s["refs"].numel(), dim, dtype=dt, device=DEV)
        s["new_length"] = torch.empty_like(length)
        s["slots"] = torch.empty(seqs, s["room"], dtype=torch.int64, device=DEV)
        if case["tree"]:
            # the accepted paths: row 0 and then rows behind the accepted count, as where the path leaves the first children
            count = 1 + torch.arange(seqs, device=DEV, dtype=torch.int32) * 5 % max(1, rows // 2)
            noise = torch.rand(seqs, rows, generator=gen, device=DEV) + (torch.arange(rows, device=DEV)[None] < count[:, None])
            pick = noise.argsort(1)
            keep = torch.arange(rows, device=DEV)[None] < (count[:, None] - 1)
            rest = torch.where(keep, pick, rows).sort(1).values
            s["path"] = torch.cat([torch.zeros(seqs, 1, dtype=torch.int64, device=DEV), rest], 1)[:, :rows].to(torch.int32).contiguous()
            s["count"] = count
        else:
            s["path"], s["count"] = None, torch.full_like(length, rows) - torch.arange(seqs, device=DEV, dtype=torch.int32) * 3
    else:
        rows = case["rows"]
        each = [-(-(n + rows) // page) for n in lens]
        s["table"], refs = _pages_of(case, seed, each, 3, max(each) + 1)
        s["kv"] = _random_kv(gen, 1, hk, refs.numel(), page, dim, dt)
        s["q"] = (torch.randn(seqs, rows, case["heads"], dim, generator=gen, device=DEV) * 1.5).to(dt)
        s["mask"] = _tree_masks(gen, seqs, rows) if case["tree"] else None
        if case["kind"] == "blocks":
            s["ksum"] = s["kv"][:, 0].float().mean(-2).to(dt)
    return s


# ---- the operators in plain form -------------------------------------------------------------------
def _give_pages(refs, want):
    """Pages for the true places of want [n, W], the lowest free ones in order: (page of each place, rows that got theirs).
    A row is served if it and all rows before it find enough pages."""
    free = (refs == 0).nonzero()[:, 0]
    ok = want.sum(1).cumsum(0) <= free.numel()
    want = want & ok[:, None]
    pages = torch.full(want.shape, -1, dtype=torch.int32, device=DEV)
    pages[want] = free[:int(want.sum())].to(torch.int32)
    return pages, ok


def _plain_fork(kv, ksum, table, length, refs, dst, src, room, share):
    page, width = kv.shape[4], table.shape[1]
    dst, from_ = dst.long(), src.clamp(min=0).long()
    n = torch.where(src >= 0, length[from_], 0)
    j = torch.arange(width, device=DEV)[None]
    full, used, total = n // page, (n + page - 1) // page, (n + room + page - 1) // page
    kept = j < full[:, None] if share else torch.zeros_like(j < full[:, None])
    moved = (j < used[:, None]) & ~kept
    given, ok = _give_pages(refs, (j < total[:, None]) & ~kept)
    rows = table[from_]
    new = torch.where(kept, rows, given)
    moved &= ok[:, None]
    a, b = rows[moved].long(), new[moved].long()
    kv[:, :, :, b] = kv[:, :, :, a]
    if not share:
        ksum[:, :, b] = ksum[:, :, a]
    old = table[dst[ok]]
    one = torch.ones((), dtype=torch.int32, device=DEV)
    refs.index_put_((new[ok][new[ok] >= 0].long(),), one, accumulate=True)
    refs.index_put_((old[old >= 0].long(),), -one, accumulate=True)
    table[dst[ok]] = new[ok]
    length[dst[ok]] = n[ok].to(torch.int32)
    return ok.to(torch.int32)


def _place(table, pos, page):
    """Pages and rows of the positions pos [n, r] of the n sequences."""
    return table.gather(1, (pos // page).clamp(max=table.shape[1] - 1)).long(), pos % page


def _plain_commit(kv, ksum, table, length, refs, count, path, room, new_length, slots):
    page, width = kv.shape[4], table.shape[1]
    n, new = length.long(), (length + count).long()
    if path is not None:
        k = torch.arange(path.shape[1], device=DEV)[None]
        live = (k < count[:, None]) & (path != k)
        b, r = live.nonzero(as_tuple=True)
        a_page, a_row = _place(table, n[:, None] + path.clamp(max=path.shape[1] - 1), page)
        b_page, b_row = _place(table, n[:, None] + k, page)
        kv[:, :, :, b_page[b, r], b_row[b, r]] = kv[:, :, :, a_page[b, r], a_row[b, r]]
    j = torch.arange(width, device=DEV)[None]
    filled = table[(j >= (n // page)[:, None]) & (j < (new // page)[:, None])].long()
    ksum[:, :, filled] = kv[:, 0][:, :, filled].float().mean(-2).to(ksum.dtype)
    want = (j >= (n // page)[:, None]) & (j < (-(-(new + room) // page))[:, None]) & (table < 0)
    pages, ok = _give_pages(refs, want)
    table.copy_(torch.where(want & ok[:, None], pages, table))
    refs[pages[pages >= 0].long()] = 1
    new_length.copy_(new)
    p, r = _place(table, new[:, None] + torch.arange(room, device=DEV)[None], page)
    slots.copy_(torch.where(p >= 0, p * page + r, -1))
    return ok.to(torch.int32)


def _softmax_rows(scores, admitted, v):
    """softmax(scores over the admitted places) v, 0 for a row that admits none."""
    scores = scores.masked_fill(~admitted, -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    return (e @ v) / torch.where(total == 0, 1.0, total)


def _tree_admits(pos, rows, mask):
    """Which of the positions behind the committed tokens (pos >= 0 their number, any shape [n, ..., t]) each row [n, rows]
    attends: bool [n, rows, t]; without masks a chain."""
    r = torch.arange(rows, device=DEV)
    if mask is None:
        return (pos[:, None, :] >= 0) & (pos[:, None, :] <= r[None, :, None])
    bits = (mask[:, :, None] >> pos.clamp(0, 63)[:, None, :]) & 1
    return (pos[:, None, :] >= 0) & (pos[:, None, :] < rows) & (bits == 1)


def _plain_paged(q, key, value, table, length, mask, reach):
    n, rows, heads, dim = q.shape
    hk, _, page, _ = key.shape
    idx = table[:, :-(-reach // page)].clamp(min=0).long()
    t = idx.shape[1] * page
    k = key[:, idx].float().reshape(hk, n, t, dim)
    v = value[:, idx].float().reshape(hk, n, t, dim)
    pos = torch.arange(t, device=DEV)[None] - length[:, None].long()
    admitted = (pos < 0)[:, None, :] | _tree_admits(pos, rows, mask)  # [n, rows, t]
    admitted = admitted[:, :, None, :].expand(n, rows, heads // hk, t).reshape(n, -1, t)
    qg = q.float().reshape(n, rows, hk, heads // hk, dim).permute(2, 0, 1, 3, 4).reshape(hk, n, -1, dim)
    o = _softmax_rows(qg @ k.transpose(-1, -2) * dim ** -0.5, admitted[None], v)
    return o.reshape(hk, n, rows, heads // hk, dim).permute(1, 2, 0, 3, 4).reshape(n, rows, heads, dim).to(q.dtype)


def _plain_blocks(q, key, value, ksum, table, length, blocks, sink, local, mask, reach):
    n, rows, heads, dim = q.shape
    hk, _, page, _ = key.shape
    groups, most = heads // hk, sink + local + blocks
    idx = table[:, :max(1, -(-reach // page))].clamp(min=0).long()
    w = idx.shape[1]
    whole = (length // page).long()  # the full pages: what is selected from
    qs = q.double().reshape(n, rows, hk, groups, dim).sum(3).permute(2, 0, 1, 3)
    score = qs @ ksum[:, idx].double().transpose(-1, -2)  # [hk, n, rows, w]
    j = torch.arange(w, device=DEV)[None]
    in_ = j < whole[:, None]
    forced = in_ & ((j < sink) | (j >= whole[:, None] - local))
    score = score.masked_fill(forced[None, :, None], math.inf).masked_fill(~in_[None, :, None], -math.inf)
    sel = score.sort(dim=-1, descending=True, stable=True).indices[..., :most]
    sel = torch.where(sel < whole[None, :, None, None], sel, w).sort(-1).values
    sel = torch.nn.functional.pad(sel, (0, most - sel.shape[-1]), value=w)
    sel = torch.where(sel < w, sel, -1)  # [hk, n, rows, most], ascending, -1 behind
    # the selected pages, then the pages behind the full ones (the tail and the rows' own)
    tail = whole[:, None] + torch.arange(-(-(page - 1 + rows) // page), device=DEV)[None]
    logical = torch.cat([sel, tail[None, :, None].expand(hk, n, rows, -1)], -1)
    at = logical.clamp(0, table.shape[1] - 1)
    pages = table.long()[torch.arange(n, device=DEV)[None, :, None, None], at].clamp(min=0)
    h = torch.arange(hk, device=DEV)[:, None, None, None]
    k = key[h, pages].float().reshape(hk, n, rows, -1, dim)
    v = value[h, pages].float().reshape(hk, n, rows, -1, dim)
    pos = (logical[..., None] * page + torch.arange(page, device=DEV)).reshape(hk, n, rows, -1) - length[None, :, None, None].long()
    live = (logical >= 0)[..., None].expand(*logical.shape, page).reshape(pos.shape)
    tree = pos.clamp(0, 63) if mask is not None else pos
    own_ = (mask[None, :, :, None] >> tree) & 1 == 1 if mask is not None else pos <= torch.arange(rows, device=DEV)[None, None, :, None]
    admitted = live & ((pos < 0) | ((pos >= 0) & (pos < rows) & own_))
    qg = q.float().reshape(n, rows, hk, groups, dim).permute(2, 0, 1, 3, 4)
    o = _softmax_rows(qg @ k.transpose(-1, -2) * dim ** -0.5, admitted[..., None, :], v)
    out = o.permute(1, 2, 0, 3, 4).reshape(n, rows, heads, dim).to(q.dtype)
    return out, sel.permute(1, 2, 0, 3).to(torch.int32)


# ---- one pass ---------------------------------------------------------------------------------------
def _ops():
    at = os.path.join(os.getcwd(), "comfy-mono-decode-xpu_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    from mdx import _C
    return _C


def run(s):
    c = s["case"]
    if c["kind"] == "fork":
        # the copies are made and dropped again: the state is as before, and the copied pages stand in the pool
        to = (s["kv"], s["ksum"], s["table"], s["length"], s["refs"], s["dst"])
        if own:
            made, gone = _ops().page_fork(*to, s["src"], c["room"], c["share"]), _ops().page_fork(*to, s["none"])
        else:
            made, gone = _plain_fork(*to, s["src"], c["room"], c["share"]), _plain_fork(*to, s["none"], 0, True)
        return dict(kv=s["kv"].view(torch.int16), ksum=s["ksum"].view(torch.int16), table=s["table"], length=s["length"], refs=s["refs"], made=made, gone=gone)
    if c["kind"] == "commit":
        a = (s["kv"], s["ksum"], s["table"], s["length"], s["refs"], s["count"], s["path"], s["room"], s["new_length"], s["slots"])
        ok = _ops().page_commit(*a) if own else _plain_commit(*a)
        return dict(kv=s["kv"].view(torch.int16), ksum=s["ksum"], table=s["table"], length=s["new_length"], refs=s["refs"], slots=s["slots"], ok=ok)
    key, value = s["kv"][0, 0], s["kv"][0, 1]
    reach = max(_lengths(c)) + c["rows"]  # what the program knows of its sequences
    if c["kind"] == "paged":
        if own:
            return _ops().attn_paged(s["q"], key, value, s["table"], s["length"], s["mask"])
        return _plain_paged(s["q"], key, value, s["table"], s["length"], s["mask"], reach)
    b = (c["blocks"], c["sink"], c["local"], s["mask"])
    if own:
        return _ops().attn_blocks(s["q"], key, value, s["ksum"][0], s["table"], s["length"], *b)
    return _plain_blocks(s["q"], key, value, s["ksum"][0], s["table"], s["length"], *b, reach)


def work(case):
    lens, page, row = _lengths(case), case["page"], 2 * case["dim"]
    if case["kind"] == "fork":
        # copied pages read and written (with their mean keys where whole pages go), the table's and the references' changes
        moved = sum(-(-n // page) if not case["share"] else int(n % page > 0) for n in lens)
        tokens = case["layers"] * 2 * case["kv_heads"] * page * row
        sums = 0 if case["share"] else case["layers"] * case["kv_heads"] * row
        entries = sum(-(-(n + case["room"]) // page) for n in lens)
        return dict(bytes=2 * moved * (tokens + sums) + 4 * 12 * entries, flops=0)
    if case["kind"] == "commit":
        rows, seqs = case["rows"], case["seqs"]
        per_row = case["layers"] * case["kv_heads"] * row
        count = [1 + i * 5 % max(1, rows // 2) if case["tree"] else rows - 3 * i for i in range(seqs)]
        moved = sum(k - 1 for k in count) if case["tree"] else 0
        filled = sum((n + k) // page - n // page for n, k in zip(lens, count))
        return dict(bytes=moved * 4 * per_row + filled * (page + 1) * per_row + seqs * (16 + 8 * rows * case["tree"]), flops=filled * page * per_row // 2)
    rows, heads, hk, dim = case["rows"], case["heads"], case["kv_heads"], case["dim"]
    inout = case["seqs"] * rows * heads * row * 2
    if case["kind"] == "paged":
        chain = 1 if not case["tree"] else 0  # a chain's row attends half of the rows, a tree's about as many
        pairs = sum(rows * n + rows * (rows + chain) // 2 for n in lens)
        return dict(bytes=inout + sum((n + rows) * hk * row * 2 + 4 * (-(-(n + rows) // page)) for n in lens), flops=4 * pairs * heads * dim)
    # blocks: every full page's mean key, the tokens of each row's selection (at least once per sequence and kv head)
    most = case["sink"] + case["local"] + case["blocks"]
    got = [min(n // page, most) * page + n % page for n in lens]
    means = sum(n // page for n in lens) * hk * row
    kv = sum(min(n, g * rows) + rows for n, g in zip(lens, got)) * hk * row * 2
    return dict(bytes=inout + means + kv + case["seqs"] * rows * hk * most * 4,
                flops=sum(rows * (4 * (g + (rows + 1) / 2) * heads * dim + 2 * (n // page) * hk * dim) for n, g in zip(lens, got)))


# ---- the definitions in 64 bits ---------------------------------------------------------------------
def exact(case, seed):
    """Sequence by sequence and row by row: the tokens a row admits gathered by position, softmax over them in float64.
    Moved pages and bookkeeping are whole numbers: nothing to compute."""
    if case["kind"] == "fork":
        return None
    s = prepare(case, seed)
    page = case["page"]
    if case["kind"] == "commit":
        ksum, n = s["ksum"].double(), s["length"].tolist()
        kv, table, count = s["kv"], s["table"].tolist(), s["count"].tolist()
        for b in range(case["seqs"]):
            order = s["path"][b].tolist() if case["tree"] else None
            for j in range(n[b] // page, (n[b] + count[b]) // page):
                keys = []
                for pos in range(j * page, (j + 1) * page):
                    if order is not None and pos >= n[b]:
                        pos = n[b] + order[pos - n[b]]
                    keys.append(kv[:, 0, :, table[b][pos // page], pos % page])
                total = keys[0].double()
                for key in keys[1:]:
                    total = total + key.double()
                ksum[:, :, table[b][j]] = total / page
        return dict(kv=None, ksum=ksum, table=None, length=None, refs=None, slots=None, ok=None)
    heads, hk, dim, rows = case["heads"], case["kv_heads"], case["dim"], case["rows"]
    lens, groups = _lengths(case), heads // hk
    out = torch.zeros(case["seqs"], rows, heads, dim, dtype=torch.float64, device=DEV)
    for b in range(case["seqs"]):
        n = lens[b]
        at = torch.arange(n + rows, device=DEV)
        pages = s["table"][b].long()[at // page]
        mask = s["mask"][b].tolist() if s["mask"] is not None else [(2 << r) - 1 for r in range(rows)]
        if case["kind"] == "paged" and s["mask"] is None:
            seen = at[None] <= n + torch.arange(rows, device=DEV)[:, None]
        else:
            own_ = torch.tensor([[i < n or bool(m >> (i - n) & 1) for i in (0, *range(n, n + rows))] for m in mask], device=DEV)
            seen = torch.cat([torch.ones(rows, n, dtype=torch.bool, device=DEV), own_[:, 1:]], 1)
        for g in range(hk):
            k = s["kv"][0, 0, g, pages, at % page].double()
            v = s["kv"][0, 1, g, pages, at % page].double()
            allowed = seen
            if case["kind"] == "blocks":
                whole = n // page
                means = s["ksum"][0, g, s["table"][b, :whole].long()].double()
                allowed = seen.clone()
                for r in range(rows):
                    want = set(range(min(case["sink"], whole))) | set(range(max(0, whole - case["local"]), whole))
                    worth = (means * s["q"][b, r, g * groups:(g + 1) * groups].double().sum(0)).sum(1).tolist()
                    left = sorted((i for i in range(whole) if i not in want), key=lambda i: (-worth[i], i))
                    want |= set(left[:max(0, case["sink"] + case["local"] + case["blocks"] - len(want))])
                    has = torch.zeros(whole + 1 + (rows + page) // page, dtype=torch.bool)
                    has[sorted(want)] = True
                    has[whole:] = True
                    allowed[r] &= has.to(DEV)[at // page]
            for h in range(g * groups, (g + 1) * groups):
                z = (s["q"][b, :, h].double() @ k.T) / math.sqrt(dim)
                w = torch.softmax(z.masked_fill(~allowed, -math.inf), 1)
                out[b, :, h] = w @ v
    return (out, None) if case["kind"] == "blocks" else out
