"""attn_blocks on the GPU: the selection equal to the oracle's, the attention over it within the float64 bound; and a run of the
paged cache's operators together against a plain contiguous sequence."""
import numpy as np
import pytest
import torch

from oracle import ref
from paged_cases import cache, check, f64, tree_masks

pytestmark = pytest.mark.gpu
BF, FH = torch.bfloat16, torch.float16


def _means(key, table, lens, T, dt):
    """Mean keys of the full pages, junk elsewhere."""
    ks = torch.full((key.shape[0], key.shape[1], key.shape[3]), float("nan"))
    for b, n in enumerate(lens):
        for j in range(n // T):
            ks[:, table[b, j]] = key[:, table[b, j]].double().mean(1).float()
    return ks.to(dt)


def _run(C, dev, dt, H, Hk, D, T, lens, S, tree, blocks, sink, local, seed=0, edit=None):
    print(f"attn_blocks {dt} H={H} Hk={Hk} D={D} T={T} lens={lens} S={S} tree={tree} blocks={blocks} sink={sink} local={local}", flush=True)
    g = torch.Generator().manual_seed(seed + D + T + S)
    key, value, table = cache(g, dt, Hk, T, D, lens, S)
    q = (torch.randn(len(lens), S, H, D, generator=g) * 1.5).to(dt)
    mask = tree_masks(g, len(lens), S) if tree else None
    ksum = _means(key, table, lens, T, dt)
    if edit:
        edit(q, key, value, table, ksum)
    n = torch.tensor(lens, dtype=torch.int32, device=dev)
    args = [x.to(dev) for x in (q, key, value, ksum, table)] + [n, blocks, sink, local, None if mask is None else mask.to(dev)]
    got, sel = C.attn_blocks(*args)
    want = ref.block_selection(f64(q), f64(ksum), table.numpy(), lens, T, blocks, sink, local)
    assert sel.dtype == torch.int32 and np.array_equal(sel.cpu().numpy(), want)

    def keep(b, s, kh, pos):
        return (pos >= lens[b] // T * T) | np.isin(pos // T, want[b, s, kh])
    check(got, dt, q, key, value, table, lens, mask, D ** -0.5, keep)
    return args, got, sel


@pytest.mark.parametrize("dt", [BF, FH])
@pytest.mark.parametrize("H,Hk,D", [(32, 8, 128), (16, 4, 256), (16, 8, 64), (32, 4, 128), (40, 2, 64), (64, 1, 128)])
def test_single_tokens(C, dev, dt, H, Hk, D):
    _run(C, dev, dt, H, Hk, D, 16, [0, 5, 16, 200, 333, 64], 1, False, 4, 1, 2)


@pytest.mark.parametrize("blocks,sink,local", [(0, 1, 0), (0, 0, 1), (1, 0, 0), (7, 0, 3), (30, 5, 5), (3, 40, 0), (0, 2, 3)])
def test_selections(C, dev, blocks, sink, local):
    _run(C, dev, BF, 8, 2, 64, 16, [700, 31, 16 * (blocks + sink + local), 16 * (blocks + sink + local + 1) + 9], 1, False, blocks, sink, local, 3)


@pytest.mark.parametrize("T", [16, 32, 128])
@pytest.mark.parametrize("H,Hk,D,S", [(8, 2, 128, 5), (8, 4, 256, 9), (4, 4, 64, 64)])
def test_trees(C, dev, T, H, Hk, D, S):
    """Every row with a selection of its own, masks over the rows' own tokens."""
    _run(C, dev, BF, H, Hk, D, T, [9 * T + 3, 0, 4 * T], S, True, 2, 1, 1, 4)


def test_chain_rows(C, dev):
    _run(C, dev, BF, 8, 2, 128, 32, [500, 40], 6, False, 3, 1, 1, 5)


@pytest.mark.parametrize("pages", [1024, 1025, 3000, 5000, 17000])
def test_many_pages(C, dev, pages):
    """Every size class of the selection, a full table and a short sequence in it."""
    _run(C, dev, BF, 4, 1, 64, 16, [16 * (pages - 1) + 7, 16 * 150], 1, False, 40, 1, 2, 6)


@pytest.mark.parametrize("pages", [900, 3000, 17000])
@pytest.mark.parametrize("levels", [1, 2, 5])
def test_few_levels_of_scores(C, dev, pages, levels):
    """More equal scores at the threshold than one work-group's threads; scores that share all but their last bits."""
    def edit(q, key, value, table, ksum):
        q.fill_(1.0)
        ksum.zero_()
        ksum[:, table[0].long().clamp(min=0), 0] = (torch.arange(table.shape[1]) * 7 % levels).float().to(BF)
        ksum[:, table[0, 500], 1] = 2.0 ** -40
        ksum[:, table[0, 700], 1] = -(2.0 ** -40)
    _run(C, dev, BF, 4, 2, 64, 16, [16 * (pages - 1) + 3], 1, False, 450, 1, 1, 13, edit)


@pytest.mark.parametrize("equal", [1.0, 0.0])
def test_ties_go_to_the_lowest_page(C, dev, equal):
    def edit(q, key, value, table, ksum):
        ksum[:] = equal
        ksum[:, table[0, 9]] = 2.0
        q.fill_(1.0)
    _, _, sel = _run(C, dev, BF, 8, 2, 64, 16, [16 * 300], 1, False, 5, 1, 1, 7, edit)
    assert sel[0, 0, 0].tolist() == [0, 1, 2, 3, 4, 9, 299]


def test_scores_of_either_sign_and_zero(C, dev):
    """-0 and 0 are one score; scores that differ in the last bits of float32 keep their order."""
    def edit(q, key, value, table, ksum):
        q.fill_(0)
        q[..., 0] = 1.0
        q[..., 1] = 2.0 ** -30
        ksum[:] = 0.0
        pages = table[0].long()
        ksum[:, pages[1:20], 0] = -1.0
        ksum[:, pages[20:40], 0] = 1.0
        ksum[:, pages[30], 1] = 1.0
        ksum[:, pages[25], 1] = -1.0
        ksum[:, pages[45], 0] = -0.0
    _, _, sel = _run(C, dev, BF, 4, 4, 64, 16, [16 * 60], 1, False, 20, 0, 1, 8, edit)
    assert sel[0, 0, 0].tolist() == list(range(20, 40)) + [59]
    _, _, sel = _run(C, dev, BF, 4, 4, 64, 16, [16 * 60], 1, False, 1, 0, 1, 8, edit)
    assert sel[0, 0, 0].tolist() == [30, 59]


def test_nan_scores_and_bad_pages_come_last(C, dev):
    def edit(q, key, value, table, ksum):
        ksum[:, table[0, 3]] = float("nan")
        ksum[:, table[0, 5]] = float("inf")
        q[..., :] = q.abs()
        table[0, 7] = -1
        table[0, 8] = 10 ** 6
    _, _, sel = _run(C, dev, BF, 8, 2, 64, 16, [16 * 12 + 3], 1, False, 8, 0, 0, 9, edit)
    assert all(5 in x and not {3, 7, 8} & set(x) for x in sel[0, 0].tolist())


def test_dense_when_everything_fits(C, dev):
    """All full pages selected: attn_paged's result (the same tokens; another split of the sums)."""
    args, got, _ = _run(C, dev, BF, 8, 2, 128, 16, [100, 40, 0], 3, True, 10, 1, 1, 10)
    q, key, value, ksum, table, n = args[:6]
    dense = C.attn_paged(q, key, value, table, n, args[9])
    assert (dense.float() - got.float()).abs().max() <= 2.0 ** -6 * dense.float().abs().max()


def test_non_finite_in_unselected_pages(C, dev):
    def edit(q, key, value, table, ksum):
        for j in range(1, 20):
            if j % 2:
                key[:, table[0, j]] = float("nan")
                value[:, table[0, j]] = float("inf")
                ksum[:, table[0, j]] = -100.0
            else:
                ksum[:, table[0, j]] = 100.0
        q.copy_(q.abs())
    _run(C, dev, BF, 8, 2, 64, 16, [16 * 20 + 5], 1, False, 8, 1, 0, 11, edit)


def test_graph_replay(C, dev):
    args, got, sel = _run(C, dev, BF, 8, 2, 128, 16, [900, 300, 31], 2, True, 6, 1, 1, 12)
    n = args[5]
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out, s2 = C.attn_blocks(*args)
    for lens in ((900, 300, 31), (100, 0, 3), (899, 170, 16), (900, 300, 31)):
        n.copy_(torch.tensor(lens, dtype=torch.int32))
        gr.replay()
        torch.cuda.synchronize()
        want, s3 = C.attn_blocks(*args)
        assert torch.equal(out, want) and torch.equal(s2, s3)
    assert torch.equal(out, got) and torch.equal(s2, sel)


def test_refusals(C, dev):
    g = torch.Generator().manual_seed(1)
    key, value, table = (x.to(dev) for x in cache(g, BF, 2, 16, 64, [40, 20], 1))
    q, n = torch.randn(2, 1, 4, 64, device=dev).to(BF), torch.tensor([40, 20], dtype=torch.int32, device=dev)
    ks = torch.zeros(2, key.shape[1], 64, dtype=BF, device=dev)
    for args, kw, match in [((q, key, value, ks.half(), table, n, 1), {}, "ksum"), ((q, key, value, ks[:, 1:], table, n, 1), {}, "ksum"),
                            ((q, key, value, ks, table, n, -1), {}, "selected blocks"), ((q, key, value, ks, table, n, 0, 0, 0), {}, "selected blocks"),
                            ((q, key, value, ks, table, n, 1), dict(sel=torch.zeros(2, 1, 2, 4, dtype=torch.int32, device=dev)), "sel"),
                            ((q.expand(2, 65, 4, 64), key, value, ks, table, n, 1), {}, "64 rows")]:
        with pytest.raises(RuntimeError, match=match):
            C.attn_blocks(*args, **kw)


def test_a_run_of_the_operators_together(C, dev):
    """Prompts into pages through the RoPE / KV operator's slots, committed, forked, decoded with drafted trees of which a path is
    accepted, over steps; against each sequence kept contiguously on the host. Page tables end as the oracle of lengths says."""
    g = torch.Generator().manual_seed(21)
    L, H, Hk, D, T, P, B, W, S = 2, 8, 2, 64, 16, 64, 4, 12, 4
    kv = torch.full((L, 2, Hk, P, T, D), float("nan"), dtype=BF, device=dev)
    ksum = torch.full((L, Hk, P, D), float("nan"), dtype=BF, device=dev)
    table = torch.full((B, W), -1, dtype=torch.int32, device=dev)
    length, refs = torch.zeros(B, dtype=torch.int32, device=dev), torch.zeros(P, dtype=torch.int32, device=dev)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    eye = torch.eye(2).reshape(1, 1, 2, 2)

    def write(slots, k, v):
        """k, v [rows, Hk, D] of every layer into the cache rows `slots`, by the RoPE / KV operator without a rotation."""
        for i in range(L):
            for r in range(0, len(slots), 16):
                kk, vv, ss = k[i][r:r + 16].to(dev), v[i][r:r + 16].to(dev), slots[r:r + 16].contiguous()
                freqs = eye.expand(len(ss), D // 2, 2, 2).contiguous().to(dev)
                C.rope_kv(torch.zeros(len(ss), Hk, D, dtype=BF, device=dev), kk, vv, freqs, kv[i, 0].view(1, Hk, P * T, D),
                          kv[i, 1].view(1, Hk, P * T, D), ss, D)

    rows = lambda n: torch.randn(L, n, Hk, D, generator=g).to(BF)  # noqa: E731
    held = {}
    for b, n in ((0, 45), (1, 16)):
        slots = torch.empty(1, n, dtype=torch.int64, device=dev)
        assert C.page_fork(kv, ksum, table, length, refs, i32([b]), i32([-1]), n, True, slots).tolist() == [1]
        k, v = rows(n), rows(n)
        write(slots[0], k, v)
        count = [-1] * B
        count[b] = n
        assert C.page_commit(kv, ksum, table, length, refs, i32(count)).tolist() == [1] * B
        held[b] = [k, v]
    assert C.page_fork(kv, ksum, table, length, refs, i32([2, 3]), i32([0, 1]), 0, True).tolist() == [1, 1]
    held[2], held[3] = [x.clone() for x in held[0]], [x.clone() for x in held[1]]
    slots = torch.empty(B, S, dtype=torch.int64, device=dev)
    C.page_commit(kv, ksum, table, length, refs, i32([0] * B), None, S, None, slots)
    paths = [[0, 1, 2, 3], [0, 2, 3, 9], [0, 3, 9, 9], [0, 9, 9, 9]]
    mask = torch.tensor([[1, 3, 7, 15], [1, 3, 5, 13], [1, 3, 5, 9], [1, 2, 4, 8]])
    for step in range(9):
        accepted = [(step + b) % (b % 3 + 2) % 4 + 1 if b < 3 else 1 for b in range(B)]
        accepted = [min(a, sum(x < 4 for x in p)) for a, p in zip(accepted, paths)]
        draft = [(rows(S), rows(S)) for _ in range(B)]
        for b in range(B):
            write(slots[b], *draft[b])
        lens = [held[b][0].shape[1] for b in range(B)]
        assert length.tolist() == lens
        q = torch.randn(B, S, H, D, generator=g).to(BF)
        seqs = [[torch.cat([held[b][i], draft[b][i]], 1) for i in range(2)] for b in range(B)]
        for i in range(L):
            # the contiguous sequences as a cache of one page each row group, for the oracle
            width = max(lens) + S
            Wc = -(-width // T)
            ck = torch.zeros(2, Hk, B * Wc, T, D, dtype=BF)
            for b in range(B):
                for m in range(2):
                    x = seqs[b][m][i].transpose(0, 1)
                    ck[m][:, b * Wc:(b + 1) * Wc].view(Hk, Wc * T, D)[:, :x.shape[1]] = x
            ct = torch.arange(B * Wc).view(B, Wc).to(torch.int32)
            got = C.attn_paged(q.to(dev), kv[i, 0], kv[i, 1], table, length, mask.to(dev))
            check(got, BF, q, ck[0], ck[1], ct, lens, mask, D ** -0.5)
            got, sel = C.attn_blocks(q.to(dev), kv[i, 0], kv[i, 1], ksum[i], table, length, 1, 1, 0, mask.to(dev))
            means = torch.stack([ksum[i, :, e].cpu() if e >= 0 else torch.zeros(Hk, D, dtype=BF) for e in table.cpu()[:, :Wc].reshape(-1).tolist()], 1)
            if table.shape[1] < Wc:
                raise AssertionError("table")
            want = ref.block_selection(f64(q), f64(means.nan_to_num(0)), ct.numpy(), lens, T, 1, 1, 0)
            assert np.array_equal(sel.cpu().numpy(), want)
            check(got, BF, q, ck[0], ck[1], ct, lens, mask, D ** -0.5,
                  lambda b, s, kh, pos: (pos >= lens[b] // T * T) | np.isin(pos // T, want[b, s, kh]))
        status = C.page_commit(kv, ksum, table, length, refs, i32(accepted), i32(paths), S, None, slots)
        assert status.tolist() == [1] * B
        for b in range(B):
            keep = paths[b][:accepted[b]]
            held[b] = [torch.cat([held[b][m], draft[b][m][:, keep]], 1) for m in range(2)]
            for j in range(held[b][0].shape[1] // T):
                mean = held[b][0][:, j * T:(j + 1) * T].double().mean(1)
                at = ksum[:, :, table[b, j].item()].cpu().double()
                assert (at - mean).abs().max() <= 2.0 ** -7 * mean.abs().max()
    C.page_fork(kv, ksum, table, length, refs, i32([0, 1, 2, 3]), i32([-1] * 4))
    assert (refs == 0).all() and (table == -1).all()


@pytest.mark.parametrize("H,Hk,D,S", [(8, 2, 128, 5), (16, 4, 256, 8), (8, 4, 64, 17), (16, 8, 64, 3)])
def test_trees_fp16(C, dev, H, Hk, D, S):
    """Scores of several rows from fp16 mean keys, selections and attention of each row."""
    _run(C, dev, FH, H, Hk, D, 16, [30 * 16 + 3, 0, 9 * 16, 700], S, True, 5, 1, 2, 14)


def test_chain_rows_fp16(C, dev):
    _run(C, dev, FH, 8, 2, 128, 32, [700, 40], 6, False, 3, 1, 1, 15)


def test_the_most_pages(C, dev):
    """A table of 65536 entries (one of them spare), a million tokens in each sequence."""
    _run(C, dev, BF, 2, 1, 64, 16, [16 * 65534 + 7, 16 * 65533], 1, False, 40, 1, 2, 16)


@pytest.mark.parametrize("H,Hk,D,T,S", [(8, 2, 64, 16, 5), (8, 2, 128, 64, 4), (16, 4, 256, 32, 8), (64, 1, 64, 16, 3), (40, 2, 128, 16, 3)])
def test_values_that_some_rows_attend(C, dev, H, Hk, D, T, S):
    """Infinite values in a page that some selections hold, in the tail and at an own row: in the rows that attend them, no others."""
    g = torch.Generator().manual_seed(S + D)
    n = 20 * T + 5
    key, value, table = cache(g, BF, Hk, T, D, [n], S)
    q = (torch.randn(1, S, H, D, generator=g) * 1.5).to(BF)
    mask = torch.tensor([[(1 << s) | 1 for s in range(S)]])
    ksum = _means(key, table, [n], T, BF)
    dirty = value.clone()
    at = {3: (9 * T + T - 1, "page"), 7: (20 * T + 2, "tail"), 11: (n + 1, "own row 1")}  # dim: token
    for d, (t, _) in at.items():
        dirty[:, table[0, t // T], t % T, d] = float("inf")
    call = lambda v: C.attn_blocks(*(x.to(dev) for x in (q, key, v, ksum, table)), torch.tensor([n], dtype=torch.int32, device=dev), 8, 1, 1, mask.to(dev))  # noqa: E731
    (got, sel), (clean, _) = call(dirty), call(value)
    got, clean, sel = got.cpu(), clean.cpu(), sel.cpu()
    hit = torch.zeros(1, S, H, D, dtype=torch.bool)
    hit[0, :, :, 3] = (sel[0] == 9).any(-1).repeat_interleave(H // Hk, 1)
    hit[..., 7] = True
    hit[0, 1, :, 11] = True
    assert (got[hit] == float("inf")).all() and got[~hit].isfinite().all()
    assert torch.equal(got[~hit], clean[~hit])
