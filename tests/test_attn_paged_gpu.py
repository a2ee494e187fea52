"""attn_paged on the GPU against the float64 oracle (bounds: tests/paged_cases.py), over pages whose unused rows hold NaN."""
import pytest
import torch

from paged_cases import cache, check, tree_masks

pytestmark = pytest.mark.gpu
BF, FH = torch.bfloat16, torch.float16


def _run(C, dev, dt, H, Hk, D, T, lens, S, tree, seed=0, width=1):
    print(f"attn_paged {dt} H={H} Hk={Hk} D={D} T={T} lens={lens} S={S} tree={tree} width={width}", flush=True)
    g = torch.Generator().manual_seed(seed + D + T + S)
    key, value, table = cache(g, dt, Hk, T, D, lens, S, width=width)
    q = (torch.randn(len(lens), S, H, D, generator=g) * 1.5).to(dt)
    mask = tree_masks(g, len(lens), S) if tree else None
    n = torch.tensor(lens, dtype=torch.int32, device=dev)
    got = C.attn_paged(q.to(dev), key.to(dev), value.to(dev), table.to(dev), n, None if mask is None else mask.to(dev))
    check(got, dt, q, key, value, table, lens, mask, D ** -0.5)


@pytest.mark.parametrize("dt", [BF, FH])
@pytest.mark.parametrize("H,Hk,D", [(32, 8, 128), (16, 4, 256), (16, 8, 64), (32, 4, 128), (3, 3, 64), (7, 1, 128), (5, 1, 256)])
def test_single_tokens(C, dev, dt, H, Hk, D):
    _run(C, dev, dt, H, Hk, D, 16, [0, 1, 15, 16, 17, 31, 32, 33, 127, 128, 300], 1, False)


@pytest.mark.parametrize("T", [16, 32, 64, 128, 1024])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_page_sizes(C, dev, T, D):
    _run(C, dev, BF, 8, 2, D, T, [T - 1, T, T + 1, 3 * T + 5, 0], 3, True, T)


@pytest.mark.parametrize("H,Hk,D,S", [(32, 8, 128, 16), (16, 4, 256, 8), (16, 4, 256, 16), (16, 4, 256, 17), (16, 8, 64, 9), (32, 8, 128, 17),
                                      (32, 4, 128, 64), (8, 8, 64, 64), (4, 4, 256, 63), (4, 1, 128, 33), (12, 4, 64, 5)])
@pytest.mark.parametrize("dt", [BF, FH])
def test_trees(C, dev, dt, H, Hk, D, S):
    _run(C, dev, dt, H, Hk, D, 64, [0, 70, 257], S, True, H)


@pytest.mark.parametrize("H,Hk,D,S", [(32, 8, 128, 1), (32, 8, 128, 5), (32, 8, 128, 16), (16, 4, 256, 3), (16, 4, 256, 8), (16, 4, 256, 16),
                                      (16, 8, 64, 3), (16, 8, 64, 12), (16, 8, 64, 30), (8, 8, 256, 64)])
@pytest.mark.parametrize("dt", [BF, FH])
@pytest.mark.parametrize("width", [12, 6000])
def test_tables_wider_than_the_sequences(C, dev, dt, H, Hk, D, S, width):
    """The forms go by what the table could hold: the same rows through those for much to stream."""
    _run(C, dev, dt, H, Hk, D, 64, [0, 70, 400, 129], S, S > 1, H, width)


@pytest.mark.parametrize("H,Hk,D,S,lens", [(32, 8, 128, 65, [0, 40]), (8, 2, 128, 300, [129]), (4, 1, 256, 130, [7, 64]), (8, 4, 64, 513, [0]),
                                           (6, 2, 128, 100, [33, 0, 1]), (10, 2, 64, 111, [77, 0, 400]), (128, 1, 128, 5, [40]), (100, 1, 64, 3, [0, 70]), (33, 1, 256, 12, [90]),
                                           (14, 2, 256, 41, [65, 3]), (16, 1, 128, 9, [50]), (8, 1, 64, 40, [500, 3])])
def test_chains(C, dev, H, Hk, D, S, lens):
    _run(C, dev, BF, H, Hk, D, 32, lens, S, False, 5)


@pytest.mark.parametrize("D,n", [(128, 5000), (256, 3100), (64, 9001)])
def test_one_long_sequence_among_short_ones(C, dev, D, n):
    """Shares of the line of steps that begin and end inside units, and units of a single step."""
    _run(C, dev, BF, 4, 2, D, 64, [3, n, 0, 40, 1], 2, True, 7)


def test_many_sequences(C, dev):
    g = torch.Generator().manual_seed(2)
    lens = [int(x) for x in torch.randint(0, 90, (300,), generator=g)]
    _run(C, dev, BF, 4, 2, 64, 16, lens, 1, False, 9)


@pytest.mark.parametrize("H,Hk,D,S,B,top,tree", [(4, 2, 64, 1, 300, 90, False), (8, 8, 128, 1, 130, 200, False), (8, 2, 128, 16, 150, 90, True),
                                                 (8, 4, 256, 9, 150, 60, True), (8, 2, 128, 70, 24, 300, False), (16, 8, 64, 100, 40, 70, False)])
def test_more_units_than_work_groups(C, dev, H, Hk, D, S, B, top, tree):
    """Shares of several units, that begin and end in, between and behind the steps of a unit; tables that could hold much more."""
    g = torch.Generator().manual_seed(B)
    lens = [int(x) for x in torch.randint(0, top, (B,), generator=g)]
    _run(C, dev, BF, H, Hk, D, 32, lens, S, tree, 13, 200)


def _small(dev, dt=BF, D=128, H=8, Hk=2, T=16, lens=(40, 0, 33), S=4, seed=11):
    g = torch.Generator().manual_seed(seed)
    lens = list(lens)
    key, value, table = cache(g, dt, Hk, T, D, lens, S)
    q = (torch.randn(len(lens), S, H, D, generator=g) * 1.5).to(dt)
    mask = tree_masks(g, len(lens), S)
    return g, q, key, value, table, lens, torch.tensor(lens, dtype=torch.int32, device=dev), mask


@pytest.mark.parametrize("D", [64, 128, 256])
def test_strides(C, dev, D):
    """A cache of token-major pages, q as a slice of wider rows, a table of wider rows, out given."""
    g, q, key, value, table, lens, n, mask = _small(dev, D=D)
    both = torch.stack([key, value], 0).permute(2, 3, 0, 1, 4).contiguous().to(dev)  # [P, T, 2, Hk, D]
    wide_q = torch.randn(3, 4, 8, 2 * D, generator=g).to(BF)
    wide_q[..., D:] = q
    wide_t = torch.full((3, table.shape[1] + 5), -1, dtype=torch.int32)
    wide_t[:, :table.shape[1]] = table
    out = torch.empty(3, 4, 8, D, dtype=BF, device=dev)
    got = C.attn_paged(wide_q.to(dev)[..., D:], both[:, :, 0].permute(2, 0, 1, 3), both[:, :, 1].permute(2, 0, 1, 3),
                       wide_t.to(dev)[:, :table.shape[1]], n, mask.to(dev), out=out)
    assert got is out
    check(got, BF, q, key, value, table, lens, mask, D ** -0.5)


def test_scale(C, dev):
    _, q, key, value, table, lens, n, mask = _small(dev)
    got = C.attn_paged(q.to(dev), key.to(dev), value.to(dev), table.to(dev), n, mask.to(dev), scale=0.31)
    check(got, BF, q, key, value, table, lens, mask, 0.31)


def test_rows_that_admit_nothing_are_zero(C, dev):
    _, q, key, value, table, lens, n, mask = _small(dev)
    mask[1, 2] = 0
    mask[2, 1] = 0
    got = C.attn_paged(q.to(dev), key.to(dev), value.to(dev), table.to(dev), n, mask.to(dev))
    assert (got[1, 2] == 0).all() and (got[2, 1] != 0).any()
    check(got, BF, q, key, value, table, lens, mask, 128 ** -0.5)


@pytest.mark.parametrize("T,S", [(16, 4), (64, 20)])
def test_bad_pages_are_not_attended(C, dev, T, S):
    """Entries that are no page (negative, past the pool) inside and behind the prefix, a sequence without pages, lengths out of
    range: nothing of them is read, the other tokens count as ever."""
    g, q, key, value, table, lens, n, mask = _small(dev, T=T, lens=(5 * T + 3, T, 2 * T, 0), S=S)
    P = key.shape[1]
    table[0, 1], table[0, 3], table[1, 0], table[2] = -7, P, 2 ** 31 - 1, -1
    table[3, 0] = P + 3
    got = C.attn_paged(q.to(dev), key.to(dev), value.to(dev), table.to(dev), n, mask.to(dev))
    check(got, BF, q, key, value, table, lens, mask, 128 ** -0.5)
    assert (got[2] == 0).all() and (got[3] == 0).all()
    n2 = torch.tensor([-5, 2 ** 31 - 1, -2 ** 31, 0], dtype=torch.int32, device=dev)
    W = table.shape[1]
    got = C.attn_paged(q.to(dev), torch.zeros_like(key).to(dev), torch.ones_like(value).to(dev), table.to(dev), n2, mask.to(dev))
    assert got.isfinite().all()
    assert W * T < 2 ** 30


@pytest.mark.parametrize("dt", [BF, FH])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("bad,width", [(float("nan"), 1), (float("inf"), 1), (float("-inf"), 1), (float("nan"), 40), (float("nan"), 20000)])
def test_non_finite_in_places_that_are_not_admitted(C, dev, dt, D, bad, width):
    """K and V of one own row non-finite: the rows that do not admit it are as without it; a row that admits it shows it."""
    _, q, key, value, table, lens, n, _ = _small(dev, dt=dt, D=D, lens=(40, 0, 31), S=4)
    table = torch.nn.functional.pad(table, (0, width), value=-1)
    mask = torch.tensor([[1, 3, 5, 9]] * 3)  # rows 1, 2, 3 children of 0
    for b, t in enumerate(lens):
        key[:, table[b, (t + 2) // 16], (t + 2) % 16] = bad
        value[:, table[b, (t + 2) // 16], (t + 2) % 16] = bad
    got = C.attn_paged(q.to(dev), key.to(dev), value.to(dev), table.to(dev), n, mask.to(dev)).cpu()
    clean_k, clean_v = key.nan_to_num(0, 0, 0), value.nan_to_num(0, 0, 0)
    check(got, dt, q, clean_k, clean_v, table, lens, mask, D ** -0.5, rows=[0, 1, 3])
    assert not got[:, 2].isfinite().all(-1).any()


def test_non_finite_values_that_are_admitted(C, dev):
    """An infinite value of the prefix reaches every row, with its sign; a NaN makes that dim NaN and no other."""
    _, q, key, value, table, lens, n, mask = _small(dev, lens=(40, 0, 33))
    value[:, table[0, 0], 3, 5] = float("inf")
    value[:, table[0, 2], 1, 9] = float("nan")
    got = C.attn_paged(q.to(dev), key.to(dev), value.to(dev), table.to(dev), n, mask.to(dev)).cpu().float()
    assert (got[0, :, :, 5] == float("inf")).all() and got[0, :, :, 9].isnan().all()
    rest = [d for d in range(128) if d not in (5, 9)]
    assert got[0][..., rest].isfinite().all() and got[1:].isfinite().all()


def test_large_scores(C, dev):
    """One token far above the others takes the row, whatever stands before it."""
    _, q, key, value, table, lens, n, mask = _small(dev, lens=(200, 100, 33), S=1)
    q, key = q * 30, key
    got = C.attn_paged(q.to(dev), key.to(dev), value.to(dev), table.to(dev), n, mask.to(dev))
    check(got, BF, q, key, value, table, lens, mask, 128 ** -0.5)


def test_same_bits_again_and_on_another_stream(C, dev):
    _, q, key, value, table, lens, n, mask = _small(dev, lens=(3000, 10, 500))
    a = [x.to(dev) for x in (q, key, value, table)] + [n, mask.to(dev)]
    one = C.attn_paged(*a)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        two = [C.attn_paged(*a) for _ in range(3)]
    main = [C.attn_paged(*a) for _ in range(3)]  # both streams at once: each call has a workspace of its own
    torch.cuda.synchronize()
    assert all(torch.equal(one, x) for x in two + main)


def test_graph_replay_follows_the_lengths(C, dev):
    """Two captured calls (their workspaces apart) replayed in turn and over lengths and tables written between replays."""
    _, q, key, value, table, lens, n, mask = _small(dev, lens=(400, 64, 33), S=2)
    qd, kd, vd, td, md = (x.to(dev) for x in (q, key, value, table, mask))
    C.attn_paged(qd, kd, vd, td, n, md)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for m in (md, None):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(C.attn_paged(qd, kd, vd, td, n, m))
        graphs.append(gr)
    for now in ((400, 64, 33), (1, 0, 20), (399, 60, 33), (17, 33, 0)):
        n.copy_(torch.tensor(now, dtype=torch.int32))
        for gr in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for o, m in zip(outs, (md, None)):
            want = C.attn_paged(qd, kd, vd, td, n, m)
            assert torch.equal(o, want), now


def test_offsets_past_32_bits(C, dev):
    """A pool of more than 4 GiB a matrix, the sequence in its last pages."""
    T, D, P = 64, 128, 270000
    pool = torch.empty(2, 1, P, T, D, dtype=BF, device=dev)
    g = torch.Generator().manual_seed(4)
    n = 150
    table = torch.tensor([[P - 1, P - 3, P - 2, -1]], dtype=torch.int32)
    small = torch.full((2, 1, 4, T, D), float("nan")).to(BF)
    small_table = torch.tensor([[3, 1, 2, -1]], dtype=torch.int32)
    t = torch.arange(n + 1)
    for i in range(2):
        small[i][:, small_table[0].long()[t // T], t % T] = torch.randn(1, n + 1, D, generator=g).to(BF)
    pool[:, :, P - 4:] = small.to(dev)
    q = torch.randn(1, 1, 4, D, generator=g).to(BF)
    length = torch.tensor([n], dtype=torch.int32, device=dev)
    got = C.attn_paged(q.to(dev), pool[0], pool[1], table.to(dev), length)
    check(got, BF, q, small[0], small[1], small_table, [n], None, D ** -0.5)


def test_refusals(C, dev):
    _, q, key, value, table, lens, n, mask = _small(dev)
    q, key, value, table, mask = (x.to(dev) for x in (q, key, value, table, mask))
    for args, kw, match in [((q.float(), key, value, table, n), {}, "bf16 or fp16"), ((q, key.half(), value, table, n), {}, "one type"),
                            ((q[:, :, :7], key, value, table, n), {}, "multiple"), ((q, key, value[:, 1:], table, n), {}, "head_dim"),
                            ((q, key, value, table.long(), n), {}, "int32"), ((q, key, value, table[:2], n), {}, "table"),
                            ((q, key, value, table, n[:2]), {}, "length"), ((q, key, value, table, n.long()), {}, "int32"),
                            ((q, key, value, table, n, mask.int()), {}, "mask"), ((q, key, value, table, n, mask[:, :3]), {}, "mask"),
                            ((q, key, value, table, n, mask.cpu()), {}, "same ROCm device"), ((q, key, value, table, n), dict(scale=-1.0), "scale"),
                            ((q, key, value, table, n), dict(out=q[:, :, :4]), "out"), ((q[0], key, value, table, n), {}, "q:"),
                            ((q.transpose(2, 3), key, value, table, n), {}, "contiguous")]:
        with pytest.raises(RuntimeError, match=match):
            C.attn_paged(*args, **kw)
    with pytest.raises(RuntimeError, match="apart from q"):
        C.attn_paged(q, key, value, table, n, out=q)
    two = torch.empty(2 * q.numel(), dtype=q.dtype, device=dev)
    with pytest.raises(RuntimeError, match="apart from q"):
        C.attn_paged(two[:q.numel()].view_as(q), key, value, table, n, out=two[q.numel() - 8:-8].view_as(q))
    assert C.attn_paged(two[:q.numel()].view_as(q).copy_(q), key, value, table, n, out=two[q.numel():].view_as(q)).isfinite().all()


def test_queries_of_all_sequences_are_one(C, dev):
    """A broadcast query (strides of 0)."""
    _, q, key, value, table, lens, n, _ = _small(dev, lens=(90, 3, 700))
    q = q[:1, :, :1].expand(3, 4, 8, 128)
    got = C.attn_paged(q[:1, :, :1].to(dev).expand(3, 4, 8, 128), key.to(dev), value.to(dev), table.to(dev), n)
    check(got, BF, q, key, value, table, lens, None, 128 ** -0.5)


@pytest.mark.parametrize("H,Hk,D,S,B,tree", [(4, 2, 64, 1, 400, False), (8, 4, 128, 3, 300, True), (4, 2, 256, 5, 200, True), (32, 4, 64, 6, 160, True)])
def test_infinite_values_in_every_other_unit(C, dev, H, Hk, D, S, B, tree):
    """Shares of several units, of which some hold an infinite value that their rows attend and others none: what a stage leaves out
    for one unit is not taken for the next one's, call after call."""
    print(f"infinite values: H={H} Hk={Hk} D={D} S={S} B={B}", flush=True)
    g = torch.Generator().manual_seed(D + S)
    lens = [int(x) for x in torch.randint(0, 150, (B,), generator=g)]
    key, value, table = cache(g, BF, Hk, 16, D, lens, S, width=200)
    q = (torch.randn(B, S, H, D, generator=g) * 1.5).to(BF)
    mask = tree_masks(g, B, S) if tree else None
    clean = value.clone()
    some = [b for b in range(B) if b % 3 != 1]
    for b in some:
        t = lens[b]  # (own row 0, the root: every row attends it)
        value[:, table[b, t // 16], t % 16, 7] = float("inf")
    a = [x.to(dev) for x in (q, key, value, table)] + [torch.tensor(lens, dtype=torch.int32, device=dev), None if mask is None else mask.to(dev)]
    got = [C.attn_paged(*a) for _ in range(10)]
    assert all(torch.equal(got[0].view(torch.int16), x.view(torch.int16)) for x in got[1:])
    out = got[0].cpu()
    assert (out[some][..., 7] == float("inf")).all()
    want = C.attn_paged(a[0], a[1], clean.to(dev), *a[3:]).cpu()
    out[some, :, :, 7] = want[some][..., 7]
    check(out, BF, q, key, clean, table, lens, mask, D ** -0.5)


def _median_us(f, n=15):
    for _ in range(3):
        f()
    torch.cuda.synchronize()
    took = []
    for _ in range(n):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        f()
        b.record()
        torch.cuda.synchronize()
        took.append(a.elapsed_time(b) * 1e3)
    return sorted(took)[n // 2]


@pytest.mark.parametrize("H,Hk,D,T,S,lens,tree", [(32, 8, 128, 64, 1, [100 + 120 * i for i in range(64)], False), (16, 4, 256, 16, 8, [1001 + 401 * i for i in range(16)], True),
                                                  (32, 8, 128, 64, 2048, [1000], False), (16, 8, 64, 32, 16, [3000, 500, 77], True)])
def test_what_no_row_attends_costs_nothing(C, dev, H, Hk, D, T, S, lens, tree):
    """NaN and infinities in the rows behind the sequences' tokens and in free pages: the bits of the same call over zeros, and its
    time. The bound of the time is twice the other's: a search through the tokens took 8 to 160 times as long."""
    print(f"unused rows: H={H} Hk={Hk} D={D} T={T} S={S} sequences={len(lens)}", flush=True)
    g = torch.Generator().manual_seed(3)
    out, us = [], []
    key, value, table = cache(g, BF, Hk, T, D, lens, S, junk=float("nan"))
    q = torch.randn(len(lens), S, H, D, generator=g).to(BF).to(dev)
    mask = tree_masks(g, len(lens), S).to(dev) if tree else None
    n = torch.tensor(lens, dtype=torch.int32, device=dev)
    for junk in (0.0, float("nan"), float("-inf")):
        k, v = (torch.where(x.isnan(), torch.tensor(junk, dtype=BF), x).to(dev) for x in (key, value))
        a = (q, k, v, table.to(dev), n, mask)
        out.append(C.attn_paged(*a))
        us.append(_median_us(lambda: C.attn_paged(*a)))
    assert all(torch.equal(out[0], x) for x in out[1:])
    assert max(us[1:]) < 2 * us[0], us


@pytest.mark.parametrize("H,Hk,D,S,tree,width", [(8, 2, 128, 6, True, 1), (4, 2, 64, 40, True, 1), (8, 2, 128, 150, False, 1), (4, 1, 256, 200, False, 1), (8, 4, 64, 300, False, 1),
                                                 (16, 8, 64, 30, True, 9000), (16, 8, 64, 30, False, 9000), (32, 8, 128, 16, True, 9000), (8, 2, 128, 8, False, 9000), (16, 4, 256, 16, True, 9000),
                                                 (8, 2, 256, 4, True, 9000), (8, 4, 64, 3, True, 9000)])
def test_values_that_some_rows_attend(C, dev, H, Hk, D, S, tree, width):
    """Infinite values at many of the rows' own tokens, far apart: every row that attends one shows it with its sign, no other does."""
    print(f"values attended by some: H={H} Hk={Hk} D={D} S={S} width={width}", flush=True)
    g = torch.Generator().manual_seed(S)
    lens = [300, 0, 41]
    key, value, table = cache(g, BF, Hk, 32, D, lens, S, width=width)
    q = torch.randn(3, S, H, D, generator=g).to(BF)
    mask = tree_masks(g, 3, S) if tree else None
    clean, hit = value.clone(), torch.zeros(3, S, D, dtype=torch.bool)
    for j in range(1, S, max(2, S // 7)):
        d = 5 * j % D
        for b, m in enumerate(lens):
            value[:, table[b, (m + j) // 32], (m + j) % 32, d] = float("-inf")
            sees = (mask[b] >> j) & 1 == 1 if tree else torch.arange(S) >= j
            hit[b, :, d] |= sees
    a = (q.to(dev), key.to(dev), value.to(dev), table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), None if mask is None else mask.to(dev))
    got = C.attn_paged(*a).cpu()
    hit = hit[:, :, None, :].expand_as(got)
    assert hit.any() and (got[hit] == float("-inf")).all() and got[~hit].isfinite().all()
    want = C.attn_paged(a[0], a[1], clean.to(dev), *a[3:]).cpu()
    check(torch.where(hit, want, got), BF, q, key, clean, table, lens, mask, D ** -0.5)


@pytest.mark.parametrize("dt,top", [(BF, 2.0 ** 18), (BF, 2.0 ** 33), (BF, 2.0 ** 62), (BF, 2.0 ** 90), (FH, 2.0 ** 18), (FH, 2.0 ** 28)])
@pytest.mark.parametrize("H,Hk,D,S,width", [(8, 2, 128, 1, 1), (8, 4, 64, 3, 6000), (4, 1, 256, 5, 1), (8, 2, 128, 40, 1), (4, 2, 256, 70, 6000)])
def test_scores_past_the_accuracy_of_their_exponent(C, dev, dt, top, H, Hk, D, S, width):
    """Scores of up to `top` whose product with scale log2(e) no fp32 number holds to a few units: one token takes the row, or
    several equal ones share it. The scores are exact in fp32 (two dims of 16 powers of two times integers below 256), an integer
    apart at least top / 2^9 before the scale, so every other weight is 0 in fp32 and the result is the token's value, or the mean
    of the sharing tokens' (each weight 1 / count and their sum exact but for fp32, one rounding to the type)."""
    print(f"large scores: {dt} top={top} H={H} Hk={Hk} D={D} S={S} width={width}", flush=True)
    g = torch.Generator().manual_seed(D + S)
    lens, T = [300, 33, 700], 32
    key, value, table = cache(g, dt, Hk, T, D, lens, S, junk=0.0, width=width)
    half = (top / 2 ** 12) ** 0.5  # 16 dims of q times k, integers to 255: 2^12 half^2
    a = 2.0 ** int(torch.tensor(half).log2().floor())
    b = 2.0 ** int(torch.tensor(top / 2 ** 12 / a).log2().floor())
    key[:] = 0
    q = torch.zeros(3, S, H, D, dtype=dt)
    q[..., 3:19] = a
    worth = []
    for i, m in enumerate(lens):
        w = torch.randint(-255, 200 if i < 2 else -20, (Hk, m + S), generator=g)
        w[:, m // 2] = w[:, m - 1] = 230 if i < 2 else -3  # two tokens above all others (the third sequence's scores are all negative)
        t = torch.arange(m + S)
        key[:, table[i, t // T].long(), t % T, 3:19] = (w[..., None] * b).to(dt)
        worth.append(w)
    for scale in (D ** -0.5, 0.31, 0.0137):
        got = C.attn_paged(q.to(dev), key.to(dev), value.to(dev), table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), scale=scale).cpu().double()
        for i, m in enumerate(lens):
            at = torch.tensor([m // 2, m - 1])
            v = value[:, table[i, at // T].long(), at % T].double().mean(1)  # [Hk, D]
            want = v.repeat_interleave(H // Hk, 0).expand(S, H, D)
            assert ((got[i] - want).abs() <= (torch.finfo(dt).eps / 2 + 2.0 ** -20) * want.abs() + 2.0 ** -24).all(), (scale, i, got[i][0, 0, :4], want[0, 0, :4])


def _sampled(C, dev, dt, H, Hk, D, T, lens, S, width, rows, seed=0):
    """A chain of S rows, checked at some rows: row s is a single token behind length + s tokens."""
    print(f"attn_paged {dt} H={H} Hk={Hk} D={D} T={T} lens={lens} S={S} width={width}", flush=True)
    g = torch.Generator().manual_seed(seed + D + S)
    key, value, table = cache(g, dt, Hk, T, D, lens, S, width=width)
    q = (torch.randn(len(lens), S, H, D, generator=g) * 1.5).to(dt)
    got = C.attn_paged(q.to(dev), key.to(dev), value.to(dev), table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev)).cpu()
    assert got.isfinite().all()
    for s in rows:
        check(got[:, s:s + 1], dt, q[:, s:s + 1], key, value, table, [n + s for n in lens], None, D ** -0.5)


@pytest.mark.parametrize("dt", [BF, FH])
@pytest.mark.parametrize("H,Hk,D,S,lens,width", [(32, 32, 64, 2085, [70], 1), (32, 8, 128, 2048, [100], 1), (32, 8, 128, 700, [90, 0, 333], 1), (32, 8, 128, 671, [90, 0, 333], 1),
                                                 (16, 4, 256, 1000, [33, 500], 1), (16, 4, 256, 991, [33, 500], 1), (20, 4, 128, 770, [40, 8, 900, 123], 1), (32, 8, 64, 600, [5] * 8, 50)])
def test_whole_units_of_many_rows(C, dev, dt, H, Hk, D, S, lens, width):
    """Row blocks enough for every work-group (512 at two per CU, 256 at head_dim 256) and just fewer; counts of rows that are no
    multiple of a block's; unequal sequences; the rows at a block's ends and in the last one."""
    spb = 128 // (H // Hk)
    _sampled(C, dev, dt, H, Hk, D, 32, lens, S, width, sorted({0, spb - 1, spb, S // 2, (S - 1) // spb * spb - 1, (S - 1) // spb * spb, S - 1}))


@pytest.mark.parametrize("H,Hk,D,S,lens", [(32, 8, 128, 65, [0, 40]), (8, 4, 64, 200, [0, 77]), (4, 1, 256, 130, [7, 64]), (8, 8, 128, 2, [100, 31])])
def test_chains_fp16(C, dev, H, Hk, D, S, lens):
    _run(C, dev, FH, H, Hk, D, 32, lens, S, False, 5)


@pytest.mark.parametrize("width", [1, 4000])
def test_lengths_out_of_range_are_clamped(C, dev, width):
    """Below 0: no committed token. Past the table: all that it holds; the rows' own have no place there."""
    g, q, key, value, table, _, _, mask = _small(dev, lens=(44, 44, 44, 12))
    table = torch.nn.functional.pad(table[:, :3], (0, width - 1), value=-1)
    W = table.shape[1]
    n = [-5, 2 ** 31 - 1, W * 16 + 1, -2 ** 31]
    got = C.attn_paged(q.to(dev), key.to(dev), value.to(dev), table.to(dev), torch.tensor(n, dtype=torch.int32, device=dev), mask.to(dev))
    # (own rows of sequences 0 and 3 stand at tokens 0..3; sequences 1 and 2 have 44 + 4 tokens in their pages)
    check(got, BF, q, key, value, table, [min(max(x, 0), W * 16) for x in n], mask, 128 ** -0.5)
    assert (got != 0).any(-1).all()


@pytest.mark.parametrize("H,Hk,D,T,lens,S", [(1, 1, 64, 1024, [100], 65535), (2, 2, 128, 16, [7], 20001)])
def test_longest_chains(C, dev, H, Hk, D, T, lens, S):
    _sampled(C, dev, BF, H, Hk, D, T, lens, S, 1, [0, 127, 128, S // 2, S - 2, S - 1])


@pytest.mark.parametrize("D,S,tree", [(64, 1, False), (128, 2, True)])
def test_the_most_sequences(C, dev, D, S, tree):
    g = torch.Generator().manual_seed(17)
    lens = [int(x) for x in torch.randint(0, 40, (1024,), generator=g)]
    lens[::7] = [0] * len(lens[::7])
    _run(C, dev, BF, 2, 1, D, 16, lens, S, tree, 17)
