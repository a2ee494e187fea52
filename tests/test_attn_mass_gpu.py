"""attn_mass on the GPU against the float64 oracle, over pages whose unused rows hold NaN."""
import numpy as np
import pytest
import torch

from oracle import ref
from paged_cases import cache, f64, rows_meet, tree_masks, views

pytestmark = pytest.mark.gpu
BF, FH = torch.bfloat16, torch.float16


def check(got, before, q, key, table, lens, lse, prior, count, path, window, sinks, scale):
    """A weight's relative error: its score's D products and sums (fp32, each within 2^-23 of the sum of magnitudes), the argument
    of its exponential (three roundings of the score's and the lse's size, 2^-23 each) and exp2 (2^-22); the sums of weights:
    one rounding per row tile and join, (rows / 16 + 40) 2^-24 of the sum. `heft` holds sum w (1 + |q k| + |lse|)."""
    D, rows = q.shape[3], q.shape[1] * q.shape[2] // key.shape[0]
    want, heft, written = ref.attention_mass(f64(q), f64(key), table.numpy(), lens, f64(lse), None if prior is None else f64(prior),
                                             None if count is None else count.numpy(), None if path is None else path.numpy(), window, sinks, scale,
                                             got.shape[2])
    lim = ((D + 4) * 2.0 ** -23 + 6 * 2.0 ** -23) * heft + (rows / 16 + 40) * 2.0 ** -24 * want
    got = f64(got)
    bad = ~(np.abs(got - want) <= lim) & written[:, None]
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist(), got[bad][:4].tolist(), want[bad][:4].tolist())
    stay = ~written[:, None] & np.ones_like(got, dtype=bool)
    assert np.array_equal(got[stay], f64(before)[stay], equal_nan=True)


def operands(g, dt, H, Hk, D, T, lens, S, width=1, spread=1.5):
    key, value, table = cache(g, dt, Hk, T, D, lens, S, width=width)
    q = (torch.randn(len(lens), S, H, D, generator=g) * spread).to(dt)
    return q, key, value, table


def _run(C, dev, dt, H, Hk, D, T, lens, S, tree=False, window=None, sinks=0, seed=0, width=1):
    print(f"attn_mass {dt} H={H} Hk={Hk} D={D} T={T} lens={lens} S={S} tree={tree} window={window} sinks={sinks} width={width}", flush=True)
    g = torch.Generator().manual_seed(seed + D + T + S)
    q, key, value, table = operands(g, dt, H, Hk, D, T, lens, S, width)
    B, N = len(lens), table.shape[1] * T
    n = torch.tensor(lens, dtype=torch.int32)
    count = path = None
    if tree:  # (some of the rows, in order; the lse of any rows will do)
        count = torch.tensor([i % (S + 1) for i in range(1, B + 1)], dtype=torch.int32)
        path = torch.stack([torch.randperm(S, generator=g).sort().values if i % 2 else torch.randperm(S, generator=g) for i in range(B)]).to(torch.int32)
    _, lse = C.attn_window(q.to(dev), key.to(dev), value.to(dev), table.to(dev), n.to(dev), window, sinks)
    prior = torch.rand(B, Hk, N, generator=g) * 3
    out = torch.full((B, Hk, N), float("nan"))
    up = lambda t: None if t is None else t.to(dev)  # noqa: E731
    got = C.attn_mass(*map(up, (q, key, table, n, lse)), prior=up(prior), count=up(count), path=up(path), window=window, sinks=sinks, out=up(out))
    check(got, out, q, key, table, lens, lse, prior, count, path, window or 1 << 30, sinks, D ** -0.5)


@pytest.mark.parametrize("dt", [BF, FH])
@pytest.mark.parametrize("H,Hk,D", [(32, 8, 128), (16, 4, 256), (16, 8, 64), (7, 1, 128), (3, 3, 64)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (70, 5), (300, 64)])
def test_single_tokens(C, dev, dt, H, Hk, D, window, sinks):
    _run(C, dev, dt, H, Hk, D, 16, [0, 1, 15, 16, 17, 63, 64, 255, 256, 257, 700], 1, False, window, sinks)


@pytest.mark.parametrize("T", [16, 32, 128, 1024])
def test_page_sizes(C, dev, T):
    _run(C, dev, BF, 8, 2, 128, T, [T - 1, T, T + 1, 3 * T + 5, 0], 5, True, None, 0, T)


@pytest.mark.parametrize("H,Hk,D,S", [(32, 8, 128, 8), (16, 4, 256, 16), (16, 8, 64, 9), (32, 4, 128, 33), (4, 4, 256, 64), (128, 1, 128, 3)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (9, 3), (200, 130)])
def test_paths(C, dev, H, Hk, D, S, window, sinks):
    _run(C, dev, BF if S % 2 else FH, H, Hk, D, 32, [0, 300, 70, 5, 129], S, True, window, sinks, 3)


@pytest.mark.parametrize("H,Hk,D,S,lens", [(32, 8, 128, 100, [0, 40]), (8, 2, 64, 500, [129]), (4, 1, 256, 130, [7, 640]), (6, 2, 128, 333, [33]), (33, 1, 256, 12, [90])])
@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 1), (100, 70)])
def test_prompts(C, dev, H, Hk, D, S, lens, window, sinks):
    _run(C, dev, BF, H, Hk, D, 64, lens, S, False, window, sinks, 4)


def test_wide_tables(C, dev):
    """More runs of tokens than the grid holds at once."""
    _run(C, dev, BF, 2, 2, 64, 16, [5000, 0] + [3] * 60, 2, False, None, 0, 5, width=9000)
    _run(C, dev, BF, 40, 2, 64, 16, [3000] + [9] * 100, 3, False, None, 0, 5, width=9000)


def test_whole_weight(C, dev):
    """A row's weights sum to one: the tokens' sums over everything are the number of rows and heads."""
    g = torch.Generator().manual_seed(6)
    q, key, value, table = (t.to(dev) for t in operands(g, BF, 16, 4, 128, 32, [77, 300, 0], 9))
    n = torch.tensor([77, 300, 0], dtype=torch.int32, device=dev)
    for window, sinks in ((None, 0), (50, 4)):
        _, lse = C.attn_window(q, key, value, table, n, window, sinks)
        got = C.attn_mass(q, key, table, n, lse, window=window, sinks=sinks)
        assert (got.sum(2) - 9 * 4).abs().max().item() < 1e-3


def test_in_place_and_strides(C, dev):
    g = torch.Generator().manual_seed(7)
    lens = [100, 37]
    q, key, value, table = operands(g, BF, 8, 2, 128, 16, lens, 4)
    n = torch.tensor(lens, dtype=torch.int32)
    wide = torch.randn(2, 4, 3, 8, 128, generator=g).to(BF)
    wide[:, :, 1] = q
    a = [wide.to(dev)[:, :, 1], key.to(dev), table.to(dev), n.to(dev)]
    _, lse = C.attn_window(a[0], a[1], value.to(dev), *a[2:], None)
    layers = torch.rand(2, 3, 2, 5, 1000, generator=g)
    state = layers.to(dev)
    view, prior = state[:, 1, :, 2], layers[:, 1, :, 2]
    got = C.attn_mass(*a, lse, prior=view, out=view)
    assert got is view
    check(view, prior, q, key, table, lens, lse, prior, None, None, 1 << 30, 0, 128 ** -0.5)
    rest = torch.ones_like(layers, dtype=torch.bool)
    rest[:, 1, :, 2] = False
    assert torch.equal(state.cpu()[rest], layers[rest])
    # fewer places than tokens: those there are
    short = torch.zeros(2, 2, 50, device=dev)
    C.attn_mass(*a, lse, prior=torch.zeros_like(short), out=short)
    check(short, short, q, key, table, lens, lse, torch.zeros(2, 2, 50), None, None, 1 << 30, 0, 128 ** -0.5)


def test_rows_and_tokens_that_are_none(C, dev):
    """Counts out of range, paths out of range, rows that attended nothing, NaN queries behind the count, pages that are none,
    NaN keys in places that a row does not attend."""
    g = torch.Generator().manual_seed(8)
    lens, S = [90, 90, 90, 90], 5
    q, key, value, table = operands(g, BF, 8, 2, 64, 16, lens, S)
    n = torch.tensor(lens, dtype=torch.int32)
    _, lse = C.attn_window(*(t.to(dev) for t in (q, key, value, table, n)), 30, 2)
    lse = lse.cpu()
    count, path = torch.tensor([3, -2, 99, 4], dtype=torch.int32), torch.arange(S, dtype=torch.int32).repeat(4, 1)
    path[2, 1], path[2, 3] = -1, S
    q[0, 3:] = float("nan")
    lse[3, 2] = -float("inf")
    table[3, 4] = -1
    table[2, 5] = key.shape[1]
    key[:, table[0, 2], 0] = float("nan")  # token 32: every row's window has passed it
    prior = torch.rand(4, 2, table.shape[1] * 16, generator=g)
    out = torch.full_like(prior, 7.0)
    up = lambda t: t.to(dev)  # noqa: E731
    got = C.attn_mass(*map(up, (q, key, table, n, lse)), prior=up(prior), count=up(count), path=up(path), window=30, sinks=2, out=up(out))
    q2, key2 = q.clone(), key.clone()
    q2[0, 3:] = 0
    key2[key2.isnan()] = 0
    check(got, out, q2, key2, table, lens, lse, prior, count, path, 30, 2, 0.125)


def test_replay_follows_the_lengths(C, dev):
    g = torch.Generator().manual_seed(9)
    q, key, value, table = operands(g, BF, 8, 2, 128, 16, [600, 600], 3)
    key.nan_to_num_(0.5), value.nan_to_num_(0.5)
    n = torch.tensor([600, 600], dtype=torch.int32, device=dev)
    a = [q.to(dev), key.to(dev), table.to(dev), n]
    lse = torch.randn(2, 3, 8, generator=g).to(dev) + 10
    state, start = torch.zeros(2, 2, 700, device=dev), torch.rand(2, 2, 700, generator=g)
    C.attn_mass(*a, lse, prior=state, out=state)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        C.attn_mass(*a, lse, prior=state, out=state)
    for now in ([0, 1], [599, 77], [64, 300]):
        n.copy_(torch.tensor(now, dtype=torch.int32))
        state.copy_(start)
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            other = C.attn_mass(*a, lse, prior=start.to(dev), out=start.to(dev))
        torch.cuda.synchronize()
        assert torch.equal(other, state)
        check(state, start, q, key, table, now, lse, start, None, None, 1 << 30, 0, 128 ** -0.5)


def test_refusals(C, dev):
    g = torch.Generator().manual_seed(10)
    q, key, _, table = (t.to(dev) for t in operands(g, BF, 4, 2, 64, 16, [20], 2))
    n, lse = torch.tensor([20], dtype=torch.int32, device=dev), torch.zeros(1, 2, 4, device=dev)
    ok = torch.zeros(1, 2, 64, device=dev)
    for kw in (dict(prior=ok.double()), dict(prior=ok[:, :1]), dict(out=ok[0]), dict(out=ok[:, :, ::2]), dict(prior=ok, out=ok[:, :, :32]), dict(window=0),
               dict(sinks=-1), dict(count=torch.ones(1, device=dev)), dict(path=torch.ones(1, 3, dtype=torch.int32, device=dev)), dict(scale=-1.0),
               dict(out=ok[:, :1].expand(1, 2, 64)), dict(out=ok.cpu())):
        with pytest.raises(RuntimeError):
            C.attn_mass(q, key, table, n, lse, **kw)
    for args in ((q.half(), key, table, n, lse), (q, key, table, n, lse.double()), (q, key, table, n, lse[:, :1]), (q, key, table[:, ::2], n, lse), (q, key, table, n.long(), lse)):
        with pytest.raises(RuntimeError):
            C.attn_mass(*args)
    assert C.attn_mass(q[:0], key, table[:0], n[:0], lse[:0]).shape[0] == 0


@pytest.mark.parametrize("H,Hk,D,S,lens", [(32, 8, 128, 300, [700]), (16, 4, 256, 200, [300, 0, 90]), (16, 8, 64, 1000, [50]), (128, 1, 128, 70, [600]), (9, 3, 128, 411, [1000, 3])])
@pytest.mark.parametrize("dt", [BF, FH])
@pytest.mark.parametrize("width", [1, 700])
def test_many_rows_with_counts(C, dev, H, Hk, D, S, lens, dt, width):
    """Rows through LDS: runs shared by several work-groups (short tables) and by one (wide ones), counts that end inside a stage."""
    g = torch.Generator().manual_seed(S)
    q, key, value, table = operands(g, dt, H, Hk, D, 16, lens, S, width)
    n = torch.tensor(lens, dtype=torch.int32)
    _, lse = C.attn_window(*(t.to(dev) for t in (q, key, value, table, n)), 400, 20)
    N = table.shape[1] * 16
    prior, out = torch.rand(len(lens), Hk, N, generator=g), torch.full((len(lens), Hk, N), 5.0)
    up = lambda t: t.to(dev)  # noqa: E731
    for c in (S, S - 1, S // 2 + 3, 17, 1, 0):
        count = torch.tensor([max(0, c - 5 * i) for i in range(len(lens))], dtype=torch.int32)
        got = C.attn_mass(*map(up, (q, key, table, n, lse)), prior=up(prior), count=up(count), window=400, sinks=20, out=up(out))
        again = C.attn_mass(*map(up, (q, key, table, n, lse)), prior=up(prior), count=up(count), window=400, sinks=20, out=up(out))
        assert torch.equal(got, again)
        if c in (S - 1, 17):
            check(got, out, q, key, table, lens, lse, prior, count, None, 400, 20, D ** -0.5)
        elif c < 2:
            assert torch.equal(got.cpu()[0, :, :lens[0]], prior[0, :, :lens[0]]) or c == 1


def test_heads_side_by_side(C, dev):
    """Sums kept as [kv heads, sequences, places]."""
    g = torch.Generator().manual_seed(11)
    q, key, value, table = (t.to(dev) for t in operands(g, BF, 8, 4, 64, 16, [70, 9], 3))
    n = torch.tensor([70, 9], dtype=torch.int32, device=dev)
    _, lse = C.attn_window(q, key, value, table, n, None)
    want = C.attn_mass(q, key, table, n, lse)
    got = torch.zeros(4, 2, want.shape[2], device=dev).transpose(0, 1)
    assert torch.equal(C.attn_mass(q, key, table, n, lse, out=got), want)


def test_longest_chain(C, dev):
    """65535 rows: every row's weights sum to one."""
    g = torch.Generator().manual_seed(12)
    S = 65535
    q, key, value, table = (t.to(dev) for t in operands(g, BF, 1, 1, 64, 1024, [100], S))
    n = torch.tensor([100], dtype=torch.int32, device=dev)
    _, lse = C.attn_window(q, key, value, table, n, 200, 4)
    got = C.attn_mass(q, key, table, n, lse, window=200, sinks=4)
    assert abs(got.double().sum().item() / S - 1) < 1e-5
    few = C.attn_mass(q[:, -40:].contiguous(), key, table, n + S - 40, lse[:, -40:].contiguous(), window=200, sinks=4)
    part = C.attn_mass(q, key, table, n, lse, count=torch.tensor([S - 40], dtype=torch.int32, device=dev), window=200, sinks=4)
    assert (part + few - got).abs().max().item() < 1e-2 and (few[0, 0, 4:S - 200] == 0).all()


def test_offsets_past_32_bits(C, dev):
    """Keys, and their sums, past 2^32 elements and bytes of their bases."""
    g = torch.Generator().manual_seed(13)
    q, key, value, table = operands(g, BF, 4, 2, 128, 1024, [1500], 70)
    n = torch.tensor([1500], dtype=torch.int32)
    P, small = 16500, key.shape[1]  # a kv head of 4.3 GB
    pool = torch.empty(2, P, 1024, 128, dtype=BF, device=dev)
    pool[:, P - small:] = key.to(dev)
    high = torch.where(table >= 0, table + (P - small), table)
    _, lse = C.attn_window(*(t.to(dev) for t in (q, key, value, table, n)), None)
    wide = torch.empty(2, 1 << 30, dtype=torch.float32, device=dev)[:, -4096:][None]
    wide.fill_(3.0)
    for rows in (70, 1):
        a = (q[:, :rows].contiguous(), lse[:, :rows].contiguous())
        got = C.attn_mass(a[0].to(dev), pool, high.to(dev), n.to(dev), a[1], out=wide)
        check(got, torch.full((1, 2, 4096), 3.0), a[0], key, table, [1500], a[1], None, None, None, 1 << 30, 0, 128 ** -0.5)
        wide.fill_(3.0)


def test_no_rows(C, dev):
    """A step without rows: the committed tokens' sums pass through, places behind stay."""
    g = torch.Generator().manual_seed(14)
    q, key, _, table = (t.to(dev) for t in operands(g, BF, 4, 2, 64, 16, [40, 0], 1))
    n, lse = torch.tensor([40, 0], dtype=torch.int32, device=dev), torch.zeros(2, 0, 4, device=dev)
    prior = torch.rand(2, 2, 60, generator=g).to(dev)
    none = torch.zeros(2, 0, dtype=torch.int32, device=dev)
    for kw in ({}, dict(count=n, path=none)):
        out = torch.full_like(prior, 7.0)
        C.attn_mass(q[:, :0], key, table, n, lse, prior=prior, out=out, **kw)
        assert torch.equal(out[0, :, :40], prior[0, :, :40]) and (out[0, :, 40:] == 7).all() and (out[1] == 7).all()
        assert (C.attn_mass(q[:, :0], key, table, n, lse, **kw) == 0).all()


def test_in_place_needs_the_same_strides(C, dev):
    g = torch.Generator().manual_seed(15)
    q, key, _, table = (t.to(dev) for t in operands(g, BF, 4, 2, 64, 16, [20, 9], 2))
    n, lse = torch.tensor([20, 9], dtype=torch.int32, device=dev), torch.zeros(2, 2, 4, device=dev)
    state = torch.zeros(2, 2, 64, device=dev)
    with pytest.raises(RuntimeError, match="in place"):
        C.attn_mass(q, key, table, n, lse, prior=state, out=state.transpose(0, 1))


def test_sums_in_the_gaps_of_others(C, dev):
    """prior and out as views of one buffer whose ranges meet and whose rows do not: as with buffers of their own."""
    g = torch.Generator().manual_seed(16)
    start = torch.rand(9000, generator=g).to(dev)
    tried = 0
    for B, Hk in ((3, 2), (1, 2), (3, 1)):
        q, key, value, table = (t.to(dev) for t in operands(g, BF, 4, Hk, 64, 16, [20, 9, 0][:B], 2))
        n = torch.tensor([20, 9, 0][:B], dtype=torch.int32, device=dev)
        _, lse = C.attn_window(q, key, value, table, n, None)
        for ob, oh, pb, ph, d in views():
            if rows_meet(B, Hk, 100, d, pb, ph, ob, oh):
                continue
            buf = start.clone()
            prior, out = buf.as_strided((B, Hk, 100), (pb, ph, 1), 4000 + d), buf.as_strided((B, Hk, 100), (ob, oh, 1), 4000)
            want = C.attn_mass(q, key, table, n, lse, prior=prior.clone(), out=out.clone())
            assert torch.equal(C.attn_mass(q, key, table, n, lse, prior=prior, out=out), want), (B, Hk, ob, oh, pb, ph, d)
            tried += 1
    assert tried > 300


def test_paths_of_many_rows_need_no_workspace(C, dev):
    """Only rows without a path are shared out to several work-groups, which leave their sums in the workspace."""
    from mdx import _lib
    g = torch.Generator().manual_seed(17)
    lens, S, H, Hk, D, T = [300, 40], 200, 8, 2, 64, 16  # (seven stages of rows: without a path two work-groups a run)
    q, key, value, table = (t.to(dev) for t in operands(g, BF, H, Hk, D, T, lens, S))
    n = torch.tensor(lens, dtype=torch.int32, device=dev)
    path = torch.arange(S, dtype=torch.int32, device=dev).repeat(2, 1)
    count = torch.tensor([17, 133], dtype=torch.int32, device=dev)
    _, lse = C.attn_window(q, key, value, table, n, None)
    want = C.attn_mass(q, key, table, n, lse, count=count, path=path)
    out, (P, W, N) = torch.zeros_like(want), (key.shape[1], table.shape[1], want.shape[2])
    L = _lib.lib()
    assert L.mdx_attn_mass_workspace(2, S, H, Hk, D, T, W, N) > 0
    p = lambda t: t.data_ptr()  # noqa: E731
    rc = L.mdx_attn_mass(p(q), *q.stride()[:3], p(key), *key.stride()[:3], _lib.DT_BF16, p(table), W, p(n), p(lse), None, 0, 0, p(count), p(path), 1 << 30, 0, p(out),
                         *out.stride()[:2], N, 2, S, H, Hk, D, P, T, W, D ** -0.5, None, 0, torch.cuda.current_stream().cuda_stream)
    assert rc == _lib.MDX_OK, L.mdx_last_error()
    assert torch.equal(out, want)


@pytest.mark.parametrize("H,Hk,D,S,lens", [(32, 8, 128, 300, [700]), (16, 4, 256, 200, [300, 0, 90]), (16, 8, 64, 1000, [50]), (128, 1, 128, 70, [600]), (9, 3, 128, 411, [1000, 3])])
@pytest.mark.parametrize("width", [1, 700])
def test_every_count_against_the_oracle(C, dev, H, Hk, D, S, lens, width):
    """All rows, half of them, one, none; each sequence with fewer than the one ahead."""
    g = torch.Generator().manual_seed(S + 1)
    q, key, value, table = operands(g, BF, H, Hk, D, 16, lens, S, width)
    n = torch.tensor(lens, dtype=torch.int32)
    _, lse = C.attn_window(*(t.to(dev) for t in (q, key, value, table, n)), 400, 20)
    N = table.shape[1] * 16
    prior, out = torch.rand(len(lens), Hk, N, generator=g), torch.full((len(lens), Hk, N), 5.0)
    up = lambda t: t.to(dev)  # noqa: E731
    for c in (S, S // 2 + 3, 1, 0):
        count = torch.tensor([max(0, c - 5 * i) for i in range(len(lens))], dtype=torch.int32)
        got = C.attn_mass(*map(up, (q, key, table, n, lse)), prior=up(prior), count=up(count), window=400, sinks=20, out=up(out))
        check(got, out, q, key, table, lens, lse, prior, count, None, 400, 20, D ** -0.5)


@pytest.mark.parametrize("D,path,dt", [(128, False, BF), (256, False, FH), (64, False, BF), (128, True, FH), (256, True, BF)])
def test_many_rows_over_wide_tables(C, dev, D, path, dt):
    """More runs of tokens than the grid holds at once, at 68 query rows per kv head: 4096 pairs leave 16 runs each, and two of the
    sequences have more."""
    B, S, H, Hk, T = 1024, 17, 16, 4, 16
    g = torch.Generator().manual_seed(18)
    lens = [i % 7 for i in range(B)]
    lens[5], lens[700] = 4600, 4300  # (runs of 256 tokens, 128 at head_dim 256, 64 and 32 with a path)
    q, key, value, table = operands(g, dt, H, Hk, D, T, lens, S)
    n = torch.tensor(lens, dtype=torch.int32)
    _, lse = C.attn_window(*(t.to(dev) for t in (q, key, value, table, n)), None)
    count = torch.zeros(B, dtype=torch.int32)
    for b in (0, 5, 6, 300, 700, 701, 1023):
        count[b] = S - b % 2
    rows = torch.stack([torch.randperm(S, generator=g) for _ in range(B)]).to(torch.int32) if path else None
    prior = torch.rand(B, Hk, table.shape[1] * T, generator=g)
    out = torch.full_like(prior, 7.0)
    up = lambda t: None if t is None else t.to(dev)  # noqa: E731
    got = C.attn_mass(*map(up, (q, key, table, n, lse)), prior=up(prior), count=up(count), path=up(rows), out=up(out))
    check(got, out, q, key, table, lens, lse, prior, count, rows, 1 << 30, 0, D ** -0.5)
