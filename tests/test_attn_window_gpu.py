"""attn_window on the GPU against the float64 oracle (outputs: the bounds of tests/paged_cases.py; lse: below), over pages whose
unused rows hold NaN."""
import numpy as np
import pytest
import torch

from oracle import ref
from paged_cases import bound, cache, f64, tree_masks

pytestmark = pytest.mark.gpu
BF, FH = torch.bfloat16, torch.float16


def lse_bound(want, heft, tokens, D):
    """How far a log-sum-exp may lie from float64: a score's error as in `bound` ((D + 4) products and sums and the argument of its
    exponential, each within 2^-23 of its size), the weights' sum (fp32, relative: (tokens / 16 + 32 + 600) 2^-24, and 2^-22 of
    exp2) as an absolute error of its logarithm, and three roundings of the logarithm's size."""
    size = np.where(np.isfinite(want), np.abs(want), 0) + 2 * heft
    return ((D + 4) * 2.0 ** -23 + 3 * 2.0 ** -23) * heft + (tokens / 16 + 632) * 2.0 ** -24 + 2.0 ** -22 + 3 * 2.0 ** -24 * size


def check(got, dt, q, key, value, table, lens, mask, scale, window, sinks, rows=slice(None)):
    out, lse = got
    keep = ref.window_keep(None if mask is None else mask.numpy(), lens, q.shape[1], window, sinks)
    a = (f64(key), table.numpy(), lens, None if mask is None else mask.numpy(), scale)
    want, spread, mass, heft = ref.paged_attention(f64(q), a[0], f64(value), *a[1:], keep)
    tokens = max(lens) + q.shape[1]
    err, lim = np.abs(f64(out) - want), bound(dt, want, spread, mass, heft, tokens, q.shape[3])
    bad = ~(err <= lim)[:, rows]
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist(), float(np.nanmax(err / np.maximum(lim, 1e-30))))
    want = ref.paged_lse(f64(q), *a, keep)
    got = f64(lse)
    with np.errstate(invalid="ignore"):
        err = np.where(got == want, 0.0, np.abs(got - want))
    bad = ~(err <= lse_bound(want, heft, tokens, q.shape[3]))[:, rows]
    assert not bad.any(), ("lse", int(bad.sum()), np.argwhere(bad)[:4].tolist(), float(np.nanmax(err)))


def _run(C, dev, dt, H, Hk, D, T, lens, S, tree, window, sinks, seed=0, width=1):
    print(f"attn_window {dt} H={H} Hk={Hk} D={D} T={T} lens={lens} S={S} tree={tree} window={window} sinks={sinks} width={width}", flush=True)
    g = torch.Generator().manual_seed(seed + D + T + S + window)
    key, value, table = cache(g, dt, Hk, T, D, lens, S, width=width)
    q = (torch.randn(len(lens), S, H, D, generator=g) * 1.5).to(dt)
    mask = tree_masks(g, len(lens), S) if tree else None
    n = torch.tensor(lens, dtype=torch.int32, device=dev)
    got = C.attn_window(q.to(dev), key.to(dev), value.to(dev), table.to(dev), n, window, sinks, None if mask is None else mask.to(dev))
    check(got, dt, q, key, value, table, lens, mask, D ** -0.5, window, sinks)


@pytest.mark.parametrize("dt", [BF, FH])
@pytest.mark.parametrize("H,Hk,D", [(32, 8, 128), (16, 4, 256), (16, 8, 64), (7, 1, 128)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (17, 4), (64, 64), (100, 3), (5000, 4)])
def test_single_tokens(C, dev, dt, H, Hk, D, window, sinks):
    _run(C, dev, dt, H, Hk, D, 16, [0, 1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300, 1000], 1, False, window, sinks)


@pytest.mark.parametrize("T", [16, 32, 128, 1024])
@pytest.mark.parametrize("window,sinks", [(33, 5), (200, 130)])
def test_page_sizes(C, dev, T, window, sinks):
    _run(C, dev, BF, 8, 2, 128, T, [T - 1, T, T + 1, 3 * T + 5, 0, 777], 3, True, window, sinks)


@pytest.mark.parametrize("H,Hk,D,S", [(32, 8, 128, 16), (16, 4, 256, 8), (16, 8, 64, 9), (32, 8, 128, 17), (32, 4, 128, 64), (8, 8, 64, 64), (4, 4, 256, 63)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (2, 2), (7, 75), (70, 0), (150, 4)])
def test_trees(C, dev, H, Hk, D, S, window, sinks):
    """Windows that end among a row's own ancestors, and first tokens that reach into them."""
    _run(C, dev, BF if S % 2 else FH, H, Hk, D, 64, [0, 3, 70, 257, 512], S, True, window, sinks, H)


@pytest.mark.parametrize("H,Hk,D,S,lens", [(32, 8, 128, 65, [0, 40]), (8, 2, 128, 300, [129]), (4, 1, 256, 130, [7, 640]), (8, 4, 64, 513, [0]),
                                           (6, 2, 128, 100, [33, 0, 700]), (33, 1, 256, 12, [90]), (16, 1, 128, 9, [500])])
@pytest.mark.parametrize("window,sinks", [(1, 0), (20, 4), (64, 150), (333, 1), (1 << 30, 0)])
def test_chains(C, dev, H, Hk, D, S, lens, window, sinks):
    _run(C, dev, BF if D != 256 else FH, H, Hk, D, 32, lens, S, False, window, sinks, 5)


@pytest.mark.parametrize("H,Hk,D,S,tree", [(32, 8, 128, 1, False), (16, 4, 256, 8, True), (16, 8, 64, 12, True), (8, 4, 64, 32, False), (8, 2, 128, 80, False)])
@pytest.mark.parametrize("window", [700, 2100])
def test_much_to_stream(C, dev, H, Hk, D, S, tree, window):
    """The forms for wide windows and tables: shares that begin and end inside units, and their join."""
    _run(C, dev, BF, H, Hk, D, 64, [0, 70, 3000, 129], S, tree, window, 4, H, 6000)


@pytest.mark.parametrize("H,Hk,D,S", [(4, 4, 128, 2), (8, 2, 64, 5), (2, 2, 256, 3)])
def test_many_units(C, dev, H, Hk, D, S):
    """More units than work-groups."""
    _run(C, dev, BF, H, Hk, D, 16, [(37 * i) % 200 for i in range(150)], S, True, 50, 2, 3)


def test_everything_is_attn_paged(C, dev):
    """A window over everything gives attn_paged's outputs, to its rounding."""
    g = torch.Generator().manual_seed(3)
    lens, S = [5, 400, 0], 6
    key, value, table = cache(g, BF, 4, 32, 128, lens, S)
    q, mask = torch.randn(3, S, 16, 128, generator=g).to(BF), tree_masks(g, 3, S)
    a = [t.to(dev) for t in (q, key, value, table)] + [torch.tensor(lens, dtype=torch.int32, device=dev)]
    want = C.attn_paged(*a, mask.to(dev))
    for window, sinks in ((None, 0), (1 << 30, 1 << 30), (1, 500)):
        got, _ = C.attn_window(*a, window, sinks, mask.to(dev))
        assert (got.float() - want.float()).abs().max().item() <= 2.0 ** -7 * want.abs().max().item()


def test_rows_that_admit_nothing(C, dev):
    """Masks of nothing behind no committed tokens, sequences without pages: 0 and -inf."""
    g = torch.Generator().manual_seed(4)
    key, value, table = cache(g, BF, 2, 16, 64, [0, 40, 30], 3)
    table[2] = -1
    mask = torch.tensor([[0, 1, 3], [0, 0, 7], [1, 3, 7]])
    q = torch.randn(3, 3, 4, 64, generator=g).to(BF)
    n = torch.tensor([0, 40, 30], dtype=torch.int32, device=dev)
    got = C.attn_window(q.to(dev), key.to(dev), value.to(dev), table.to(dev), n, 5, 1, mask.to(dev))
    check(got, BF, q, key, value, table, [0, 40, 30], mask, 0.125, 5, 1)
    assert (got[0][0, 0] == 0).all() and (got[1][0, 0] == -float("inf")).all() and (got[0][2] == 0).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("D,S,tree,width", [(128, 4, True, 1), (64, 1, False, 3000), (256, 3, True, 1), (128, 200, False, 1)])
def test_non_finite_outside_of_the_windows(C, dev, bad, D, S, tree, width):
    """Committed tokens that every window has passed, and those that only the first rows' windows hold."""
    g = torch.Generator().manual_seed(int(D + S))
    lens, window, sinks = [300, 90], 40, 2
    key, value, table = cache(g, BF, 2, 16, D, lens, S, width=width)
    q = torch.randn(2, S, 8, D, generator=g).to(BF)
    mask = tree_masks(g, 2, S) if tree else None
    for b, n in enumerate(lens):
        for t in (2, 30, max(3, n - window - S)):  # passed by every row
            key[:, table[b, t // 16], t % 16] = bad
            value[:, table[b, t // 16], t % 16] = bad
    n = torch.tensor(lens, dtype=torch.int32, device=dev)
    args = (q.to(dev), key.to(dev), value.to(dev), table.to(dev), n, window, sinks, None if mask is None else mask.to(dev))
    check(C.attn_window(*args), BF, q, key, value, table, lens, mask, D ** -0.5, window, sinks)
    # a value that some rows attend and the others do not: a chain's row s attends tokens past n + s - window
    t = lens[0] - window + S // 2
    value[:, table[0, t // 16], t % 16] = bad
    out, lse = C.attn_window(args[0], args[1], value.to(dev), *args[3:])
    keep = ref.window_keep(None if mask is None else mask.numpy(), lens, S, window, sinks)
    for s in range(S):
        seen = bool(keep(0, s, 0, np.array([t]))[0])
        assert torch.isfinite(out[0, s].float()).all().item() == (not seen), s
    assert torch.isfinite(out[1].float()).all() and torch.isfinite(lse).all()


def test_strides_and_outputs(C, dev):
    g = torch.Generator().manual_seed(9)
    lens, S = [100, 260], 4
    kv = torch.zeros(3, 2, 2, 24, 32, 128, dtype=BF)
    k0, v0, table = cache(g, BF, 2, 32, 128, lens, S)
    kv[1, 0, :, :k0.shape[1]], kv[1, 1, :, :k0.shape[1]] = k0, v0
    wide = torch.randn(2, S, 3, 8, 128, generator=g).to(BF)
    q = wide[:, :, 1]
    out, lse = torch.full((2, S, 8, 128), 7.0, dtype=BF, device=dev), torch.full((2, S, 8), 7.0, device=dev)
    d = kv.to(dev)
    n = torch.tensor(lens, dtype=torch.int32, device=dev)
    got = C.attn_window(wide.to(dev)[:, :, 1], d[1, 0], d[1, 1], table.to(dev), n, 50, 4, scale=0.2, out=out, lse=lse)
    assert got[0] is out and got[1] is lse
    check(got, BF, q, kv[1, 0], kv[1, 1], table, lens, None, 0.2, 50, 4)


def test_large_scores(C, dev):
    """Scores of thousands, and differences that pass exp's range."""
    g = torch.Generator().manual_seed(10)
    for dt, size in ((BF, 40.0), (FH, 12.0)):
        key, value, table = cache(g, dt, 2, 16, 64, [200], 2)
        q = (torch.randn(1, 2, 4, 64, generator=g) * size).to(dt)
        n = torch.tensor([200], dtype=torch.int32, device=dev)
        got = C.attn_window(q.to(dev), key.to(dev), value.to(dev), table.to(dev), n, 90, 10)
        check(got, dt, q, key, value, table, [200], None, 0.125, 90, 10)


def test_replay_follows_the_lengths(C, dev):
    """A captured call beside an eager one on another stream, over changing lengths."""
    g = torch.Generator().manual_seed(11)
    lens, S = [900, 900, 900], 2
    key, value, table = cache(g, BF, 2, 16, 128, lens, S, junk=0.5)
    q = torch.randn(3, S, 16, 128, generator=g).to(BF)
    n = torch.tensor(lens, dtype=torch.int32, device=dev)
    args = (q.to(dev), key.to(dev), value.to(dev), table.to(dev), n, 300, 4)
    C.attn_window(*args)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        out = C.attn_window(*args)
    for now in ([0, 1, 2], [898, 5, 303], [300, 299, 64]):
        n.copy_(torch.tensor(now, dtype=torch.int32))
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            eager = C.attn_window(*args)
        torch.cuda.synchronize()
        assert torch.equal(out[0], eager[0]) and torch.equal(out[1], eager[1])
        check(out, BF, q, key, value, table, now, None, 128 ** -0.5, 300, 4)


def test_refusals(C, dev):
    g = torch.Generator().manual_seed(12)
    key, value, table = (t.to(dev) for t in cache(g, BF, 2, 16, 64, [20], 2))
    q, n = torch.randn(1, 2, 4, 64, generator=g).to(BF).to(dev), torch.tensor([20], dtype=torch.int32, device=dev)
    for args, kw in (((q, key, value, table, n, 0), {}), ((q, key, value, table, n, -3), {}), ((q, key, value, table, n, 4, -1), {}),
                     ((q, key, value, table, n, (1 << 30) + 1), {}), ((q, key, value, table, n, 4, 1 << 31), {}), ((q, key, value.half(), table, n, 4), {}),
                     ((q, key, value, table, n, 4), dict(lse=torch.empty(1, 2, 4, dtype=torch.float64, device=dev))),
                     ((q, key, value, table, n, 4), dict(lse=torch.empty(1, 4, 2, device=dev))), ((q, key, value, table, n, 4), dict(lse=torch.empty(1, 2, 4))),
                     ((q, key, value, table, n, 4), dict(out=q)), ((q, key, value, table, n, 4), dict(scale=0.0)), ((q, key, value, table, n.long(), 4), {})):
        with pytest.raises(RuntimeError):
            C.attn_window(*args, **kw)
    with pytest.raises(TypeError):
        C.attn_window(q, key, value, table, n, 2.5)
    out, lse = C.attn_window(q[:0], key, value, table[:0], n[:0], 4)
    assert out.shape == (0, 2, 4, 64) and lse.shape == (0, 2, 4)


@pytest.mark.parametrize("width", [1, 3000])
def test_lengths_out_of_range_are_clamped(C, dev, width):
    g = torch.Generator().manual_seed(13)
    key, value, table = cache(g, BF, 2, 16, 64, [60, 40], 4, width=width)
    q = torch.randn(2, 4, 8, 64, generator=g).to(BF)
    a = [t.to(dev) for t in (q, key, value, table)]
    n = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    top = table.shape[1] * 16
    for got, want in ((n(-5, 40), n(0, 40)), (n(60, 2 ** 31 - 1), n(60, top)), (n(-2 ** 31, top + 1), n(0, top))):
        x, y = C.attn_window(*a, got, 20, 3), C.attn_window(*a, want, 20, 3)
        assert torch.equal(x[0], y[0]) and torch.equal(x[1], y[1])


def test_the_most_sequences(C, dev):
    g = torch.Generator().manual_seed(14)
    lens = [i % 50 for i in range(1024)]
    key, value, table = cache(g, BF, 1, 16, 64, lens, 2)
    q = torch.randn(1024, 2, 2, 64, generator=g).to(BF)
    got = C.attn_window(*(t.to(dev) for t in (q, key, value, table)), torch.tensor(lens, dtype=torch.int32, device=dev), 20, 3)
    check(got, BF, q, key, value, table, lens, None, 0.125, 20, 3)


def test_longest_chain(C, dev):
    """65535 rows: the first and the last are as those of short calls over the same tokens."""
    g = torch.Generator().manual_seed(15)
    S, T = 65535, 1024
    key, value, table = (t.to(dev) for t in cache(g, BF, 1, T, 64, [100], S))
    q = torch.randn(1, S, 1, 64, generator=g).to(BF).to(dev)
    n = torch.tensor([100], dtype=torch.int32, device=dev)
    out, lse = C.attn_window(q, key, value, table, n, 300, 5)
    for s in (0, 1, 40000, S - 3):
        a, b = C.attn_window(q[:, s:s + 3].contiguous(), key, value, table, n + s, 300, 5)
        assert (a.float() - out[:, s:s + 3].float()).abs().max().item() <= 2.0 ** -6 and (b - lse[:, s:s + 3]).abs().max().item() <= 1e-5
