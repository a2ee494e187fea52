"""verify_drafts against its oracle in float64: every output is a whole number and has to be equal. (A draw or an acceptance could
only differ where a uniform lies within some 1e-14 of a border, relative to the whole: with the fixed inputs here none does.)"""
import numpy as np
import pytest
import torch

from oracle import ref

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def f64(t):
    return t.detach().cpu().double().numpy()


def inputs(seed, B, R, V, dt, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    base = torch.randn(B, R, V, generator=g) * spread
    logits = (base + 0.5 * torch.randn(B, R, V, generator=g)).to(DT[dt])
    draft = (base[:, :R - 1] + 0.5 * torch.randn(B, R - 1, V, generator=g)).to(DT[dt])
    tokens = torch.zeros(B, R, dtype=torch.int64)
    if R > 1:
        noise = torch.empty(B, R - 1, V).exponential_(generator=g)
        tokens[:, 1:] = (draft.float() - noise.log()).argmax(-1)
    return logits, draft, tokens, torch.rand(B, R + 1, generator=g, dtype=torch.float64)


def check(C, logits, tokens, uniform, draft=None, parent=None, heat=1.0, dev="cuda"):
    up = lambda t: t.to(dev) if torch.is_tensor(t) else t  # noqa: E731
    got = C.verify_drafts(up(logits), up(tokens), up(uniform), draft=up(draft), parent=up(parent), temperature=up(heat))
    want = ref.verify_drafts(f64(logits), tokens.numpy(), uniform.numpy(), None if draft is None else f64(draft),
                             None if parent is None else parent.numpy(), heat.numpy() if torch.is_tensor(heat) else heat)
    for g, w, what in zip(got, want, ("count", "path", "next")):
        assert g.cpu().numpy().tolist() == w.tolist(), what
    return want


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("B,R,V", [(1, 2, 1), (3, 4, 7), (2, 5, 4097), (5, 3, 8185), (2, 2, 8193), (1, 8, 32768), (2, 3, 151936), (33, 2, 501)])
def test_chains_with_draft_probabilities(C, dt, B, R, V):
    logits, draft, tokens, uniform = inputs(V + R, B, R, V, dt)
    check(C, logits, tokens, uniform, draft, heat=torch.linspace(0.6, 1.4, B))


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("B,R,V", [(1, 1, 9), (4, 8, 1000), (2, 16, 8191), (1, 64, 257), (3, 5, 40000)])
def test_trees(C, dt, B, R, V):
    """Random trees whose children carry likely tokens, some of them twice, some none, some rows behind no row ahead of them."""
    logits, _, tokens, uniform = inputs(V * 3 + R, B, R, V, dt, spread=2.0)
    g = torch.Generator().manual_seed(R)
    parent = (torch.rand(B, R, generator=g) * torch.arange(R)).to(torch.int32)
    best = logits.float().topk(min(4, V), -1).indices
    for b in range(B):
        for r in range(1, R):
            tokens[b, r] = best[b, parent[b, r], int(torch.randint(0, best.shape[-1], (1,), generator=g))]
    if R > 4:
        tokens[0, 3], tokens[0, 4] = -1, V
        parent[-1, 2], parent[-1, 4] = 2, -7
    check(C, logits, tokens, uniform, parent=parent, heat=0.5)
    low = uniform.clone()
    low[:, :R] *= 0.05  # (the first children: long paths)
    check(C, logits, tokens, low, parent=parent, heat=torch.full((B,), 0.5))
    check(C, logits, tokens, uniform, heat=0.5)  # a chain of drafts that are no samples


def test_long_accepted_chains(C):
    """Draft and target alike: every token is accepted, the answer comes from the last row."""
    logits, _, tokens, uniform = inputs(5, 4, 9, 3000, "bf16")
    same = logits[:, :8].contiguous()
    g = torch.Generator().manual_seed(1)
    tokens[:, 1:] = torch.randint(0, 3000, (4, 8), generator=g)
    assert (check(C, logits, tokens, uniform, same)[0] == 9).all()


def test_greedy(C):
    logits, draft, tokens, uniform = inputs(9, 4, 5, 20000, "bf16")
    logits[:, :, 777] = logits[:, :, 15000] = 60.0  # a tie: the lowest index
    tokens[0, 1:] = 777
    tokens[1, 1:3] = 777
    heat = torch.tensor([0.0, 0.0, -1.0, 0.7])
    want = check(C, logits, tokens, uniform, draft, heat=heat)
    assert want[0][0] == 5 and want[2][0] == 777 and want[2][2] == 777
    assert check(C, logits, tokens, uniform, heat=0.0)[0].tolist()[:2] == [5, 3]


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
def test_masked_and_odd_logits(C, dt):
    """-inf over most of the vocabulary, rows of nothing, NaN, +inf, the type's lowest value, all logits alike."""
    logits, draft, tokens, uniform = inputs(11, 8, 3, 9000, dt)
    logits[0, :, :8990] = float("-inf")
    logits[1] = float("-inf")
    logits[2, :, ::2] = float("nan")
    logits[3, :, 55] = logits[3, :, 8600] = float("inf")
    logits[4] = torch.finfo(DT[dt]).min
    logits[4, :, 4000] = torch.finfo(DT[dt]).max
    logits[5] = 0.0
    logits[6, 0, :8192] = float("-inf")
    draft[7] = float("-inf")
    tokens[0, 1] = 8995
    for heat in (1.0, torch.linspace(0.5, 2.0, 8), 0.0):
        want = check(C, logits, tokens, uniform, draft, heat=heat)
        assert want[2][1] == -1
        check(C, logits, tokens, uniform, heat=heat)


def test_refused_without_a_rest(C):
    """A token without probability in p and q, and p == q: p answers; uniforms at the ends of their range."""
    logits, _, tokens, uniform = inputs(13, 6, 2, 20000, "fp16")
    logits[:, :, 123] = float("-inf")
    tokens[:, 1] = 123
    uniform[0], uniform[1] = 0.0, 1.0 - 2.0 ** -53
    assert (check(C, logits, tokens, uniform, logits[:, :1].contiguous())[0] == 1).all()


def test_extreme_temperatures(C):
    logits, draft, tokens, uniform = inputs(14, 5, 3, 5000, "fp32")
    heat = torch.tensor([1e-30, 1e-3, 50.0, 1e30, 2.0 ** -140])
    check(C, logits, tokens, uniform, draft, heat=heat)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_strided_rows(C, dev, dt):
    """Rows of a wider buffer that stand at every offset to the 16-byte boundaries, the draft's otherwise than the target's."""
    logits, draft, tokens, uniform = inputs(15, 3, 4, 8190, dt)
    for off, pad in ((1, 3), (3, 0), (5, 8), (7, 1)):
        wide = torch.full((3, 4, 8190 + off + pad), 99.0, dtype=DT[dt], device=dev)
        view = wide[:, :, off:off + 8190]
        view.copy_(logits)
        dwide = torch.full((3, 3, 8191 + pad), 99.0, dtype=DT[dt], device=dev)
        dview = dwide[:, :, 1:8191]
        dview.copy_(draft)
        got = C.verify_drafts(view, tokens.to(dev), uniform.to(dev), draft=dview, temperature=0.9)
        want = ref.verify_drafts(f64(logits), tokens.numpy(), uniform.numpy(), f64(draft), heat=0.9)
        assert [g.cpu().tolist() for g in got] == [w.tolist() for w in want]
    # one row of logits for every sequence and row
    one = logits[:1, :1].to(dev).expand(3, 4, 8190)
    got = C.verify_drafts(one, tokens.to(dev), uniform.to(dev))
    want = ref.verify_drafts(f64(one), tokens.numpy(), uniform.numpy())
    assert [g.cpu().tolist() for g in got] == [w.tolist() for w in want]


def test_captured_and_replayed_beside_another_stream(C, dev):
    """Two calls of one shape at once, one of them a captured graph that is replayed over changing inputs."""
    a = [inputs(20 + i, 6, 5, 30000, "bf16") for i in range(4)]
    hold = [t.to(dev) for t in a[0]]
    other = [t.to(dev) for t in a[3]]
    C.verify_drafts(hold[0], hold[2], hold[3], draft=hold[1])
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        out = C.verify_drafts(hold[0], hold[2], hold[3], draft=hold[1])
    want_other = ref.verify_drafts(f64(a[3][0]), a[3][2].numpy(), a[3][3].numpy(), f64(a[3][1]))
    for i in (1, 2, 0, 1):
        for h, t in zip(hold, a[i]):
            h.copy_(t)
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            beside = C.verify_drafts(other[0], other[2], other[3], draft=other[1])
        torch.cuda.synchronize()
        want = ref.verify_drafts(f64(a[i][0]), a[i][2].numpy(), a[i][3].numpy(), f64(a[i][1]))
        assert [g.cpu().tolist() for g in out] == [w.tolist() for w in want]
        assert [g.cpu().tolist() for g in beside] == [w.tolist() for w in want_other]


def test_refusals(C, dev):
    logits, draft, tokens, uniform = (t.to(dev) for t in inputs(30, 2, 3, 64, "bf16"))
    parent = torch.zeros(2, 3, dtype=torch.int32, device=dev)
    for args, kw in (((logits.half(), tokens, uniform), dict(draft=draft)), ((logits.transpose(1, 2), tokens, uniform), {}),
                     ((logits, tokens.int(), uniform), {}), ((logits, tokens, uniform.float()), {}), ((logits, tokens, uniform[:, :3]), {}),
                     ((logits, tokens, uniform), dict(draft=draft, parent=parent)), ((logits, tokens, uniform), dict(parent=parent.long())),
                     ((logits, tokens, uniform), dict(draft=draft[:, :1])), ((logits, tokens, uniform), dict(temperature=-1.0)),
                     ((logits, tokens, uniform), dict(temperature=torch.ones(3, device=dev))), ((logits, tokens.cpu(), uniform), {}),
                     ((logits.double(), tokens, uniform), {})):
        with pytest.raises(RuntimeError):
            C.verify_drafts(*args, **kw)
    with pytest.raises((RuntimeError, TypeError)):
        C.verify_drafts(logits, tokens, uniform, temperature="warm")
    count, path, answer = C.verify_drafts(logits[:0], tokens[:0], uniform[:0])
    assert count.shape == (0,) and path.shape == (0, 3) and answer.shape == (0,)


def test_padded_batches(C):
    """Chains of unequal lengths in one batch: a token of -1 (or any outside of the vocabulary) ends a sequence's chain."""
    logits, draft, tokens, uniform = inputs(16, 6, 6, 3000, "bf16")
    for b in range(6):
        tokens[b, 1 + b:] = (-1, 3000, 2 ** 40, -(2 ** 40), -5, 0)[b]
    uniform[:, :6] *= 0.2
    want = check(C, logits, tokens, uniform, draft)
    assert want[0].tolist()[0] == 1 and want[0].max() > 2
    check(C, logits, tokens, uniform)


def test_no_drafted_rows(C, dev):
    logits, _, tokens, uniform = inputs(17, 5, 1, 7777, "fp16")
    want = check(C, logits, tokens, uniform)
    got = C.verify_drafts(logits.to(dev), tokens.to(dev), uniform.to(dev), draft=torch.empty(5, 0, 7777, dtype=torch.float16, device=dev))
    assert got[2].tolist() == want[2].tolist() and got[0].tolist() == [1] * 5


@pytest.mark.parametrize("B,R,V", [(1024, 3, 40), (1, 2, (1 << 24) - 1), (2, 64, 2100)])
def test_the_largest(C, B, R, V):
    """The most sequences, the largest vocabulary (more runs than the draw holds at once), the most rows."""
    logits, draft, tokens, uniform = inputs(18, B, R, V, "bf16")
    check(C, logits, tokens, uniform, draft, heat=0.9)


def test_draws_in_every_run(C, dev):
    """Equal weights: the draw is u of the vocabulary itself, at either side of every run's border."""
    V, B = 151936, 1024
    logits = torch.zeros(1, 1, V, dtype=torch.bfloat16, device=dev).expand(B, 1, V)
    u = torch.zeros(B, 2, dtype=torch.float64)
    at = torch.tensor([min(V - 1, i // 2 * 512 + (i % 2) * 511) for i in range(B)])
    u[:, 1] = (at.double() + 0.5) / V
    got = C.verify_drafts(logits, torch.zeros(B, 1, dtype=torch.int64, device=dev), u.to(dev))
    assert torch.equal(got[2].cpu(), at)


@pytest.mark.parametrize("B,R,V", [(1024, 3, 40), (1, 2, (1 << 24) - 1), (2, 64, 2100), (3, 64, 30000)])
def test_the_largest_without_draft_probabilities(C, B, R, V):
    """As chains, and as trees whose rows are all children of the first one, distinct tokens and (in the last sequence) one alone."""
    logits, _, tokens, uniform = inputs(31, B, R, V, "bf16")
    check(C, logits, tokens, uniform, heat=0.9)
    tokens[:, 1:] = logits[:, 0].float().topk(R - 1, -1).indices.flip(-1)
    tokens[-1, 1:] = tokens[-1, 1]
    for u in (uniform, 0.9 + 0.1 * uniform):
        check(C, logits, tokens, u, parent=torch.zeros(B, R, dtype=torch.int32), heat=0.9)


@pytest.mark.parametrize("V", [5000, 9000])
def test_many_short_vocabularies(C, V):
    """Work-groups of several runs each."""
    logits, draft, tokens, uniform = inputs(32, 1024, 2, V, "bf16")
    check(C, logits, tokens, uniform, draft)


def test_extreme_temperatures_without_draft_probabilities(C):
    """References far from zero that differ between the waves of a row, runs far below it, masked ones."""
    logits, _, tokens, uniform = inputs(33, 8, 3, 60000, "fp32")
    logits[6, :, :30000] -= 3000.0
    logits[7, :, 700:] = float("-inf")
    heat = torch.tensor([1e-30, 1e-3, 50.0, 1e30, 2.0 ** -140, 0.004, 1.0, 0.01])
    best = logits.topk(3, -1).indices
    for rank in (0, 1):
        tokens[:, 1:] = best[:, :2, rank]
        check(C, logits, tokens, uniform, heat=heat)
        # A uniform of 0 is passed by any weight. Which ones there are depends on where the range of a 64-bit exponential ends:
        # the oracle's at 2^-1074 of the largest; the kernel's at 2^-1009 of a reference that is up to 2^900 above that (0 while
        # the largest logit's own exponent is within 900 of it). No weight below the answer's is 2^(900 - 1009) of the largest.
        out = C.verify_drafts(logits.cuda(), tokens.cuda(), uniform.cuda() * 0, temperature=heat.cuda())
        want = ref.verify_drafts(f64(logits), tokens.numpy(), uniform.numpy() * 0, heat=heat.numpy())
        assert out[0].tolist() == want[0].tolist() and out[1].tolist() == want[1].tolist()
        for b, got in enumerate(out[2].tolist()):
            x = f64(logits[b, int(want[1][b][want[0][b] - 1])])
            steps = (x - x.max()) / float(heat[b]) / np.log(2.0)
            assert 0 <= got and np.isfinite(x[got]) and (steps[:got] < 900 - 1009 + 1e-6).all()
    check(C, logits, tokens, 1.0 - (1.0 - uniform) * 2.0 ** -20, heat=heat)


def test_likely_children_refused(C):
    """A child that has nearly all of a run's weight, or of the row's, is refused: the draw is from what its run has beside it."""
    B, V = 12, 4096
    logits, _, tokens, uniform = inputs(34, B, 3, V, "fp32", spread=0.2)
    at = torch.arange(B) * 341 + 5
    for b in range(B):
        logits[b, :, at[b]] = 8.0 + 3.0 * b  # (up to e^41 times the others)
        tokens[b, 1] = at[b]
        tokens[b, 2] = at[b] + 1
    parent = torch.zeros(B, 3, dtype=torch.int32)
    p = torch.tensor([1.0 - ref.token_probabilities(f64(logits[b, 0]), 1.0)[[int(at[b]), int(at[b]) + 1]].sum() for b in range(B)], dtype=torch.float64)
    uniform[:, 0] = torch.clamp(1.0 - p * 0.25, max=1.0 - 2.0 ** -53)
    want = check(C, logits, tokens, uniform, parent=parent)
    assert (want[0][:9] == 1).all()
    assert all(int(t) not in (int(i), int(i) + 1) for t, i in zip(want[2][:9], at[:9]))


def test_strided_rows_without_draft_probabilities(C, dev):
    for dt in ("bf16", "fp32"):
        logits, _, tokens, uniform = inputs(35, 3, 4, 8190, dt)
        tokens[:, 1:] = logits[:, :3].float().argmax(-1)
        for off, pad in ((1, 3), (3, 0), (5, 8), (7, 1)):
            wide = torch.full((3, 4, 8190 + off + pad), 99.0, dtype=DT[dt], device=dev)
            view = wide[:, :, off:off + 8190]
            view.copy_(logits)
            got = C.verify_drafts(view, tokens.to(dev), uniform.to(dev), temperature=0.9)
            want = ref.verify_drafts(f64(logits), tokens.numpy(), uniform.numpy(), heat=0.9)
            assert [g.cpu().tolist() for g in got] == [w.tolist() for w in want]


def test_replay_without_draft_probabilities(C, dev):
    a = [inputs(40 + i, 5, 6, 40000, "bf16") for i in range(3)]
    parent = torch.tensor([[0, 0, 0, 1, 1, 2]] * 5, dtype=torch.int32)
    for _, _, tokens, uniform in a:
        uniform[:, :6] *= 0.3
    for x in a:
        best = x[0].float().topk(2, -1).indices
        for r in range(1, 6):
            x[2][:, r] = best[:, parent[0, r], r % 2]
    hold = [t.to(dev) for t in (a[0][0], a[0][2], a[0][3], parent)]
    C.verify_drafts(*hold[:3], parent=hold[3])
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        out = C.verify_drafts(*hold[:3], parent=hold[3])
    for i in (1, 2, 0, 1):
        for h, t in zip(hold, (a[i][0], a[i][2], a[i][3])):
            h.copy_(t)
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            beside = C.verify_drafts(a[2][0].to(dev), a[2][2].to(dev), a[2][3].to(dev), parent=parent.to(dev))
        torch.cuda.synchronize()
        for got, x in ((out, a[i]), (beside, a[2])):
            want = ref.verify_drafts(f64(x[0]), x[2].numpy(), x[3].numpy(), parent=parent.numpy())
            assert [g.cpu().tolist() for g in got] == [w.tolist() for w in want]


@pytest.mark.parametrize("B,R,V", [(1, 1, 9000), (3, 3, 9000), (64, 3, 60000), (512, 2, 20000), (1, 2, 600000)])
def test_runs_that_the_largest_leaves_nothing_of(C, B, R, V):
    """Runs within the exponentials' range by themselves, ahead of a logit that leaves them less than that range holds: a uniform of
    0 passes none of them. (Weights of 2^-1154 of the largest at most: none in 64 bits.)"""
    g = torch.Generator().manual_seed(36)
    logits = torch.rand(B, R, V, generator=g) * 12 - 6  # (866 octaves at most at a temperature of 0.01)
    at = 2048 + torch.randint(0, V - 2048, (B, R), generator=g)
    logits.scatter_(2, at[..., None], 14.0)  # 2020
    tokens = torch.zeros(B, R, dtype=torch.int64)
    uniform = torch.rand(B, R + 1, generator=g, dtype=torch.float64)
    uniform[:, R] = 0.0
    tokens[:, 1:] = at[:, :R - 1]
    want = check(C, logits, tokens, uniform, heat=0.01)
    assert (want[0] == R).all() and want[2].tolist() == at[:, -1].tolist()
    tokens[:, 1:] = 7  # (refused)
    want = check(C, logits, tokens, uniform, heat=0.01)
    assert (want[0] == 1).all() and want[2].tolist() == at[:, 0].tolist()


def test_uniforms_beside_the_borders(C, dev):
    """Uniforms 1e-14 to either side of a border of the cumulative probabilities (80-bit oracle), logits within 4 of 0. A weight's
    relative error: the exponential's polynomial 1.2e-15 and table 3.4e-16, the argument's two roundings (4 2^-53 each, and the rate's
    4 2^-52), its own 2^-53: under 4e-15 in all; a border moves by at most half of that and some roundings of 2^-53: under 3e-15."""
    g = torch.Generator().manual_seed(37)
    B, V = 1024, 5
    logits = torch.rand(B, 1, V, generator=g) * 8 - 4
    w = np.exp(logits[:, 0].double().numpy().astype(np.longdouble))
    p = w / w.sum(1, keepdims=True)
    upto = np.cumsum(p, 1)
    at = np.arange(B) % (V - 1)
    border = upto[np.arange(B), at]
    none = torch.full((B, 2), -1, dtype=torch.int64)
    for side, want in ((-1, at), (1, at + 1)):
        uniform = torch.zeros(B, 3, dtype=torch.float64)
        uniform[:, 1] = uniform[:, 2] = torch.from_numpy((border + side * np.longdouble(1e-14)).astype(np.float64))
        one = C.verify_drafts(logits.to(dev), none[:, :1].to(dev), uniform[:, :2].contiguous().to(dev))
        assert one[2].tolist() == want.tolist()
        two = logits.expand(B, 2, V).to(dev)  # (with draft probabilities: no token behind row 0)
        assert C.verify_drafts(two, none.to(dev), uniform.to(dev), draft=two[:, :1])[2].tolist() == want.tolist()
        # children of one row split [0, 1) at the same borders
        tokens = torch.arange(-1, V).repeat(B, 1)
        uniform = torch.zeros(B, V + 2, dtype=torch.float64)
        uniform[:, 0] = torch.from_numpy((border + side * np.longdouble(1e-14)).astype(np.float64))
        got = C.verify_drafts(logits.expand(B, V + 1, V).to(dev), tokens.to(dev), uniform.to(dev), parent=torch.zeros(B, V + 1, dtype=torch.int32, device=dev))
        assert got[1][:, 1].tolist() == (want + 1).tolist()
    # acceptance: u q(x) against p(x)
    other = torch.rand(B, 1, V, generator=g) * 8 - 4
    w = np.exp(other[:, 0].double().numpy().astype(np.longdouble))
    q = w / w.sum(1, keepdims=True)
    x = (q - p).argmax(1)
    ratio = p[np.arange(B), x] / q[np.arange(B), x]
    tokens = torch.stack([torch.zeros(B, dtype=torch.int64), torch.from_numpy(x)], 1)
    for side, want in ((-1, 2), (1, 1)):
        uniform = torch.full((B, 3), 0.5, dtype=torch.float64)
        uniform[:, 0] = torch.from_numpy((ratio * (1 + side * np.longdouble(2e-14))).astype(np.float64))
        got = C.verify_drafts(logits.expand(B, 2, V).to(dev), tokens.to(dev), uniform.to(dev), draft=other.to(dev))
        assert got[0].tolist() == [want] * B
