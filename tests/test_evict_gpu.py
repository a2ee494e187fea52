"""page_evict on the GPU against the oracle's sequential restatement: kept tokens, moved rows, masses and bookkeeping equal, mean
keys within fp32 sums and one rounding."""
import numpy as np
import pytest
import torch

from oracle import ref
from paged_cases import UNIT

pytestmark = pytest.mark.gpu
BF, FH = torch.bfloat16, torch.float16
NAMES = ("kv", "ksum", "table", "length", "refs", "mass")


class State:
    """A small cache of B sequences in a pool of P pages with the masses of their tokens, on the host."""

    def __init__(self, seed, lens, L=2, Hk=2, P=60, T=16, D=64, W=8, dt=BF, extra=0, ties=False):
        g = torch.Generator().manual_seed(seed)
        self.kv = torch.randn(L, 2, Hk, P, T, D, generator=g).to(dt)
        self.ksum = torch.randn(L, Hk, P, D, generator=g).to(dt)
        self.table = torch.full((len(lens), W), -1, dtype=torch.int32)
        order, at = torch.randperm(P, generator=g), 0
        self.refs = torch.zeros(P, dtype=torch.int32)
        for b, n in enumerate(lens):
            e = min(W, -(-n // T))
            self.table[b, :e] = order[at:at + e]
            self.refs[order[at:at + e]] = 1
            at += e
        self.length = torch.tensor(lens, dtype=torch.int32)
        self.mass = torch.randn(L, len(lens), Hk, W * T + extra, generator=g).exp()
        if ties:
            self.mass = torch.randint(-1, 3, self.mass.shape, generator=g).float()

    def tensors(self):
        return [self.kv, self.ksum, self.table, self.length, self.refs, self.mass]

    def dev(self, dev):
        return [x.to(dev) for x in self.tensors()]

    def host(self):
        return [x.float().numpy() if x.is_floating_point() else x.numpy().astype(np.int64) for x in self.tensors()]


def i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def compare(st, got, want, status, kept, slots):
    dt = st.kv.dtype
    for g, w, what in zip(got + [status, kept, slots], list(want), NAMES + ("status", "kept", "slots")):
        g = g.detach().cpu()
        if what == "ksum":
            # T fp32 sums, each within 2^-24 of the sum of magnitudes (at most T times the largest), and the rounding to the type
            g, T = g.double().numpy(), st.kv.shape[4]
            lim = UNIT[dt] * np.abs(w) + T * 2.0 ** -24 * st.kv.abs().max().item() + 2.0 ** -24 * (dt == FH)
            assert (np.abs(g - w) <= lim).all(), what
            continue
        g = g.float().numpy() if g.is_floating_point() else g.numpy()
        assert np.array_equal(g, np.asarray(w).astype(g.dtype), equal_nan=g.dtype.kind == "f"), what


def evict(C, dev, st, dst, src, keep, sinks=0, recent=0, room=0):
    print(f"page_evict dst={dst} src={src} keep={keep} sinks={sinks} recent={recent} room={room} kv={tuple(st.kv.shape)} lens={st.length.tolist()[:12]}", flush=True)
    d = st.dev(dev)
    slots = torch.full((len(dst), room), -9, dtype=torch.int64, device=dev)
    status, kept = C.page_evict(*d, i32(dst, dev), i32(src, dev), keep, sinks, recent, room, slots)
    want = ref.page_evict(*st.host(), dst, src, keep, sinks, recent, room)
    compare(st, d, want, status, kept, slots)
    return status.tolist()


@pytest.mark.parametrize("keep,sinks,recent", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (5, 4, 3), (30, 0, 16), (16, 16, 16), (64, 30, 34), (500, 0, 0), (0, 7, 9)])
@pytest.mark.parametrize("ties", [False, True])
def test_in_place_and_as_copies(C, dev, keep, sinks, recent, ties):
    st = State(1, [0, 1, 15, 16, 17, 40, 64, 127, 128, 0, 33, 5], P=120, ties=ties)
    assert set(evict(C, dev, st, [7, 5, 9, 0, 6, 1, 3], [7, 5, 7, 0, 8, 1, 8], keep, sinks, recent, 3 if keep + sinks + recent < 100 else 0)) == {1}


@pytest.mark.parametrize("dt", [BF, FH])
@pytest.mark.parametrize("T,D", [(16, 64), (16, 256), (32, 128), (64, 64), (128, 128), (256, 256), (1024, 64)])
def test_page_sizes(C, dev, dt, T, D):
    lens = [3 * T + 5, 2 * T, T - 1, 0]
    st = State(T + D, lens, L=1, Hk=3, P=20, T=T, D=D, W=4, dt=dt)
    evict(C, dev, st, [0, 3, 2], [0, 1, 2], T + 3, 2, T // 2, 5)
    evict(C, dev, st, [3], [0], 2 * T - 1, 0, 1)


@pytest.mark.parametrize("n", [16383, 16384, 16385, 40000])
@pytest.mark.parametrize("ties", [False, True])
def test_long_sequences(C, dev, n, ties):
    """Rounds of 16384 tokens: thresholds whose ties span them."""
    st = State(3, [n, 9], L=1, Hk=2, P=2 * (n // 64) + 20, T=64, W=n // 64 + 2, ties=ties)
    evict(C, dev, st, [0], [0], n // 2 + 11, 5, 100)
    evict(C, dev, st, [1, 0], [0, 0], 300, 0, 0, 70)


def test_masses_of_every_kind(C, dev):
    """Zeros of both signs, negative and denormal masses, infinities, NaN, all alike; rows that stand at no 16-byte boundary."""
    for extra in (0, 1, 3):
        st = State(4, [120, 120, 120, 120, 100], P=80, extra=extra)
        st.mass[:, 0, :, ::3] = 0.0
        st.mass[:, 0, :, 1::3] = -0.0
        st.mass[:, 1, :, ::2] *= -1
        st.mass[:, 1, :, 10:20] = 1e-42
        st.mass[:, 2, :, ::4] = float("nan")
        st.mass[:, 2, :, 1::4] = float("inf")
        st.mass[:, 2, :, 2::8] = -float("inf")
        st.mass[:, 3] = 2.5
        for keep in (10, 45, 80, 100):
            evict(C, dev, st, [0, 1, 2, 3, 4], [0, 1, 2, 3, 2], keep, 2, 3)


def test_reads_the_state_before_the_call(C, dev):
    """Sequences that change places, thinned."""
    st = State(5, [100, 90, 80, 0], P=80)
    evict(C, dev, st, [0, 1, 2, 3], [1, 2, 0, 0], 20, 1, 1, 4)


def test_shared_pages_stay(C, dev):
    """A fork and its source, one of them thinned: the other's pages keep their rows and references."""
    st = State(6, [100, 0, 30], P=60)
    d = st.dev(dev)
    C.page_fork(*d[:5], i32([1], dev), i32([0], dev))
    st.kv, st.ksum, st.table, st.length, st.refs, st.mass = (x.cpu() for x in d)
    evict(C, dev, st, [1], [1], 10, 4, 10, 2)
    evict(C, dev, st, [0, 1], [1, 0], 30, 4, 10, 2)


def test_too_few_pages_and_refused(C, dev):
    st = State(7, [120, 120, 30, 0], P=22)  # 18 pages in use
    assert evict(C, dev, st, [0, 1, 2, 3], [0, 1, 2, 1], 40, 0, 0) == [1, 0, 1, 0]
    assert evict(C, dev, st, [2, 0], [2, 2], 100, 0, 0, 200) == [-1, -1]
    assert evict(C, dev, st, [0, 0, 4, -1, 1, 2], [2, 1, 0, 0, -1, 4], 10) == [1, -1, -1, -1, -1, -1]
    st.refs[st.refs == 0] = 1
    assert evict(C, dev, st, [2, 0], [2, 0], 60, 0, 0) == [1, 0]


def test_room_of_sequences_that_stay(C, dev):
    """A sequence with no more than the kept tokens: its missing entries alone are given."""
    st = State(8, [40, 17, 0], P=40)
    assert evict(C, dev, st, [0, 1, 2], [0, 1, 2], 64, 0, 0, 60) == [1, 1, 1]
    st.table[0, 4] = 40  # (no page)
    assert evict(C, dev, st, [0], [0], 64, 0, 0, 60) == [1]


def test_bad_entries_and_lengths(C, dev):
    st = State(9, [100, 90, 500, -4], P=60)
    st.table[0, 2], st.table[0, 4] = -1, 60
    evict(C, dev, st, [0, 1, 2, 3], [0, 0, 1, 3], 50, 3, 10, 4)
    st = State(9, [100, 90, 500, -4], P=60)
    evict(C, dev, st, [0, 2], [2, 3], 50, 3, 10, 4)


def test_many_pairs_and_layers(C, dev):
    st = State(10, [(7 * i) % 65 for i in range(300)], L=3, Hk=2, P=1500, W=5)
    evict(C, dev, st, list(range(300)), [(i * 7 + 3) % 300 for i in range(300)], 12, 1, 5, 1)


def test_without_mean_keys(C, dev):
    st = State(11, [100, 0], P=40)
    d = st.dev(dev)
    ksum = d[1].clone()
    status, kept = C.page_evict(d[0], None, *d[2:], i32([1], dev), i32([0], dev), 30)
    want = ref.page_evict(*st.host(), [1], [0], 30, 0, 0, 0)
    assert torch.equal(d[1], ksum) and status.tolist() == [1] and kept.cpu().numpy().tolist() == want[7].tolist()
    assert np.array_equal(d[0].cpu().float().numpy(), want[0])


def test_replay(C, dev):
    """A captured eviction beside eager ones on another cache and stream, over changing masses and lengths."""
    st = State(12, [100, 128, 60], P=60)
    d, w = st.dev(dev), st.dev(dev)
    dst, src = i32([0, 1, 2], dev), i32([0, 1, 2], dev)
    slots = torch.zeros(3, 2, dtype=torch.int64, device=dev)
    C.page_evict(*w, dst, src, 20, 2, 8, 2, slots)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        status, kept = C.page_evict(*d, dst, src, 20, 2, 8, 2, slots)
    for k, lens in enumerate(([100, 128, 60], [30, 31, 90], [77, 0, 128])):
        st = State(13 + k, lens, P=60)
        for x, y, z in zip(d, w, st.tensors()):
            x.copy_(z), y.copy_(z)
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            other = C.page_evict(*w, dst, src, 20, 2, 8, 2)
        torch.cuda.synchronize()
        want = ref.page_evict(*st.host(), [0, 1, 2], [0, 1, 2], 20, 2, 8, 2)
        compare(st, d, want, status, kept, slots)
        compare(st, w, want, *other, slots)


def test_refusals(C, dev):
    st = State(14, [50, 20], P=20)
    d, two = st.dev(dev), i32([0, 1], dev)
    kv, ksum, table, length, refs, mass = d
    for args, match in (((kv, ksum, table, length, refs, mass.double(), two, two, 5), "mass"), ((kv, ksum, table, length, refs, mass[:1], two, two, 5), "mass"),
                        ((kv, ksum, table, length, refs, mass[..., :64].contiguous(), two, two, 5), "mass"), ((kv, ksum, table, length, refs, mass[..., ::2], two, two, 5), "mass"),
                        ((kv, ksum, table, length, refs, mass, two, i32([0], dev), 5), "src"), ((kv, ksum, table, length, refs, mass, two.long(), two, 5), "dst"),
                        ((kv, ksum, table, length, refs, mass, two, two, 0), "kept"), ((kv, ksum, table, length, refs, mass, two, two, -1, 5), "kept"),
                        ((kv, ksum, table, length, refs, mass, two, two, 5, 0, 0, -1), "room"), ((kv.float(), ksum, table, length, refs, mass, two, two, 5), "kv"),
                        ((kv, ksum, table, length, refs, mass, two, two, 1 << 29), "too many"), ((kv, ksum, table, length, refs, mass.cpu(), two, two, 5), "same ROCm device")):
        with pytest.raises(RuntimeError, match=match):
            C.page_evict(*args)
    with pytest.raises(RuntimeError, match="slots"):
        C.page_evict(*d, two, two, 5, room=3, slots=torch.zeros(2, 2, dtype=torch.int64, device=dev))
    status, kept = C.page_evict(*d, two[:0], two[:0], 5)
    assert status.shape == (0,) and kept.shape == (0, 2, 2, 5)


def test_offsets_past_32_bits(C, dev):
    """Kept rows and fresh pages past 2^32 bytes of a chunk's base."""
    st = State(15, [90, 0, 40], L=1, Hk=1, P=12, T=32, D=256, W=4)
    P = 270000  # a chunk of 4.4 GB
    base = P - 12
    kv = torch.empty(1, 2, 1, P, 32, 256, dtype=BF, device=dev)
    kv[:, :, :, base:] = st.kv.to(dev)
    ksum = torch.zeros(1, 1, P, 256, dtype=BF, device=dev)
    ksum[:, :, base:] = st.ksum.to(dev)
    refs = torch.ones(P, dtype=torch.int32, device=dev)
    refs[base:] = st.refs.to(dev)
    table = torch.where(st.table >= 0, st.table + base, st.table).to(dev)
    length, mass = st.length.to(dev), st.mass.to(dev)
    slots = torch.zeros(2, 3, dtype=torch.int64, device=dev)
    status, kept = C.page_evict(kv, ksum, table, length, refs, mass, i32([0, 1], dev), i32([0, 2], dev), 30, 2, 5, 3, slots)
    want = ref.page_evict(*st.host(), [0, 1], [0, 2], 30, 2, 5, 3)
    got = [kv[:, :, :, base:], ksum[:, :, base:], torch.where(table >= 0, table - base, table), length, refs[base:], mass]
    compare(st, got, want, status, kept, torch.where(slots >= 0, slots - base * 32, slots))


def test_the_most_pairs(C, dev):
    st = State(16, [(5 * i) % 33 for i in range(1024)], L=1, Hk=1, P=4000, W=3)
    evict(C, dev, st, list(range(1024)), list(range(1024)), 7, 1, 3, 2)


def test_more_kept_than_a_table_holds(C, dev):
    st = State(17, [100, 128, 0], P=60)
    assert evict(C, dev, st, [0, 1, 2], [1, 1, 0], 5000, 100, 100) == [1, 1, 1]


@pytest.mark.parametrize("L,Hk,T,D,W,B,long,keep,sinks,recent", [(129, 8, 16, 64, 2, 1024, 0, 5, 1, 2), (32, 8, 16, 128, 133, 1024, 2100, 2043, 1, 4)])
def test_more_units_than_a_launch_has_work_groups(C, dev, L, Hk, T, D, W, B, long, keep, sinks, recent):
    """1024 pairs of many layers and heads: over 2^20 selections; 2^24 moves, as the table's width has it. The sequences become thinned
    copies of 40 short ones (and of a long one)."""
    g = torch.Generator().manual_seed(19)
    src = torch.randint(0, 40, (B,), generator=g)
    lens = torch.randint(0, min(33, W * T + 1), (B,), generator=g)
    lens[40:] = 0
    if long:
        lens[3] = long
        src[src == 3] = 4
        src[7] = src[B - 1] = 3
    used, most = -(-lens // T), keep + sinks + recent
    P = int(used.sum()) + int((-(-lens.clamp(max=most) // T))[src].sum())
    print(f"page_evict {B} pairs of {L} layers of {Hk} heads, {P} pages", flush=True)
    order, table, at = torch.randperm(P, generator=g), torch.full((B, W), -1, dtype=torch.int32), 0
    refs = torch.zeros(P, dtype=torch.int32)
    for b in range(40):
        e = int(used[b])
        table[b, :e] = order[at:at + e]
        refs[order[at:at + e]] = 1
        at += e
    kv = torch.empty(L, 2, Hk, P, T, D, dtype=BF, device=dev)
    for part in kv.view(L, -1):
        part.normal_()
    mass = torch.rand(L, 40, Hk, W * T, generator=g).to(dev)
    whole = torch.zeros(L, B, Hk, W * T, device=dev)
    whole[:, :40] = mass
    rows = []  # (what the sources' tokens hold, before the call)
    for b in range(40):
        t = torch.arange(int(lens[b]))
        rows.append(kv[:, :, :, table[b, t // T].long().to(dev), (t % T).to(dev)])
    table, refs = table.to(dev), refs.to(dev)
    status, kept = C.page_evict(kv, None, table, lens.to(torch.int32).to(dev), refs, whole, i32(range(B), dev), i32(src.tolist(), dev), keep, sinks, recent)
    assert (status == 1).all()
    want = []  # the kept tokens of every source: forced ones ahead of the masses, ties at the lowest
    for b in range(40):
        n = int(lens[b])
        worth = mass[:, b, :, :n].clone()
        worth[..., :sinks] = worth[..., max(0, n - recent):] = 2.0
        want.append(worth.sort(dim=-1, descending=True, stable=True).indices[..., :most].sort(-1).values)
    table = table.cpu()
    for i in range(B):
        keys, held = want[int(src[i])], rows[int(src[i])]
        n = keys.shape[-1]
        if int(src[i]) == i and n == int(lens[i]):
            continue  # (it stays)
        assert torch.equal(kept[i, :, :, :n].long(), keys) and (kept[i, :, :, n:] == -1).all(), i
        t = torch.arange(n)
        got = kv[:, :, :, table[i, t // T].long().to(dev), (t % T).to(dev)]
        assert torch.equal(got, held.gather(3, keys[:, None, :, :, None].expand(L, 2, Hk, n, D))), i
        assert torch.equal(whole[:, i, :, :n], mass[:, int(src[i])].gather(2, keys)), i


@pytest.mark.parametrize("pairs", [1, 3, 4, 300])
def test_sources_with_a_token_in_no_page_are_refused(C, dev, pairs):
    """Its place in a fresh page would be attended, with the rows that a sequence before left there. What is behind the source's last
    token, and a sequence that stays, need no page."""
    st = State(20, [100, 100, 90, 40] + [20 + i % 13 for i in range(296)], P=1000)
    st.kv[:, :, :, st.refs == 0] = 7.0  # (the pool's free pages hold something)
    for bad in (-1, 1000, 2 ** 31 - 1, -2 ** 31):
        for at, refused in ((0, 1), (6, 1), (7, 0)):  # (the first, the last of 100 tokens, one behind them)
            st.table[1, at], was = bad, st.table[1, at].clone()
            src = [1, 0, 2, 1] if pairs < 300 else [(i * 7 + 1) % 300 for i in range(300)]
            status = evict(C, dev, st, list(range(pairs)), src[:pairs], 50, 2, 8, 3)
            assert [x == -1 for x in status] == [bool(refused) and s == 1 for s in src[:pairs]]  # (of 300 the last find too few pages)
            st.table[1, at] = was
    st.table[3, 1], st.table[2, 0] = -1, -1
    assert evict(C, dev, st, [3, 2, 0], [3, 2, 0], 50, 2, 8, 3) == [1, -1, 1]  # (40 tokens stay as they are)


def test_a_hole_in_a_long_table(C, dev):
    """The last entry of 3001."""
    st = State(21, [48010, 0], L=1, Hk=1, P=3010, T=16, W=3002)
    for at, want in ((3000, -1), (1500, -1), (3001, 1)):
        st.table[0, at], was = -1, st.table[0, at].clone()
        assert evict(C, dev, st, [1], [0], 20, 1, 5) == [want]
        st.table[0, at] = was


def test_no_page_for_tokens_that_a_staying_sequence_has(C, dev):
    """The page that its length ends in is missing: a fresh one would make its tokens another sequence's rows."""
    st = State(22, [40, 48, 40, 33], P=60)
    st.kv[:, :, :, st.refs == 0] = 7.0
    st.table[0, 2], st.table[1, 2], st.table[2, 1] = -1, -1, 60
    for room in (0, 20):
        assert evict(C, dev, st, [0, 1, 2, 3], [0, 1, 2, 3], 50, 2, 8, room) == [-1, 1, 1, 1]  # (48 tokens end at a page's end)
