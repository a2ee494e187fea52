"""page_fork and page_commit on the GPU against the oracle's sequential restatement: moved rows and bookkeeping equal, mean keys
within fp32 sums and one rounding."""
import numpy as np
import pytest
import torch

from oracle import ref
from paged_cases import UNIT

pytestmark = pytest.mark.gpu
BF, FH = torch.bfloat16, torch.float16


class State:
    """A small cache of B sequences in a pool of P pages, on the host; dev() gives the tensors that the operators take."""

    def __init__(self, seed, lens, L=2, Hk=2, P=40, T=16, D=64, W=8, held=0, dt=BF):
        g = torch.Generator().manual_seed(seed)
        self.kv = torch.randn(L, 2, Hk, P, T, D, generator=g).to(dt)
        self.ksum = torch.randn(L, Hk, P, D, generator=g).to(dt)
        self.table = torch.full((len(lens), W), -1, dtype=torch.int32)
        order, at = torch.randperm(P, generator=g), 0
        self.refs = torch.zeros(P, dtype=torch.int32)
        for b, n in enumerate(lens):
            e = min(W, -(-(n + held) // T))
            self.table[b, :e] = order[at:at + e]
            self.refs[order[at:at + e]] = 1
            at += e
        self.length = torch.tensor(lens, dtype=torch.int32)

    def dev(self, dev):
        return [x.to(dev) for x in (self.kv, self.ksum, self.table, self.length, self.refs)]

    def host(self):
        return [x.float().numpy() if x.is_floating_point() else x.numpy().astype(np.int64)
                for x in (self.kv, self.ksum, self.table, self.length, self.refs)]


def _same(got, want, what):
    got = got.detach().cpu()
    got = got.float().numpy() if got.is_floating_point() else got.numpy()
    assert np.array_equal(got, np.asarray(want).astype(got.dtype)), what


def _fork(C, dev, st, dst, src, room=0, share=True):
    print(f"page_fork dst={dst} src={src} room={room} share={share} kv={tuple(st.kv.shape)}", flush=True)
    d = st.dev(dev)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    slots = torch.full((len(dst), room), -9, dtype=torch.int64, device=dev)
    status = C.page_fork(*d, i32(dst), i32(src), room, share, slots)
    kv, ksum, table, length, refs, st_, sl = ref.page_fork(*st.host(), dst, src, room, share)
    for got, want, what in zip(d + [status, slots], (kv, ksum, table, length, refs, st_, sl), ("kv", "ksum", "table", "length", "refs", "status", "slots")):
        _same(got, want, what)
    return status.tolist()


@pytest.mark.parametrize("share", [True, False])
@pytest.mark.parametrize("lens", [[0, 1, 15, 16, 17], [33, 64, 47, 5, 0]])
def test_fork(C, dev, share, lens):
    st = State(1, lens + [20, 0, 0, 40, 9], P=90, held=6)
    assert _fork(C, dev, st, [5, 6, 7, 8, 9], [0, 1, 2, 3, 4], 18, share) == [1] * 5


def test_fork_reads_the_state_before_the_call(C, dev):
    """A permutation of beams, one parent taken twice, a place kept, a place emptied."""
    st = State(2, [20, 37, 48, 5, 63], P=60, held=4)
    assert _fork(C, dev, st, [0, 1, 2, 3, 4], [1, 0, 1, 3, -1], 20) == [1] * 5


def test_fork_of_a_fork_and_drops(C, dev):
    """Shared pages' references over several calls: nothing is lost when all sequences are dropped."""
    st = State(3, [70, 0, 0, 0], P=40, held=2)
    d = st.dev(dev)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    free = int((d[4] == 0).sum())
    C.page_fork(*d, i32([1, 2]), i32([0, 0]))
    C.page_fork(*d, i32([3]), i32([1]))
    assert d[4].max().item() == 4 and d[3].tolist() == [70] * 4
    C.page_fork(*d, i32([0, 1]), i32([-1, -1]))
    assert d[4].max().item() == 2 and d[3].tolist() == [0, 0, 70, 70]
    C.page_fork(*d, i32([2, 3]), i32([-1, -1]))
    assert (d[4] == 0).all() and (d[2] == -1).all() and free < d[4].numel()


def test_fork_without_pages_and_refused(C, dev):
    st = State(4, [60, 33, 10, 0, 0], P=12, held=0, W=5)
    # 4 + 3 + 1 pages held, 4 free: copies of 60 + 8 tokens need five; 10 + 20 tokens two, and then 60 + 20 five more
    assert _fork(C, dev, st, [3, 4, 2], [0, 1, 2], 8, False) == [0, 0, 0]
    assert _fork(C, dev, st, [3, 4], [2, 0], 20, False) == [1, 0]
    assert _fork(C, dev, st, [3, 4], [2, 0], 20, True) == [1, 1]
    assert _fork(C, dev, st, [3, 3, 7, -1, 4, 2], [2, 1, 0, 0, 5, 0], 0) == [1, -1, -1, -1, -1, 1]
    assert _fork(C, dev, st, [3], [0], 21) == [-1]


def test_fork_new_sequences_and_many_pairs(C, dev):
    st = State(5, [10] + [0] * 300, P=700, T=16, W=6, L=1, Hk=1)
    assert _fork(C, dev, st, list(range(1, 301)), [-1, 0] * 150, 17) == [1] * 300


def test_fork_bad_entries_and_lengths(C, dev):
    """Entries that are no page are neither copied nor counted; a length past the table is clamped."""
    st = State(6, [50, 20, 0, 0], P=40, held=0)
    st.table[0, 1], st.table[1, 1] = 99, -5
    assert _fork(C, dev, st, [2, 3], [0, 1], 3) == [1, 1]
    st.length[1] = -4
    assert _fork(C, dev, st, [2, 3], [0, 1], 3, False) == [1, 1]


def test_fork_large_pool(C, dev):
    """More references than one round of the search, the free ones at the end and unaligned."""
    st = State(7, [40, 0, 0], P=40001, L=1, Hk=1, T=16, D=8, W=5)
    st.refs[:] = 1
    st.refs[[39000, 39999, 40000, 17001, 16384]] = 0
    assert _fork(C, dev, st, [1, 2], [0, 0], 20) == [1, 1]


@pytest.mark.parametrize("dt", [BF, FH])
def test_fork_other_sizes(C, dev, dt):
    st = State(8, [300, 0], P=30, L=3, Hk=3, T=128, D=256, W=4, dt=dt)
    assert _fork(C, dev, st, [1], [0], 100, False) == [1]


def _commit(C, dev, st, count, path=None, room=0, in_place=True):
    print(f"page_commit count={count} path={path} room={room} kv={tuple(st.kv.shape)}", flush=True)
    d = st.dev(dev)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    new = None if in_place else torch.full_like(d[3], -9)
    slots = torch.full((len(count), room), -9, dtype=torch.int64, device=dev)
    status = C.page_commit(*d, i32(count), None if path is None else i32(path), room, new, slots)
    host = st.host()
    kv, table, length, refs, st_, sl, filled = ref.page_commit(host[0], *host[2:], count, path, room)
    for got, want, what in ((d[0], kv, "kv"), (d[2], table, "table"), (d[3] if in_place else new, length, "length"), (d[4], refs, "refs"),
                            (status, st_, "status"), (slots, sl, "slots")):
        _same(got, want, what)
    if not in_place:
        _same(d[3], st.length, "the old lengths")
    ksum, T = d[1].cpu().double().numpy(), st.kv.shape[4]
    for page, mean in filled:
        # T fp32 additions (each within 2^-24 of the sums' magnitude, at most the sum of |key|), one rounding
        heft = np.abs(kv[:, 0, :, page].astype(np.float64)).mean(-2)
        lim = T * 2.0 ** -24 * heft + UNIT[st.kv.dtype] * (np.abs(mean) + T * 2.0 ** -24 * heft) + 2.0 ** -24 * (st.kv.dtype == FH)
        assert (np.abs(ksum[:, :, page] - mean) <= lim).all()
    refused = [b for b, s in enumerate(st_) if s < 0]
    mine = {int(e) for b in refused for e in host[2][b] if e >= 0} | {p for p, _ in filled}
    others = [p for p in range(st.kv.shape[3]) if p not in mine]
    _same(d[1][:, :, others], host[1][:, :, others], "mean keys of other pages")
    return status.tolist()


@pytest.mark.parametrize("dt", [BF, FH])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_commit_trees(C, dev, dt, D):
    """Paths that overlap what they move over, whole and empty ones, pages that fill with moved rows, room over a page's end."""
    st = State(11, [0, 10, 14, 16, 31, 25, 3], P=40, held=8, D=D, dt=dt)
    path = [[0, 1, 2, 3, 4, 5, 6, 7], [0, 2, 3, 5, 7, 0, 0, 0], [1, 2, 3, 4, 5, 6, 7, 7], [0, 0, 0, 0, 0, 0, 0, 0], [7, 9, 9, 9, 9, 9, 9, 9],
            [0, 4, 6, 9, 9, 9, 9, 9], [0, 1, 2, 3, 4, 5, 6, 7]]
    assert _commit(C, dev, st, [8, 5, 7, 1, 1, 3, 0], path, 9) == [1] * 7


def test_commit_a_path_of_64(C, dev):
    st = State(12, [30, 77], P=40, held=64, W=12, L=3, Hk=5, D=256)
    path = [list(range(0, 64)), list(range(1, 64)) + [99]]
    assert _commit(C, dev, st, [64, 63], path, 3, in_place=False) == [1, 1]


@pytest.mark.parametrize("T,n,rows", [(16, 0, 100), (64, 37, 1000), (1024, 5, 3000), (32, 32, 32), (16, 3, 12)])
def test_commit_prompts(C, dev, T, n, rows):
    W = -(-(n + rows) // T) + 2
    st = State(13, [n, n + 1, 0], P=3 * W + 3, held=rows, W=W, T=T, L=1, D=128)
    assert _commit(C, dev, st, [rows, rows - 1, 1], None, T + 1) == [1, 1, 1]


def test_commit_refused_and_idle(C, dev):
    """Out of order, out of range, more rows than the path, rows without pages, a length past the table; -1: left alone."""
    st = State(14, [10, 20, 30, 40, 50, 60, 5, 127], P=60, held=4)
    st.table[4, 3] = -1
    st.table[5, 3] = 60
    path = [[0, 1, 1, 3], [0, 1, 2, 4], [0, 1, 2, 3], [-1, 1, 2, 3], [0, 1, 2, 3], [0, 1, 2, 3], [0, 1, 2, 3], [0, 1, 2, 3]]
    assert _commit(C, dev, st, [3, 4, 5, 2, 2, 2, -1, 2], path, 4) == [-1, -1, -1, -1, -1, -1, 1, -1]
    st.length[0] = -3
    assert _commit(C, dev, st, [1, 2, 3, 0, 0, 1, 0, 1], None, 4) == [-1, 1, 1, 1, -1, -1, 1, 1 if st.table.shape[1] * 16 >= 132 else 0]


def test_commit_without_pages(C, dev):
    """Too few free pages: committed all the same, the room of the first sequences given; room past the table's width."""
    st = State(15, [14, 30, 47, 0], P=10, held=2, W=4)
    assert _commit(C, dev, st, [2, 2, 1, 0], None, 17) == [1, 0, 0, 0]
    st = State(16, [60, 10], P=20, held=4, W=4)
    assert _commit(C, dev, st, [4, 1], None, 5) == [0, 1]


def test_commit_large_room(C, dev):
    """Room of many pages for one sequence beside small ones, not all of it in the table for another."""
    st = State(21, [14, 300, 0], P=900, held=2, W=300, L=1, Hk=1)
    assert _commit(C, dev, st, [2, 1, 0], None, 4000) == [1, 1, 1]
    st = State(22, [14, 900, 0], P=900, held=2, W=300, L=1, Hk=1)
    st.table[2, 5], st.table[2, 100] = st.table[1, 50], 10 ** 6
    assert _commit(C, dev, st, [2, 1, 0], None, 4000) == [1, 0, 1]


def test_commit_many_sequences(C, dev):
    g = torch.Generator().manual_seed(5)
    lens = [int(x) for x in torch.randint(0, 60, (1000,), generator=g)]
    st = State(17, lens, P=6000, held=3, L=1, Hk=1, W=6)
    path = [[0, 1, 2] if i % 2 else [0, 2, 9] for i in range(1000)]
    assert _commit(C, dev, st, [i % 4 % 3 + (i % 2) for i in range(1000)], path, 5) == [1] * 1000


def test_without_mean_keys(C, dev):
    st = State(18, [20, 0], P=20, held=4)
    d = st.dev(dev)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    assert C.page_fork(d[0], None, *d[2:], i32([1]), i32([0]), 4, False).tolist() == [1]
    assert C.page_commit(d[0], None, *d[2:], i32([4, 4])).tolist() == [1, 1]
    assert d[3].tolist() == [24, 24]


def test_replay(C, dev):
    """A captured commit replayed: every replay commits the next rows, as eager calls do."""
    st = State(19, [5, 30], P=60, held=8, W=10)
    d, e = st.dev(dev), st.dev(dev)
    count = torch.tensor([2, 3], dtype=torch.int32, device=dev)
    path = torch.tensor([[0, 3, 4], [0, 1, 5]], dtype=torch.int32, device=dev)
    slots, slots_e = (torch.empty(2, 8, dtype=torch.int64, device=dev) for _ in range(2))
    w = st.dev(dev)
    C.page_commit(*w, count, path, 8, slots=slots)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        status = C.page_commit(*d, count, path, 8, slots=slots)
    for _ in range(5):
        gr.replay()
        torch.cuda.synchronize()
        want = C.page_commit(*e, count, path, 8, slots=slots_e)
        for a, b in zip(d + [slots, status], e + [slots_e, want]):
            assert torch.equal(a, b)


def test_refusals(C, dev):
    st = State(20, [5, 30], P=20)
    kv, ksum, table, length, refs = st.dev(dev)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    two = i32([0, 1])
    for args, match in [((kv.float(), ksum, table, length, refs, two), "kv"), ((kv[:, :, :, ::2], ksum, table, length, refs, two), "kv"),
                        ((kv, ksum[:1], table, length, refs, two), "ksum"), ((kv, ksum, table.long(), length, refs, two), "table"),
                        ((kv, ksum, table.t(), length, refs, two), "table"), ((kv, ksum, table, length[:1], refs, two), "length"),
                        ((kv, ksum, table, length, refs[:5], two), "refs"), ((kv, ksum, table, length, refs, two.long()), "int32"),
                        ((kv, ksum, table, length, refs, two.cpu()), "same ROCm device")]:
        with pytest.raises(RuntimeError, match=match):
            C.page_commit(*args)
        with pytest.raises(RuntimeError, match=match):
            C.page_fork(*args, two)
    with pytest.raises(RuntimeError, match="64 rows"):
        C.page_commit(kv, ksum, table, length, refs, two, torch.zeros(2, 65, dtype=torch.int32, device=dev))
    with pytest.raises(RuntimeError, match="slots"):
        C.page_commit(kv, ksum, table, length, refs, two, None, 4, None, torch.zeros(2, 3, dtype=torch.int64, device=dev))
    with pytest.raises(RuntimeError, match="src"):
        C.page_fork(kv, ksum, table, length, refs, two, i32([0]))
    with pytest.raises(RuntimeError, match="room"):
        C.page_fork(kv, ksum, table, length, refs, two, two, -1)


@pytest.mark.parametrize("with_path", [True, False])
def test_commit_into_other_lengths(C, dev, with_path):
    """One launch for the move, the means and the plan: the same as in place, refused and starved sequences among them."""
    st = State(23, [10, 20, 30, 40, 47, 60, 5, 0], P=26, held=8, W=5)
    st.table[4, 3], st.table[5, 4] = -1, 70
    path = [[0, 1, 2, 3], [0, 2, 3, 3], [1, 0, 2, 3], [0, 1, 2, 4], [0, 1, 2, 3], [0, 1, 2, 3], [0, 3, 3, 3], [0, 1, 2, 3]]
    assert _commit(C, dev, st, [4, 3, 2, 4, 2, 4, 2, 0], path if with_path else None, 13, in_place=False)
    assert _commit(C, dev, st, [4, 3, 2, 4, 2, 4, -1, 0], path if with_path else None, 13)


@pytest.mark.parametrize("share", [True, False])
def test_fork_replay(C, dev, share):
    """A captured fork and one on another stream in turn with eager calls: the same tables, references and pages."""
    st = State(29, [37, 70, 0], P=90, held=8, W=10)
    d, e, w = st.dev(dev), st.dev(dev), st.dev(dev)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    dst, src, slots, slots_e = i32(2, 0), i32(0, 1), *(torch.empty(2, 5, dtype=torch.int64, device=dev) for _ in range(2))
    C.page_fork(*w, dst, src, 5, share, slots)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        status = C.page_fork(*d, dst, src, 5, share, slots)
    side = torch.cuda.Stream()
    for k in range(4):
        src.copy_(i32(*[(0, 1), (1, -1), (1, 0), (2, 2)][k]))
        torch.cuda.synchronize()
        if k == 2:
            with torch.cuda.stream(side):
                status.copy_(C.page_fork(*d, dst, src, 5, share, slots))
        else:
            gr.replay()
        torch.cuda.synchronize()
        want = C.page_fork(*e, dst, src, 5, share, slots_e)
        for a, b in zip(d + [slots, status], e + [slots_e, want]):
            assert torch.equal(a.view(torch.int16) if a.dtype == torch.bfloat16 else a, b.view(torch.int16) if b.dtype == torch.bfloat16 else b), k


@pytest.mark.parametrize("past", [40, 41, 99, 2 ** 31 - 1])
def test_fork_kept_sequence_with_entries_past_the_pool(C, dev, past):
    """dst == src: entries that are no page are given one like missing ones, and every slot lies inside the cache."""
    st = State(31, [20, 37, 5], P=40, held=2, W=8)
    st.table[0, 3], st.table[1, 4], st.table[2, 1], st.table[2, 2] = past, past, past, -9
    assert _fork(C, dev, st, [0, 1, 2], [0, 1, 2], 60) == [1, 1, 1]
    d = st.dev(dev)
    slots = torch.empty(3, 60, dtype=torch.int64, device=dev)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    C.page_fork(*d, i32([0, 1, 2]), i32([0, 1, 2]), 60, True, slots)
    assert (slots >= 0).all() and (slots < 40 * 16).all()
    assert int((d[4] > 0).sum()) == 2 + 3 + 1 + (5 - 2) + (7 - 3) + (5 - 1)


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("path", [None, [[0, 1, 2, 3]] * 5])
def test_commit_of_sequences_that_need_no_page_beside_starved_ones(C, dev, in_place, path):
    """Status 0 is for sequences whose own room is not all given: not for those behind them that have all their pages."""
    st = State(33, [14, 30, 0, 40, 8], P=10, held=4, W=6)
    assert int((st.refs == 0).sum()) == 0
    assert _commit(C, dev, st, [2, 2, 1, 3, 4], path, 4, in_place) == [1, 1, 1, 1, 1]
    st = State(34, [14, 30, 0, 40, 8], P=12, held=4, W=6)
    st.table[2, 1] = int((st.refs == 0).nonzero()[0])
    st.refs[st.table[2, 1].long()] = 1  # (the third sequence has its pages; one is free for the other four)
    assert _commit(C, dev, st, [2, 2, 1, 3, 4], path, 17, in_place) == [1, 0, 1, 0, 0]
    assert _commit(C, dev, st, [2, 0, 1, 3, -1], path, 17, in_place) == [1, 1, 1, 0, 1]


def test_fork_pairs_that_need_no_page_beside_starved_ones(C, dev):
    """Drops, shares of full pages and sequences that stay are done where pairs in front of them find too few pages."""
    st = State(35, [20, 32, 0, 0, 3], P=5, W=4)
    assert int((st.refs == 0).sum()) == 0
    assert _fork(C, dev, st, [2, 0, 3, 4, 1], [0, -1, 1, 4, 4], 0) == [0, 1, 1, 1, 0]
    assert _fork(C, dev, st, [2, 0, 3, 4, 1], [0, -1, 1, 4, -1], 0, False) == [0, 1, 0, 1, 1]
    lens = [20 + i % 29 for i in range(400)]
    st = State(36, lens, P=sum(-(-n // 16) for n in lens) + 40, W=3, L=1, Hk=1, D=8)  # (40 free pages for some 130 copies)
    pairs = [(200 + i, i if i % 3 else -1) for i in range(200)]
    done = _fork(C, dev, st, [d for d, _ in pairs], [s for _, s in pairs], 0)
    assert all(x == 1 for x, (_, s) in zip(done, pairs) if s < 0) and 0 in done


def test_the_most_pairs_and_sequences(C, dev):
    """1024 pairs of a fork, 1024 sequences of a commit with paths of 64 rows."""
    g = torch.Generator().manual_seed(9)
    lens = [int(x) for x in torch.randint(1, 60, (1024,), generator=g)]
    st = State(37, lens + [0] * 1024, P=9000, W=5, L=1, Hk=1, D=8)
    assert _fork(C, dev, st, list(range(1024, 2048)), list(range(1024)), 3) == [1] * 1024
    st = State(38, lens, P=9000, held=64, W=9, L=1, Hk=1)
    path = [list(range(i % 3, 64)) + [0] * (i % 3) for i in range(1024)]
    assert _commit(C, dev, st, [64 - i % 3 for i in range(1024)], path, 3) == [1] * 1024
