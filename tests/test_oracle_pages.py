"""The paged cache's oracle (oracle/ref.py) against closed forms and against the one-sequence oracle, and the refusals of the
entry points before any device work (no GPU needed)."""
import os

import numpy as np
import pytest
import torch

from conftest import PKG
from oracle import ref


def _scattered(rng, lens, T, own, spare=2):
    each = [-(-(n + own) // T) for n in lens]
    order = rng.permutation(sum(each) + spare)
    table = np.full((len(lens), max(each) + 1), -1, dtype=np.int64)
    at = 0
    for i, n in enumerate(each):
        table[i, :n] = order[at:at + n]
        at += n
    return table, len(order)


@pytest.mark.parametrize("parents", [[-1, 0, 0, 1], [-1, 0, 1, 2]])
def test_paged_attention_is_the_contiguous_one(parents):
    """Pages in any order, read back as one sequence each: the tree-verify oracle's values."""
    rng = np.random.default_rng(3)
    lens, T, H, Hk, D, S = [37, 0, 16], 16, 4, 2, 8, len(parents)
    table, P = _scattered(rng, lens, T, S)
    key, value = rng.standard_normal((2, Hk, P, T, D))
    q = rng.standard_normal((3, S, H, D))
    mask = np.array([ref.tree_mask(parents)] * 3)
    out, spread, mass, heft = ref.paged_attention(q, key, value, table, lens, mask, D ** -0.5)
    for b, n in enumerate(lens):
        pos = np.arange(n + S)
        k, v = (x[:, table[b, pos // T], pos % T] for x in (key, value))
        want = ref.attention_f64(q[b].swapaxes(0, 1), k[:, :n + 1], v[:, :n + 1], n, k[:, n:], v[:, n:], ref.tree_mask(parents))
        assert np.abs(out[b] - want).max() < 1e-12
    assert (spread <= 2 * mass + 1e-12).all() and (heft > 0).all()


def test_paged_attention_chain_and_missing_pages():
    """Without masks row s attends j <= s; a sequence without pages gives 0; equal values come out unchanged."""
    rng = np.random.default_rng(4)
    table, P = _scattered(rng, [20, 5], 16, 2)
    table[1] = -1
    key = rng.standard_normal((1, P, 16, 8))
    value = np.full_like(key, 3.0)
    q = rng.standard_normal((2, 2, 3, 8))
    out, spread, _, _ = ref.paged_attention(q, key, value, table, [20, 5], None, 0.3)
    assert np.abs(out[0] - 3).max() < 1e-12 and (out[1] == 0).all() and spread.max() < 1e-12


def test_block_selection_by_hand():
    """One head, D = 1: scores are the mean keys themselves; ties go to the lowest page, NaN last, few pages are all taken."""
    ksum = np.array([[[0.], [5.], [2.], [5.], [float("nan")], [1.], [9.]]])
    q = np.ones((1, 1, 1, 1))
    table = np.arange(7)[None]
    pick = lambda n, blocks, sink, local: ref.block_selection(q, ksum, table, [n], 16, blocks, sink, local)[0, 0, 0].tolist()  # noqa: E731
    assert pick(7 * 16, 1, 1, 1) == [0, 1, 6]
    assert pick(7 * 16, 2, 1, 1) == [0, 1, 3, 6]
    assert pick(7 * 16 + 5, 5, 0, 1) == [0, 1, 2, 3, 5, 6]
    assert pick(2 * 16 + 15, 2, 1, 1) == [0, 1, -1, -1]
    assert pick(7 * 16, 0, 2, 1) == [0, 1, 6]


def test_fork_and_commit_by_hand():
    kv = np.arange(6, dtype=np.float64).reshape(1, 1, 1, 6, 1, 1) * 100 + np.arange(16).reshape(1, 1, 1, 1, 16, 1)
    kv = np.concatenate([kv, -kv], 1)
    ksum = np.zeros((1, 1, 6, 1))
    table = np.array([[4, 2, -1], [-1, -1, -1]])
    length, refs = np.array([20, 0]), np.array([0, 0, 1, 0, 1, 0])
    kv2, _, t2, n2, r2, st, sl = ref.page_fork(kv, ksum, table, length, refs, [1], [0], 14, True)
    assert t2.tolist() == [[4, 2, -1], [4, 0, 1]] and n2.tolist() == [20, 20] and r2.tolist() == [1, 1, 1, 0, 2, 0]
    assert st.tolist() == [1] and sl[0].tolist() == [4 + i for i in range(12)] + [16, 17]
    assert (kv2[:, :, :, 0] == kv[:, :, :, 2]).all() and (kv2[:, :, :, 1:] == kv[:, :, :, 1:]).all()
    kv3, t3, n3, r3, st, sl, filled = ref.page_commit(kv2, t2, n2, r2, [-1, 3], np.array([[0, 0, 0, 0], [0, 2, 3, 9]]), 11)
    assert n3.tolist() == [20, 23] and st.tolist() == [1, 1] and filled == [] and (t3 == t2).all()
    assert kv3[0, 0, 0, 0, 4:8, 0].tolist() == [204, 206, 207, 207] and sl[1].tolist() == [7 + i for i in range(9)] + [16, 17]
    *_, n4, _, st, _, filled = ref.page_commit(kv2, t2, n2, r2, [0, 12], None, 0)
    assert n4.tolist() == [20, 32] and [e for e, _ in filled] == [0] and filled[0][1][0, 0, 0] == 207.5
    *_, n5, _, st, _, _ = ref.page_commit(kv2, t2, n2, r2, [1, 2], np.array([[1, 0], [1, 1]]), 0)
    assert st.tolist() == [1, -1] and n5.tolist() == [21, 20]


def test_a_kept_sequence_gets_pages_for_entries_that_are_none():
    """dst == src: an entry past the pool is no page, as one below 0 is none: both are given a page, and the slots lie in the cache."""
    kv, ksum = np.zeros((1, 2, 1, 6, 16, 1)), np.zeros((1, 1, 6, 1))
    table = np.array([[4, 9, -3, 2 ** 31 - 1]])
    *_, t2, n2, r2, st, sl = ref.page_fork(kv, ksum, table, np.array([16]), np.array([0, 1, 0, 0, 1, 0]), [0], [0], 20, True)
    assert st.tolist() == [1] and t2.tolist() == [[4, 0, 2, 2 ** 31 - 1]] and r2.tolist() == [1, 1, 1, 0, 1, 0]
    assert sl[0].tolist() == list(range(16)) + [32, 33, 34, 35]


def test_a_commit_that_needs_no_page_is_done_whatever_the_others_need():
    """One free page; 17 more tokens take the first sequence two, the second none, the third one: only the second has all its room."""
    kv = np.zeros((1, 2, 1, 6, 16, 1))
    table = np.array([[0, -1, -1, -1], [1, 2, 4, -1], [3, -1, -1, -1]])
    refs = np.array([1, 1, 1, 1, 1, 0])
    _, t2, n2, _, st, sl, _ = ref.page_commit(kv, table, np.array([10, 16, 14]), refs, [6, 2, 1], None, 17)
    assert st.tolist() == [0, 1, 0] and n2.tolist() == [16, 18, 15] and (t2 == table).all() and (sl[1] >= 0).all()
    _, t2, _, _, st, _, _ = ref.page_commit(kv, table, np.array([10, 16, 14]), refs, [-1, 2, 1], None, 17)
    assert st.tolist() == [1, 1, 1] and t2[2].tolist() == [3, 5, -1, -1]


def test_a_drop_behind_a_starved_pair_is_done():
    """A pair that needs no page (a drop, a share without a tail, a sequence that has its room) is done where others find too few;
    the pages it gives back serve the next call."""
    kv, ksum = np.zeros((1, 2, 1, 5, 16, 1)), np.zeros((1, 1, 5, 1))
    table = np.array([[0, 1], [2, 3], [-1, -1], [-1, -1], [4, -1]])
    length, refs = np.array([20, 32, 0, 0, 3]), np.ones(5, dtype=np.int64)
    _, _, t2, n2, r2, st, _ = ref.page_fork(kv, ksum, table, length, refs, [2, 0, 3, 4, 1], [0, -1, 1, 4, 4], 0, True)
    assert st.tolist() == [0, 1, 1, 1, 0] and n2.tolist() == [0, 32, 0, 32, 3]
    assert t2.tolist() == [[-1, -1], [2, 3], [-1, -1], [2, 3], [4, -1]] and r2.tolist() == [0, 0, 2, 2, 1]


# ---- refusals --------------------------------------------------------------------------------------
@pytest.mark.skipif(not os.path.exists(os.path.join(PKG, "mdx", "libmdx.so")), reason="libmdx.so not built")
def test_refusals_before_any_device_work():
    """Every contract violation is an error from the checks (the addresses are never used)."""
    from mdx import _lib
    A = 1 << 12  # an aligned address that nothing reads

    def attn(q=A, key=A, value=A, dt=_lib.DT_BF16, table=A, length=A, mask=None, out=1 << 44, B=1, S=1, H=4, Hk=2, D=128, P=8, T=16, W=400,
             scale=0.1, ws=A, nb=1 << 40, kt=128, kp=2048, qs=512, ts=400):
        return _lib.lib().mdx_attn_paged(q, 512, qs, 128, key, kp * 8, kp, kt, value, kp * 8, kp, kt, dt, table, ts, length, mask,
                                         out, B, S, H, Hk, D, P, T, W, scale, ws, nb, None)

    def blocks(blocks=4, sink=1, local=1, ksum=A, sel=A, out=1 << 44, S=1, H=4, sp=128, nb=1 << 40):
        return _lib.lib().mdx_attn_blocks(A, 512, 512, 128, A, 16384, 2048, 128, A, 16384, 2048, 128, ksum, 1024, sp, _lib.DT_BF16,
                                          A, 4, A, None, out, sel, blocks, sink, local, 1, S, H, 2, 128, 8, 16, 4, 0.1, A, nb, None)

    def fork(kv=A, ksum=A, L=2, Hk=2, P=8, T=16, D=128, table=A, ts=4, B=4, W=4, pairs=2, room=1, ws=A, nb=1 << 20, refs=A):
        return _lib.lib().mdx_page_fork(kv, ksum, L, Hk, P, T, D, table, ts, B, W, A, refs, A, A, pairs, room, 1, None, A, ws, nb, None)

    def commit(kv=A, dt=_lib.DT_BF16, T=16, D=128, B=4, W=4, ts=4, path=A, R=8, room=1, count=A, nb=1 << 20, new=A):
        return _lib.lib().mdx_page_commit(kv, A, dt, 2, 2, 8, T, D, A, ts, B, W, A, new, A, count, path, R, room, None, A, A, nb, None)

    bad = [(attn, dict(q=None)), (attn, dict(length=None)), (attn, dict(dt=_lib.DT_F32)), (attn, dict(D=192)), (attn, dict(T=24)),
           (attn, dict(T=8)), (attn, dict(T=2048)), (attn, dict(H=5)), (attn, dict(H=258)), (attn, dict(B=0)), (attn, dict(B=1025)), (attn, dict(S=0)),
           (attn, dict(S=65, mask=A)), (attn, dict(S=65536)), (attn, dict(W=0)), (attn, dict(ts=3)), (attn, dict(W=1 << 28)),
           (attn, dict(scale=0.0)), (attn, dict(scale=float("inf"))), (attn, dict(scale=float("nan"))), (attn, dict(q=A + 8)),
           (attn, dict(kt=64)), (attn, dict(kt=132)), (attn, dict(kp=-2048)), (attn, dict(qs=516)), (attn, dict(ws=None)),
           (attn, dict(nb=64)), (attn, dict(S=65535, W=1 << 20, ts=1 << 20, B=1024)),
           (blocks, dict(blocks=0, sink=0, local=0)), (blocks, dict(blocks=-1)), (blocks, dict(ksum=None)), (blocks, dict(sel=None)),
           (blocks, dict(S=65)), (blocks, dict(H=2 * 65)), (blocks, dict(sp=64)), (blocks, dict(nb=64)), (blocks, dict(blocks=65536)),
           (fork, dict(kv=None)), (fork, dict(refs=None)), (fork, dict(T=20)), (fork, dict(D=12)), (fork, dict(pairs=0)),
           (fork, dict(pairs=1025)), (fork, dict(room=-1)), (fork, dict(ts=3)), (fork, dict(kv=A + 4)), (fork, dict(nb=16)),
           (fork, dict(ws=None)), (fork, dict(P=0)),
           (commit, dict(kv=None)), (commit, dict(count=None)), (commit, dict(dt=_lib.DT_F32)), (commit, dict(T=17)), (commit, dict(D=96)),
           (commit, dict(B=1025)), (commit, dict(R=0)), (commit, dict(R=65)), (commit, dict(room=-1)), (commit, dict(nb=16)),
           (commit, dict(ts=2)),
           (attn, dict(out=A)), (attn, dict(out=A + 1008)), (blocks, dict(out=A)), (attn, dict(qs=-512)),
           (fork, dict(pairs=1024, W=1 << 20, ts=1 << 20, nb=1 << 40)), (commit, dict(B=1024, W=1 << 20, ts=1 << 20, nb=1 << 40)),
           (commit, dict(new=A + 4)), (commit, dict(new=A - 12))]
    for f, kw in bad:
        assert f(**kw) == _lib.MDX_EINVAL, (f.__name__, kw)
        assert _lib.lib().mdx_last_error(), (f.__name__, kw)


@pytest.mark.skipif(not os.path.exists(os.path.join(PKG, "mdx", "libmdx.so")), reason="libmdx.so not built")
def test_a_line_of_steps_that_nearly_fills_32_bits_is_refused():
    """64 units of 2^30 - 288 tokens are 2^31 - 192 steps of 32 with their fixed cost; of 256 shares the last begins at 255 * 2^23 and
    its end, 2^31, is no 32-bit number."""
    from mdx import _lib
    A, tokens = 1 << 12, (1 << 30) - 288
    steps = 64 * (-(-(tokens + 1) // 32) + 5)
    share = -(-steps // 256)
    assert steps == (1 << 31) - 192 and 256 * share >= 1 << 31
    rc = _lib.lib().mdx_attn_paged(A, 80 * 256, 80 * 256, 256, A, 1 << 20, 4096, 256, A, 1 << 20, 4096, 256, _lib.DT_BF16, A, tokens // 16, A, None,
                                   1 << 44, 64, 1, 80, 1, 256, 8, 16, tokens // 16, 0.1, A, 1 << 40, None)
    assert rc == _lib.MDX_EINVAL and b"too many" in _lib.lib().mdx_last_error()


def test_host_tensors_are_refused():
    from mdx import _C
    z = torch.zeros
    kv, ks = z(1, 2, 2, 4, 16, 64, dtype=torch.bfloat16), z(1, 2, 4, 64, dtype=torch.bfloat16)
    i = lambda *s: z(*s, dtype=torch.int32)  # noqa: E731
    for call in (lambda: _C.page_fork(kv, ks, i(2, 4), i(2), i(4), i(1), i(1)), lambda: _C.page_commit(kv, ks, i(2, 4), i(2), i(4), i(2)),
                 lambda: _C.attn_paged(z(2, 1, 4, 64, dtype=torch.bfloat16), kv[0, 0], kv[0, 1], i(2, 4), i(2)),
                 lambda: _C.attn_blocks(z(2, 1, 4, 64, dtype=torch.bfloat16), kv[0, 0], kv[0, 1], ks[0], i(2, 4), i(2), 1)):
        with pytest.raises(RuntimeError, match="ROCm device"):
            call()


def test_a_missing_binding_is_an_error(monkeypatch):
    import sys

    import mdx
    from mdx import _lib
    monkeypatch.setitem(sys.modules, "mdx._bind", None)
    monkeypatch.delattr(mdx, "_bind", raising=False)
    monkeypatch.setattr(_lib, "_bound", None)
    with pytest.raises(_lib.MdxError, match="build.py"):
        _lib.bind()
