"""The oracles of windows, drawn weights and eviction by hand, and the entry points' refusals before any device work (no GPU)."""
import os

import numpy as np
import pytest

from conftest import PKG
from oracle import ref
from paged_cases import rows_meet, views


def test_kept_tokens_by_hand():
    mass = np.array([9.0, 1.0, 5.0, 5.0, np.nan, 0.0, 5.0, 2.0, 1.0])
    assert ref.kept_tokens(mass, 9, 2, 0, 0) == [0, 2]
    assert ref.kept_tokens(mass, 9, 2, 1, 1) == [0, 2, 3, 8]
    assert ref.kept_tokens(mass, 9, 6, 1, 1) == [0, 1, 2, 3, 5, 6, 7, 8]
    assert ref.kept_tokens(mass, 5, 5, 0, 0) == [0, 1, 2, 3, 4]


def test_window_by_hand():
    keep = ref.window_keep(None, [4], 3, 2, 1)
    pos = np.arange(7)
    assert [np.flatnonzero(keep(0, s, 0, pos) & (pos <= 4 + s)).tolist() for s in range(3)] == [[0, 3, 4], [0, 4, 5], [0, 5, 6]]
    keep = ref.window_keep(np.array([[0b1, 0b11, 0b101]]), [1], 3, 2, 2)  # first tokens that reach among the own ones
    assert [np.flatnonzero(keep(0, s, 0, pos)).tolist() for s in range(3)] == [[0, 1], [0, 1, 2], [0, 1, 3]]


def test_weights_sum_to_the_rows():
    rng = np.random.default_rng(2)
    table = np.array([[2, 0, 1]])
    key, q = rng.standard_normal((2, 3, 16, 8)), rng.standard_normal((1, 5, 4, 8))
    keep = ref.window_keep(None, [30], 5, 9, 2)
    lse = ref.paged_lse(q, key, table, [30], None, 0.4, keep)
    out, _, written = ref.attention_mass(q, key, table, [30], lse, None, None, None, 9, 2, 0.4, 48)
    assert np.allclose(out.sum(2), 10) and written.sum() == 35 and (out[:, :, 35:] == 0).all()
    out, _, _ = ref.attention_mass(q, key, table, [30], lse, np.ones((1, 2, 48)), np.array([2]), np.array([[3, 4, 0, 0, 0]]), 1 << 30, 0, 0.4, 48)
    assert out[0, 0, 32] == 0 and (out[0, :, :30] > 1).all()


def test_refusals_before_any_device_work():
    if not os.path.exists(os.path.join(PKG, "mdx", "libmdx.so")):
        pytest.skip("libmdx.so not built")
    from mdx import _lib
    L, p = _lib.lib(), 4096  # (never read: the checks come first)
    need = L.mdx_page_evict_workspace(2, 8, 2, 2, 10)
    assert need > 0 and need % 16 == 0 and L.mdx_page_evict_workspace(1025, 8, 2, 2, 10) == 0 and L.mdx_page_evict_workspace(2, 8, 2, 2, 0) == 0

    def evict(**k):
        a = dict(kv=p, ksum=p, dt=_lib.DT_BF16, L=2, Hk=2, P=20, T=16, D=64, table=p, ts=8, B=3, W=8, length=p, refs=p, mass=p, N=128, dst=p, src=p, pairs=2,
                 keep=10, sinks=0, recent=0, room=0, slots=None, status=p, kept=p, ws=p, n=need)
        a.update(k)
        return L.mdx_page_evict(*a.values(), None), L.mdx_last_error().decode()

    for k in (dict(kv=None), dict(kept=None), dict(mass=None), dict(dt=_lib.DT_F32), dict(T=24), dict(D=96), dict(L=0), dict(P=1 << 28), dict(W=0), dict(ts=7),
              dict(N=127), dict(pairs=0), dict(pairs=1025), dict(room=-1), dict(keep=-1), dict(keep=0), dict(keep=1 << 30), dict(kv=p + 8), dict(ws=None),
              dict(n=need - 1), dict(keep=1 << 29), dict(B=0)):
        rc, msg = evict(**k)
        assert rc == _lib.MDX_EINVAL and msg, k

    def mass(**k):
        a = dict(q=p, qb=128, qs=128, qh=64, key=p, kh=1024, kp=1024, kt=64, dt=_lib.DT_F16, table=p, ts=8, length=p, lse=p, prior=None, pb=0, ph=0, count=None,
                 path=None, window=4, sinks=0, out=p, ob=256, oh=128, N=128, B=2, S=3, H=4, Hk=2, D=64, P=20, T=16, W=8, scale=0.1, ws=None, n=0)
        a.update(k)
        return L.mdx_attn_mass(*a.values(), None), L.mdx_last_error().decode()

    for k in (dict(q=None), dict(lse=None), dict(dt=_lib.DT_F32), dict(D=32), dict(T=8), dict(S=0), dict(S=65536), dict(H=3), dict(H=258), dict(kt=60), dict(qs=4),
              dict(key=p + 8), dict(N=0), dict(oh=100), dict(ob=200), dict(prior=p, pb=-1), dict(window=0), dict(sinks=-1), dict(scale=0.0), dict(W=1 << 27),
              dict(out=p + 2), dict(S=2000, N=1024, oh=1024, ob=2048, W=64, ts=64)):
        rc, msg = mass(**k)
        assert rc == _lib.MDX_EINVAL and msg, k

    def window(**k):
        a = dict(q=p, qb=768, qs=256, qh=64, key=p, kh=1024, kp=1024, kt=64, value=p, vh=1024, vp=1024, vt=64, dt=_lib.DT_BF16, table=p, ts=8, length=p, mask=None,
                 out=1 << 20, lse=p, window=4, sinks=0, B=2, S=3, H=4, Hk=2, D=64, P=20, T=16, W=8, scale=0.1, ws=None, n=0)
        a.update(k)
        return L.mdx_attn_window(*a.values(), None), L.mdx_last_error().decode()

    for k in (dict(lse=None), dict(window=0), dict(window=(1 << 30) + 1), dict(sinks=-1), dict(sinks=(1 << 30) + 1), dict(S=65, mask=p), dict(q=None), dict(out=p),
              dict(W=4000, ts=4000, window=60000), dict(scale=float("nan"))):
        rc, msg = window(**k)
        assert rc == _lib.MDX_EINVAL and msg, k
    assert L.mdx_attn_window_workspace(2, 3, 4, 2, 64, 16, 8, 4, 0) == 0 < L.mdx_attn_window_workspace(2, 3, 4, 2, 64, 16, 4000, 60000, 0)
    assert L.mdx_attn_window_workspace(2, 3, 4, 2, 64, 16, 4000, 300, 4) == 0


def test_log_sum_exps_over_the_outputs_or_queries_are_refused():
    """Rows are written while others' queries are read: 12 rows of 64 elements of 2 bytes, 12 log-sum-exps of 4."""
    if not os.path.exists(os.path.join(PKG, "mdx", "libmdx.so")):
        pytest.skip("libmdx.so not built")
    from mdx import _lib
    L, q, out = _lib.lib(), 1 << 20, 1 << 21  # (never read: the checks come first)

    def window(lse, qs=256):
        rc = L.mdx_attn_window(q, 3 * qs, qs, 64, 1 << 24, 1024, 1024, 64, 1 << 25, 1024, 1024, 64, _lib.DT_BF16, 1 << 26, 8, 1 << 26, None, out, lse, 4, 0, 2, 3, 4,
                               2, 64, 20, 16, 8, 0.1, None, 0, None)
        return rc, L.mdx_last_error().decode()

    rows, sums = 2 * 3 * 4 * 64 * 2, 2 * 3 * 4 * 4
    for lse in (out, out + 4, out + rows - 4, out - sums + 4, q, q + rows - 4, q - sums + 4):
        rc, msg = window(lse)
        assert rc == _lib.MDX_EINVAL and "apart" in msg, lse
    rc, msg = window(q + 2 * rows - 4, 512 + 64)  # (rows further apart)
    assert rc == _lib.MDX_EINVAL and "apart" in msg


def test_sums_over_what_is_read_are_refused():
    """prior and out of [3, 2, 100] places in one buffer: views that meet without being one; out over q or lse."""
    if not os.path.exists(os.path.join(PKG, "mdx", "libmdx.so")):
        pytest.skip("libmdx.so not built")
    from mdx import _lib
    L, q, lse, base = _lib.lib(), 1 << 20, 1 << 21, 1 << 28  # (never read: the checks come first)

    def mass(prior, pb, ph, out, ob, oh, B=3, Hk=2, N=100):
        rc = L.mdx_attn_mass(q, 768, 256, 64, 1 << 24, 1024, 1024, 64, _lib.DT_BF16, 1 << 26, 8, 1 << 26, lse, prior, pb, ph, None, None, 4, 0, out, ob, oh, N, B,
                             3, 4, Hk, 64, 20, 16, 8, 0.1, None, 0, None)
        return rc, L.mdx_last_error().decode()

    tried = 0
    for B, Hk in ((3, 2), (1, 2), (3, 1)):
        for ob, oh, pb, ph, d in views():
            if rows_meet(B, Hk, 100, d, pb, ph, ob, oh):
                rc, msg = mass(base + 4 * d, pb, ph, base, ob, oh, B, Hk)
                assert rc == _lib.MDX_EINVAL and "apart" in msg, (B, Hk, ob, oh, pb, ph, d)
                tried += 1
    assert tried > 300
    for out in (lse, lse + 140, q, q + 4, lse - 2396):
        rc, msg = mass(None, 0, 0, out, 200, 100)
        assert rc == _lib.MDX_EINVAL and "apart" in msg, out
