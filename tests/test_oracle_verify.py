"""The verification's oracle against what it has to give, and the entry point's refusals before any device work (no GPU)."""
import os

import numpy as np
import pytest
import torch

from conftest import PKG
from oracle import ref


def test_answers_are_distributed_as_the_target():
    """One drafted token of q over five tokens, both uniforms over an even grid: the committed token (the draft's where it is
    accepted, the answer where not) has p's distribution, to within the grid's steps."""
    rng = np.random.default_rng(1)
    p_logits, q_logits = rng.standard_normal((2, 5)) * 1.5
    p, q = ref.token_probabilities(p_logits, 1.0), ref.token_probabilities(q_logits, 1.0)
    n, got = 200, np.zeros(5)
    logits, draft = np.stack([p_logits, p_logits])[None], q_logits[None, None]
    grid = (np.arange(n) + 0.5) / n
    for x in range(5):
        accepted = int((grid * q[x] < p[x]).sum())
        got[x] += q[x] * accepted / n
        if accepted == n:
            continue
        for u in grid:
            count, _, answer = ref.verify_drafts(logits, [[0, x]], np.array([[1 - 1e-9, 0.0, u]]), draft)
            assert count[0] == 1
            got[answer[0]] += q[x] * (1 - accepted / n) / n
    assert np.abs(got - p).max() < 5 * 2 / n


def test_children_split_the_unit_interval():
    """Without draft probabilities: the children's parts of [0, 1) in row order, and the rest without them."""
    logits = np.log(np.array([[[0.1, 0.2, 0.3, 0.4]] * 4]))
    tokens, parent = [[9, 2, 1, 2]], [[0, 0, 0, 0]]
    for u, want in ((0.29, [0, 1]), (0.31, [0, 2]), (0.49, [0, 2]), (0.51, [0])):
        count, path, answer = ref.verify_drafts(logits, tokens, np.array([[u, 0, 0, 0, 0.5]]), parent=parent)
        assert path[0, :count[0]].tolist() == want and count[0] == len(want)
        assert answer[0] == (2 if len(want) > 1 else 3)  # of 0.1, 0.4 half is passed in token 3; of all, in token 2
    assert ref.verify_drafts(logits, tokens, np.array([[0.6, 0, 0, 0, 0.1]]), parent=parent)[2][0] == 0


def test_nothing_left_and_nothing_there():
    none, one = np.full((1, 2, 3), -np.inf), np.array([[[0.0, -np.inf, 1.0]] * 2])
    u = np.array([[0.5, 0.5, 0.2]])
    assert ref.verify_drafts(none, [[0, 1]], u)[2][0] == -1
    # token 1 has no probability in p and q alike: refused, p - q is empty, p answers
    count, _, answer = ref.verify_drafts(one, [[0, 1]], u, one[:, :1])
    assert count[0] == 1 and answer[0] == 0
    assert ref.draw_token(np.array([0.0, 1.0, 0.0]), 1.0) == 1


def test_refusals_before_any_device_work():
    lib = os.path.join(PKG, "mdx", "libmdx.so")
    if not os.path.exists(lib):
        pytest.skip("libmdx.so not built")
    from mdx import _C, _lib
    L = _lib.lib()
    need = L.mdx_verify_drafts_workspace(2, 4, 1000, 1)
    assert need > 0 and need % 16 == 0
    assert L.mdx_verify_drafts_workspace(2, 65, 1000, 1) == 0 and L.mdx_verify_drafts_workspace(2, 4, 1 << 24, 0) == 0
    p = 4096  # (never read: the checks come first)

    def call(**k):
        a = dict(logits=p, lb=4000, lr=1000, draft=p, db=3000, dr=1000, dt=_lib.DT_BF16, tokens=p, parent=None, uniform=p, heats=None, heat=1.0,
                 count=p, path=p, next=p, B=2, R=4, V=1000, ws=p, n=need)
        a.update(k)
        rc = L.mdx_verify_drafts(a["logits"], a["lb"], a["lr"], a["draft"], a["db"], a["dr"], a["dt"], a["tokens"], a["parent"], a["uniform"], a["heats"],
                                 a["heat"], a["count"], a["path"], a["next"], a["B"], a["R"], a["V"], a["ws"], a["n"], None)
        return rc, L.mdx_last_error().decode()

    for k in (dict(logits=None), dict(tokens=None), dict(uniform=None), dict(next=None), dict(dt=_lib.DT_FP8E4M3), dict(B=0), dict(B=1025), dict(R=65),
              dict(R=0), dict(V=0), dict(V=1 << 24), dict(parent=p), dict(lb=-1), dict(dr=-1), dict(heat=-1.0), dict(heat=float("nan")),
              dict(heat=float("inf")), dict(ws=None), dict(ws=p + 8), dict(n=need - 1)):
        rc, msg = call(**k)
        assert rc == _lib.MDX_EINVAL and msg, k
    with pytest.raises(RuntimeError, match="ROCm device"):
        _C.verify_drafts(torch.zeros(1, 2, 8), torch.zeros(1, 2, dtype=torch.int64), torch.zeros(1, 3, dtype=torch.float64))
    with pytest.raises(RuntimeError, match="logits"):
        _C.verify_drafts(None, None, None)


def test_more_rows_times_logits_than_a_launch_holds():
    """Rows of one broadcast buffer: the launch would have 2^32 threads or more. Refused before any device work."""
    lib = os.path.join(PKG, "mdx", "libmdx.so")
    if not os.path.exists(lib):
        pytest.skip("libmdx.so not built")
    from mdx import _lib
    L, p = _lib.lib(), 4096  # (never read)
    most = 255 * 16384  # logits of a row: 255 work-groups of 16384
    for R, draft, V in ((64, None, most + 16384 - 6), (64, None, (1 << 24) - 1), (33, p, most + 16384), (64, p, most)):
        assert L.mdx_verify_drafts_workspace(1024, R, V, draft is not None) == 0, (R, V)
        rc = L.mdx_verify_drafts(p, 0, 0, draft, 0, 0, _lib.DT_BF16, p, None, p, None, 1.0, p, p, p, 1024, R, V, p, 1 << 50, None)
        assert rc == _lib.MDX_EINVAL and "too many" in L.mdx_last_error().decode(), (R, V)
    assert L.mdx_verify_drafts_workspace(1024, 64, most - 7, 0) > 0 and L.mdx_verify_drafts_workspace(1024, 32, most - 7, 1) > 0
