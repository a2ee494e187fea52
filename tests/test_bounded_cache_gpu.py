"""A server's steps over bounded caches: windowed attention, verification, commit, drawn weights and eviction, one behind the other
over two layers, every call against its oracle on the state that it found."""
import numpy as np
import pytest
import torch

from oracle import ref
from paged_cases import f64
from test_attn_mass_gpu import check as check_mass
from test_attn_window_gpu import check as check_window

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


class Server:
    L, Hk, H, D, T, W, P, B, R, V, window, sinks = 2, 2, 4, 64, 16, 12, 90, 3, 4, 700, 40, 3

    def __init__(self, dev, seed=0):
        s, g = self, torch.Generator().manual_seed(seed)
        lens = [60, 21, 5]
        s.dev, s.g = dev, g
        s.kv = torch.randn(s.L, 2, s.Hk, s.P, s.T, s.D, generator=g).to(BF).to(dev)
        s.ksum = torch.zeros(s.L, s.Hk, s.P, s.D, dtype=BF, device=dev)
        s.table = torch.full((s.B, s.W), -1, dtype=torch.int32)
        s.refs = torch.zeros(s.P, dtype=torch.int32)
        at = 0
        for b, n in enumerate(lens):
            e = -(-(n + s.R) // s.T)
            s.table[b, :e] = torch.arange(at, at + e)
            s.refs[at:at + e] = 1
            at += e
        s.table, s.refs = s.table.to(dev), s.refs.to(dev)
        s.length = torch.tensor(lens, dtype=torch.int32, device=dev)
        s.next = torch.empty_like(s.length)
        s.mass = torch.rand(s.L, s.B, s.Hk, s.W * s.T, generator=g).to(dev)

    def draw(self):
        """What the model would give: the step's rows (their K / V at the rows' places), queries, logits, the drafted tokens."""
        s, g = self, self.g
        q = (torch.randn(s.L, s.B, s.R, s.H, s.D, generator=g) * 1.5).to(BF).to(s.dev)
        rows = torch.randn(s.L, 2, s.Hk, s.B, s.R, s.D, generator=g).to(BF).to(s.dev)
        parent = (torch.rand(s.B, s.R, generator=g) * torch.arange(s.R)).to(torch.int32)
        mask = torch.zeros(s.B, s.R, dtype=torch.int64)
        for b in range(s.B):
            for r in range(s.R):
                mask[b, r] = (int(mask[b, parent[b, r]]) if r else 0) | (1 << r)
        logits = (torch.randn(s.B, s.R, s.V, generator=g) * 2).to(BF)
        best = logits.float().topk(s.R, -1).indices
        tokens = torch.zeros(s.B, s.R, dtype=torch.int64)
        for b in range(s.B):
            for r in range(1, s.R):
                tokens[b, r] = best[b, parent[b, r], r - 1]
        uniform = torch.rand(s.B, s.R + 1, generator=g, dtype=torch.float64)
        uniform[:, :s.R] *= 0.2
        return q, rows, mask.to(s.dev), logits.to(s.dev), tokens.to(s.dev), uniform.to(s.dev), parent.to(s.dev)

    def write(self, rows):
        pos = self.length[:, None].long() + torch.arange(self.R, device=self.dev)
        page = self.table.gather(1, pos // self.T).long()
        self.kv[:, :, :, page, pos % self.T] = rows

    def step(self, C, q, mask, logits, tokens, uniform, parent):
        """The calls of a step, into other lengths; returns what they give."""
        s = self
        out = [C.attn_window(q[l], s.kv[l, 0], s.kv[l, 1], s.table, s.length, s.window, s.sinks, mask=mask) for l in range(s.L)]
        count, path, token = C.verify_drafts(logits, tokens, uniform, parent=parent, temperature=0.8)
        ok = C.page_commit(s.kv, s.ksum, s.table, s.length, s.refs, count, path, s.R, s.next)
        for l in range(s.L):
            C.attn_mass(q[l], s.kv[l, 0], s.table, s.length, out[l][1], prior=s.mass[l], count=count, path=path, window=s.window, sinks=s.sinks, out=s.mass[l])
        return out, count, path, token, ok


def test_steps_against_the_oracles(C, dev):
    s = Server(dev)
    all_seqs = torch.arange(s.B, dtype=torch.int32, device=dev)
    evicted = 0
    for step in range(14):
        q, rows, mask, logits, tokens, uniform, parent = s.draw()
        s.write(rows)
        kv, table, lens, mass = s.kv.clone(), s.table.cpu(), s.length.tolist(), s.mass.clone()
        out, count, path, token, ok = s.step(C, q, mask, logits, tokens, uniform, parent)
        for l in range(s.L):
            check_window(out[l], BF, q[l].cpu(), kv[l, 0].cpu(), kv[l, 1].cpu(), table, lens, mask.cpu(), s.D ** -0.5, s.window, s.sinks)
        want = ref.verify_drafts(f64(logits), tokens.cpu().numpy(), uniform.cpu().numpy(), parent=parent.cpu().numpy(), heat=0.8)
        assert [x.tolist() for x in (count, path, token)] == [x.tolist() for x in want]
        assert ok.tolist() == [1] * s.B and s.next.tolist() == [n + c for n, c in zip(lens, count.tolist())]
        for l in range(s.L):
            check_mass(s.mass[l], mass[l], q[l].cpu(), s.kv[l, 0].cpu(), table, lens, out[l][1], mass[l], count.cpu(), path.cpu(), s.window, s.sinks, s.D ** -0.5)
        s.length, s.next = s.next, s.length
        if max(s.length.tolist()) > 80 or step == 6:
            host = [x.float().cpu().numpy() if x.is_floating_point() else x.cpu().numpy().astype(np.int64) for x in (s.kv, s.ksum, s.table, s.length, s.refs, s.mass)]
            status, kept = C.page_evict(s.kv, s.ksum, s.table, s.length, s.refs, s.mass, all_seqs, all_seqs, 20, s.sinks, 12, s.R)
            want = ref.page_evict(*host, range(s.B), range(s.B), 20, s.sinks, 12, s.R)
            for g, w in zip((s.kv, s.table, s.length, s.refs, s.mass, status, kept), (want[0], *want[2:6], *want[6:8])):
                assert np.array_equal(g.float().cpu().numpy(), np.asarray(w, dtype=np.float32))
            evicted += int((s.length <= 35).sum())
    assert evicted >= 3


def test_a_captured_step(C, dev):
    """The whole step as one graph, replayed over new inputs and beside an eager server on another stream: the same bits."""
    a, b = Server(dev, 1), Server(dev, 1)
    inputs = list(a.draw())
    b.draw()
    hold = [t.clone() for t in inputs]
    w = Server(dev, 1)
    w.step(C, *(t for i, t in enumerate(hold) if i != 1))
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        got = a.step(C, *(t for i, t in enumerate(hold) if i != 1))
    for _ in range(4):
        inputs = a.draw()
        for h, t in zip(hold, inputs):
            h.copy_(t)
        a.write(inputs[1])
        b.write(inputs[1])
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            want = b.step(C, *(t for i, t in enumerate(inputs) if i != 1))
        torch.cuda.synchronize()
        for x, y in zip((*got[0][0], *got[0][1], *got[1:], a.kv, a.table, a.next, a.mass), (*want[0][0], *want[0][1], *want[1:], b.kv, b.table, b.next, b.mass)):
            assert torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8))
        for s in (a, b):
            s.length.copy_(s.next)
