"""Verification of trees of drafted tokens on the GPU against the definition, step by step in float64: every refusal
takes max(r - q', 0) and normalises, with whole laws. Results are whole numbers. A decision may differ only where the
definition's two sides lie within 1e-9 of each other, which the inputs are checked not to do."""
import numpy as np
import pytest
import torch

import ctox_hip as ch
from tree_model import NO, flat, random_tree, starts
from test_gpu_tree_ops import dev, host, stream

pytestmark = pytest.mark.gpu

FAILED = 0xfffffffe
EDGE = 1e-9


def say(*a):
    print(*a, flush=True)


def softmax(x, T):
    x = x.astype(np.float64) / T
    e = np.exp(x - x.max())
    return e / e.sum()


class Verify:
    def __init__(self, seed, nodes, vocab, width=4, T=1.0, drawn="without", draft_vocab=None, std=3.0, noise=0.9, chain=0.0,
                 skew=0, forest=None, sharp=1.0):
        rng = self.rng = np.random.default_rng(seed)
        self.nodes, self.V, self.width, self.T, self.drawn = nodes, vocab, width, T, drawn
        self.forest = forest or [random_tree(rng, n, width, chain) for n in nodes]
        self.starts = starts(nodes)
        M = self.M = int(self.starts[-1])
        DV = self.DV = draft_vocab or vocab
        self.ids = np.arange(vocab) if DV == vocab else np.sort(rng.permutation(vocab)[:DV])
        self.target = (rng.standard_normal((M, vocab)) * std).astype(np.float32)
        self.draft = (self.target[:, self.ids] * sharp + noise * rng.standard_normal((M, DV))).astype(np.float32)
        self.inverse = np.full(vocab, NO, np.uint32)
        self.inverse[self.ids] = np.arange(DV)
        self.tokens = rng.integers(0, vocab, max(M, 1)).astype(np.uint32)
        for r, parent in enumerate(self.forest):
            for u in range(len(parent)):
                kids = [i for i, p in enumerate(parent) if p == u]
                if not kids:
                    continue
                row = self.starts[r] + u
                q = softmax(self.draft[row], T or 1.0)
                if drawn == "point" or T == 0:
                    pick = np.argsort(-q)[:len(kids)]
                else:
                    n = len(kids)
                    pick = rng.choice(DV, n, p=q) if drawn == "with" else rng.choice(DV, n, replace=False, p=q)
                self.tokens[[self.starts[r] + k for k in kids]] = self.ids[pick]
        self.u = rng.random(max(M, 1)).astype(np.float32)
        self.s = rng.random(len(nodes)).astype(np.float32)
        self.skew = skew  # values between rows and in front of the first

    def law(self, row):
        p = softmax(self.target[row], self.T)
        q = np.zeros(self.V)
        q[self.ids] = softmax(self.draft[row], self.T)
        return p, q

    def expect(self, width=None):
        width, out = width or self.width, []
        for r, parent in enumerate(self.forest):
            if not parent:
                out.append(([], NO))
                continue
            path, node = [0], 0
            while True:
                row = self.starts[r] + node
                kids = [i for i, p in enumerate(parent) if p == node][:width]
                took = None
                if self.T == 0:
                    best = int(np.flatnonzero(self.target[row] == self.target[row].max())[-1])
                    took = next((k for k in kids if self.tokens[self.starts[r] + k] == best), None)
                else:
                    rest, q = self.law(row)
                    gone = []
                    for k in kids:
                        token, u = int(self.tokens[self.starts[r] + k]), float(self.u[self.starts[r] + k])
                        if self.drawn == "point":
                            qq = np.zeros(self.V)
                            qq[token] = 1.0
                        else:
                            qq = q.copy()
                            if self.drawn == "without":
                                qq[gone] = 0.0
                                if qq.sum() < 2.0 ** -40:
                                    break
                                qq /= qq.sum()
                        assert abs(u * qq[token] - rest[token]) > EDGE * (rest[token] + qq[token]), "a decision on its edge"
                        if u * qq[token] < rest[token]:
                            took = k
                            break
                        gone.append(token)
                        if self.drawn == "point":
                            rest[token] = 0.0
                        else:
                            rest = np.maximum(rest - qq, 0.0)
                        rest /= rest.sum()
                if took is None:
                    break
                node = took
                path.append(node)
            if self.T == 0:
                out.append((path, best))
                continue
            run = np.cumsum(rest)
            goal = float(self.s[r]) * run[-1]
            token = int(np.searchsorted(run, goal, side="right"))
            near = run[max(0, token - 1):token + 1]
            assert np.abs(near - goal).min() > EDGE * run[-1], "a draw on its edge"
            out.append((path, token))
        return out

    def op(self, hip, max_children=None):
        t, k = self.skew, self.width if max_children is None else max_children
        self.d = {"target": self.padded(self.target), "draft": None if self.drawn == "point" else self.padded(self.draft),
                  "inverse": None if self.DV == self.V else dev(self.inverse), "tokens": dev(self.tokens),
                  "parents": dev(flat(self.forest, 1)), "starts": dev(self.starts.astype(np.uint32)), "u": dev(self.u), "s": dev(self.s),
                  "counts": dev(np.full(len(self.nodes), 7, np.uint32)), "path": dev(np.full(max(1, self.M), 7, np.uint32)),
                  "next": dev(np.full(len(self.nodes), 7, np.uint32))}
        p = {n: None if v is None else v.data_ptr() for n, v in self.d.items()}
        p["target"] += 4 * t
        if p["draft"]:
            p["draft"] += 4 * t
        op = ch.VerifyTree(p["target"], p["tokens"], p["parents"], p["starts"], p["counts"], p["path"], p["next"],
                           requests=len(self.nodes), rows=self.M, vocab=self.V, max_children=k, temperature=self.T,
                           d_draft=p["draft"], d_draft_inverse=p["inverse"], d_accept_draws=p["u"], d_sample_draws=p["s"],
                           draft_vocab=self.DV, without_replacement=self.drawn == "without",
                           target_stride=self.V + t if t else 0, draft_stride=self.DV + t if t else 0)
        self.ws = torch.full((max(16, hip.verify_tree_workspace(op)),), 255, dtype=torch.uint8, device="cuda")
        op.bind_workspace(self.ws.data_ptr(), self.ws.numel())
        return op

    def padded(self, x):
        out = np.full((len(x) + 1, x.shape[1] + self.skew), np.nan, np.float32)
        out.reshape(-1)[self.skew:][:len(x) * out.shape[1]].reshape(len(x), -1)[:, :x.shape[1]] = x
        return dev(out)

    def got(self):
        counts, path, nxt = (host(self.d[n]).tolist() for n in ("counts", "path", "next"))
        out = []
        for r, n in enumerate(self.nodes):
            a = int(self.starts[r])
            assert path[a + counts[r]:a + n] == [NO] * (n - counts[r])
            out.append((path[a:a + counts[r]], nxt[r]))
        return out

    def check(self, hip, **kw):
        op = self.op(hip, **kw)
        hip.verify_tree_device(op, stream())
        want, got = self.expect(kw.get("max_children")), self.got()
        assert got == want, [(g, w) for g, w in zip(got, want) if g != w][:3]
        return want


@pytest.mark.parametrize("drawn", ["without", "with", "point"])
@pytest.mark.parametrize("vocab,draft_vocab", [(40, None), (4099, 700), (9000, None)])
@pytest.mark.parametrize("T", [0.0, 0.6, 1.0])
def test_trees(hip, drawn, vocab, draft_vocab, T):
    say("verify", drawn, vocab, draft_vocab, T)
    accepted = 0
    for seed in range(3):
        v = Verify(seed, [64, 1, 9, 0, 17, 33, 5], vocab, 4 if seed else 1, T, drawn, draft_vocab, std=1.5)
        accepted += sum(len(p) > 1 for p, _ in v.check(hip))
    assert accepted or vocab > 40  # (few of a flat law's tokens are drafted)


@pytest.mark.parametrize("vocab,skew", [(1, 0), (2, 1), (63, 3), (4095, 1), (4096, 0), (4097, 2), (8192, 1), (70001, 1),
                                        (270000, 0), (270001, 1)])
def test_vocabularies_and_alignments(hip, vocab, skew):
    say("verify", vocab, skew)
    for drawn in ("without", "point", "with"):
        v = Verify(vocab, [7, 4, 1], vocab, min(3, vocab), 1.0, drawn, std=2.0, skew=skew)
        v.check(hip)


def test_many_refusals(hip):
    """Drafts that are far from the target: several refusals at a node, eight and more children."""
    for seed in range(6):
        for drawn in ("without", "with", "point"):
            v = Verify(seed, [40, 30, 64], 500, 12, 1.0, drawn, std=1.0, noise=3.0, sharp=-0.5)
            v.check(hip)
            v.check(hip, max_children=2)


@pytest.mark.parametrize("drawn,draft_vocab,noise", [("without", 5000, 0.9), ("with", None, 2.5), ("point", None, 0.9),
                                                     ("without", None, 2.5)])
def test_many_requests_and_long_rows(hip, drawn, draft_vocab, noise):
    """Enough rows that the first round's tests have a launch of their own."""
    say("many", drawn, draft_vocab)
    nodes = [int(x) for x in np.random.default_rng(1).integers(0, 14, 100)]
    Verify(3, nodes, 20000, 4, 0.8, drawn, draft_vocab, noise=noise).check(hip)


def test_a_chain_is_the_chain_rule(hip):
    """One child a node: accepted iff u q < p, else max(p - q, 0) is drawn from."""
    for seed in range(8):
        Verify(seed, [5, 8, 2], 3000, 1, 0.7, "without", chain=1.0).check(hip)


def test_law_of_the_next_token(hip):
    """Whatever the drafts, the first token behind the root follows the target: 4000 trees of one law."""
    for drawn in ("without", "with"):
        rng = np.random.default_rng(17)
        n, V = 4000, 6
        v = Verify(5, [4] * n, V, 3, 1.0, drawn, std=1.0, noise=1.5, forest=[[-1, 0, 0, 0]] * n)
        row, draft = v.target[0].copy(), v.draft[0].copy()
        v.target[:] = row
        v.draft[:] = draft
        q = softmax(draft, 1.0)
        for r in range(n):
            v.tokens[4 * r + 1:4 * r + 4] = rng.choice(V, 3, p=q, replace=drawn == "with")
        hip.verify_tree_device(v.op(hip), stream())
        first = [int(v.tokens[4 * r + p[1]]) if len(p) > 1 else t for r, (p, t) in enumerate(v.got())]
        share, p = np.bincount(first, minlength=V) / n, softmax(row, 1.0)
        assert (np.abs(share - p) < 5 * np.sqrt(p * (1 - p) / n)).all()  # five standard deviations


def test_ruled_out_and_equal_logits(hip):
    v = Verify(1, [9, 9, 9], 300, 4, 1.0, "without", std=1.0)
    v.target[:, 100:] = -np.inf  # tokens that are ruled out
    v.draft[:, 250:] = -np.inf
    v.tokens[:] = v.rng.integers(0, 250, v.M)
    for r in range(3):  # siblings differ
        for u in range(9):
            kids = [i for i, p in enumerate(v.forest[r]) if p == u]
            v.tokens[[9 * r + k for k in kids]] = v.rng.choice(250, len(kids), replace=False)
    v.check(hip)
    v = Verify(2, [9, 9], 64, 4, 0.0, "point")
    v.target[:] = 1.0  # ties: the later token
    v.tokens[1:9] = 63
    v.check(hip)
    v.target[:, 5:] = -np.inf
    v.check(hip)


def test_extreme_laws(hip):
    """A law of one token, in target and draft; large logits; a hot and a cold temperature; the draws 0 and just below 1."""
    for T in (0.01, 1.0, 100.0):
        for drawn in ("without", "with", "point"):
            v = Verify(7, [12, 12, 12], 200, 4, T, drawn, std=2.0)
            v.target[:12, 17] = 3000.0
            v.draft[12:24, 33] = 3000.0
            v.tokens[13:24] = 33
            v.u[:] = np.where(np.arange(v.M) % 3 == 0, 0.0, np.where(np.arange(v.M) % 3 == 1, 1 - 2.0 ** -24, v.u))
            v.s[:] = [0.0, 1 - 2.0 ** -24, 0.5]
            hip.verify_tree_device(v.op(hip), stream())
            for r, (path, token) in enumerate(v.got()):
                assert path[0] == 0 and token < 200
                # the last node's law gives the token some mass
                assert softmax(v.target[12 * r + path[-1]], T)[token] > 0
            if T == 1.0:
                assert v.got()[0][1] == 17 or 17 in [int(v.tokens[n]) for n in v.got()[0][0][1:]]


@pytest.mark.parametrize("T", [0.0, 1.0])
def test_rows_without_a_law_fail_closed(hip, T):
    """No number in a row on the path: nothing of that request is accepted, the others stand."""
    for value in (np.nan, np.inf, None):
        v = Verify(11, [3, 3, 3], 5000, 1, T, "without" if T else "point", chain=1.0, noise=0.05)
        v.u[:] = 0.0  # every draft is accepted
        if T == 0:
            v.tokens[:] = np.roll(v.target.argmax(1), 1)
        want = v.expect()
        assert all(len(p) == 3 for p, _ in want)
        bad = v.target.copy()
        bad[4] = -np.inf if value is None else v.target[4]
        if value is not None:
            bad[4, 4500] = value
        good, v.target = v.target, bad
        hip.verify_tree_device(v.op(hip), stream())
        got = v.got()
        assert got[0] == want[0] and got[2] == want[2] and got[1] == ([], FAILED)
        # off the path it does not matter
        v.target = good.copy()
        v.target[5] = np.nan
        v.forest = [[-1, 0, 1], [-1, 0, 0], [-1, 0, 1]]
        hip.verify_tree_device(v.op(hip, max_children=1), stream())
        assert v.got()[1][0] == [0, 1]


def test_tokens_outside_the_vocabulary_are_refused(hip):
    for drawn in ("without", "point"):
        v = Verify(12, [4], 100, 3, 1.0, drawn, forest=[[-1, 0, 0, 0]])
        v.u[:] = 0.0
        v.tokens[1:3] = [100, NO]
        hip.verify_tree_device(v.op(hip), stream())
        assert v.got()[0][0] == [0, 3]


def test_graph_and_streams(hip):
    """A captured verification replayed over changed numbers, beside one on another stream."""
    a, b = Verify(21, [20, 9, 30], 6000, 4, 1.0, "without"), Verify(22, [64], 9000, 4, 0.9, "with")
    oa, ob = a.op(hip), b.op(hip)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    hip.verify_tree_device(oa, stream())
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        hip.verify_tree_device(oa, stream())
    for i in range(4):
        a.u = np.random.default_rng(i).random(a.M).astype(np.float32)
        a.s = np.random.default_rng(i + 9).random(3).astype(np.float32)
        a.d["u"].copy_(dev(a.u))
        a.d["s"].copy_(dev(a.s))
        torch.cuda.synchronize()
        g.replay()
        hip.verify_tree_device(ob, s.cuda_stream)
        torch.cuda.synchronize()
        assert a.got() == a.expect() and b.got() == b.expect()


def test_workspace(hip):
    v = Verify(31, [30, 30], 9000, 4, 1.0, "without")
    op, big = v.op(hip), v.ws
    w = Verify(32, [5, 3], 4000, 2, 1.0, "without", 500)
    ow = w.op(hip)
    ow.bind_workspace(big.data_ptr(), big.numel())  # one for the most serves less
    hip.verify_tree_device(ow, stream())
    assert w.got() == w.expect()
    op.bind_workspace(big.data_ptr(), big.numel() - 1)
    with pytest.raises(ch.MemoryBudget):
        hip.verify_tree_device(op, stream())


@pytest.mark.parametrize("drawn", ["without", "with", "point"])
@pytest.mark.parametrize("skew", [0, 3])
def test_draw_of_nothing_passes_parts_without_a_weight(hip, drawn, skew):
    """The draw 0 takes the first token that weighs anything. Here everything in front of token 9000 lies 30 / 0.01 below
    the largest logit, e^-3000 of it, and token 0 is ruled out: a root alone, an accepted leaf, a refused child."""
    v = Verify(41, [1, 2, 2], 20000, 2, 0.01, drawn, std=0.05, skew=skew, forest=[[-1], [-1, 0], [-1, 0]])
    for x in (v.target, v.draft):
        x[:, :9000] -= 30.0
        x[:, 0] = -np.inf
    v.tokens[2] = 15000
    v.u[:] = [0.0, 0.0, 0.0, 0.0, 1 - 2.0 ** -24]
    v.tokens[4] = 77  # of no weight: never accepted
    v.s[:] = 0.0
    v.target[1, 15000] = 2.0  # so that request 1's child is accepted
    hip.verify_tree_device(v.op(hip), stream())
    got = v.got()
    assert [p for p, _ in got] == [[0], [0, 1], [0]], got
    # (std 0.05 over T = 0.01 is at most 2^-60 of the largest weight; only r = max(p - q, 0) may leave out more)
    assert got[0][1] == 9000 and got[1][1] == 9000 and 9000 <= got[2][1] < 20000, got


@pytest.mark.parametrize("T", [0.0, 1.0])
def test_more_nodes_than_a_tree_has_fail_closed(hip, T):
    """65 rows and more are no tree of these calls: nothing of that request is accepted, the others stand."""
    for n in (65, 70, 200):
        v = Verify(n, [3, n, 64, 5], 700, 4, T, "without", std=1.5)
        want = v.expect()
        want[1] = ([], FAILED)
        hip.verify_tree_device(v.op(hip), stream())
        assert v.got() == want


@pytest.mark.parametrize("drawn,vocab,draft_vocab,T,requests,skew,pieces", [
    ("without", 60000, None, 1.0, 60, 1, 2), ("with", 60001, 20000, 0.8, 70, 0, 2), ("point", 60000, None, 1.0, 110, 3, 2),
    ("without", 60000, None, 0.0, 110, 2, 2), ("without", 90000, None, 1.2, 60, 0, 3), ("without", 130000, 129999, 1.0, 66, 1, 4)])
def test_statistics_of_longer_parts(hip, drawn, vocab, draft_vocab, T, requests, skew, pieces):
    """Rows enough that the first statistics take parts of several times the later rounds' 4096 tokens: roots alone, leaves
    that are accepted, nodes whose children are refused."""
    say("parts", drawn, vocab, draft_vocab, T, requests, skew, pieces)
    nodes = [int(x) for x in np.random.default_rng(requests).integers(0, 13, requests)]
    nodes[:4] = [1, 12, 1, 12]
    v = Verify(vocab + pieces, nodes, vocab, 4, T, drawn, draft_vocab, skew=skew)
    # (what follows restates when the library takes longer parts, so that this test does not lose its subject)
    chunks, cus = -(-(vocab + 3) // 4096), torch.cuda.get_device_properties(0).multi_processor_count
    reads = v.M * chunks * (2 if T and drawn != "point" else 1)
    assert min(4, 1 + reads // (32 * cus)) == pieces
    want = v.check(hip)
    ends = [len(parent) > 1 and path[-1] in parent for parent, (path, _) in zip(v.forest, want) if parent]
    leaves = [len(path) > 1 and path[-1] not in parent for parent, (path, _) in zip(v.forest, want) if parent]
    assert any(ends) and any(leaves)
