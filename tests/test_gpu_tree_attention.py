"""GPU parity of attention over trees of drafted tokens: the ragged batch's attention with masks over the last rows.

Against the formula in float64 over the values that the pages stand for, with the tolerance that is derived in
test_gpu_paged_attention_rows.py: the arithmetic of a (row, token) pair is the same, only which pairs there are differs.
"""
import numpy as np
import pytest
import torch

import ctox_hip as ch
import test_gpu_paged_attention_rows as rows
from test_gpu_paged_attention_rows import HD, dev
from tree_model import masks, random_tree

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)


class Trees(rows.Batch):
    """Requests (cached, nodes); masks: [rows] words (of random trees where none are given)."""

    def __init__(self, seed, requests, page, heads, kv_heads, masks_=None, chain=0.3, **kw):
        super().__init__(seed, requests, page, heads, kv_heads, **kw)
        rng = np.random.default_rng(seed + 1)
        self.forest = [random_tree(rng, n, 4, chain) for _, n in requests]
        own = np.concatenate([masks(p) for p in self.forest] + [np.zeros(0, np.uint64)])
        self.masks = own if masks_ is None else np.asarray(masks_, np.uint64)
        self.masks = np.concatenate([self.masks, np.full(len(self.q) - self.M, 2 ** 64 - 1, np.uint64)])

    def expect(self):
        want, tol = np.zeros((self.M, self.H, HD)), np.zeros((self.M, self.H, HD))
        G, e = self.H // self.KV, 2.0 ** -24
        for r, (cached, n) in enumerate(self.requests):
            if n == 0:
                continue
            K, V, present = self.token_values(r)
            j = np.arange(self.tokens[r])
            for t in range(n):
                at = self.starts[r] + t
                m = int(self.masks[at])
                see = present & np.array([x < cached or bool(m >> (x - cached) & 1) for x in j.tolist()], bool)
                if not see.any():
                    continue
                for h in range(self.H):
                    k, v, q = K[see, h // G], V[see, h // G], self.q[at, h].astype(np.float64)
                    s = k @ q / 16.0
                    S = (np.abs(k) @ np.abs(q) / 16.0).max()
                    p = np.exp(s - s.max())
                    p /= p.sum()
                    want[at, h] = p @ v
                    tol[at, h] = (p @ np.abs(v)) * e * (4 * (144 * S + 4 * max(1, 2 * S)) + 72 + 3 * see.sum())
        return want, tol

    def tree_op(self, hip, max_rows=0):
        inner = self.op(hip)
        pointers = [getattr(inner, n) for n in ("query", "out", "q2_pages", "q4_pages", "descriptors", "row_starts", "tokens")]
        self.d["masks"] = dev(self.masks.view(np.int64))
        t = ch.PagedGqaTree(*pointers, self.d["masks"].data_ptr(), rows=inner.rows, requests=inner.requests,
                            params=inner.params, max_rows=max_rows)
        self.ws = torch.full((max(16, hip.paged_gqa_tree_workspace(t)),), 255, dtype=torch.uint8, device="cuda")
        t.bind_workspace(self.ws.data_ptr(), self.ws.numel())
        return t

    def check(self, hip, max_rows=0):
        t = self.tree_op(hip, max_rows)
        hip.paged_gqa_tree_device(t, torch.cuda.current_stream().cuda_stream)
        got = self.d["out"].cpu().numpy()
        want, tol = self.expect()
        off = np.abs(got[:self.M] - want)
        assert (off <= tol).all(), (off / np.maximum(tol, 1e-30)).max()
        assert (got[self.M:] == 7.0).all()  # rows behind the last request
        return got


@pytest.mark.parametrize("page,heads,kv", [(16, 24, 4), (24, 6, 2), (7, 8, 8), (128, 4, 1)])
@pytest.mark.parametrize("requests", [[(0, 1)], [(0, 64)], [(40, 64)], [(300, 12)], [(31, 33), (0, 7), (100, 0), (513, 20)],
                                      [(64, 2), (5, 1), (0, 0)]])
def test_trees(hip, page, heads, kv, requests):
    say("trees", page, heads, kv, requests)
    Trees(page + heads + len(requests), requests, page, heads, kv, pad=3, q2=lambda r, p: p % 3 == 1 and (p + 1) * page <= requests[r][0]).check(hip)


@pytest.mark.parametrize("max_rows", [0, 2, 5, 10, 64])
def test_kernels_by_bound(hip, max_rows):
    """The kernels of 16, 32 and 128 queries, alone and together."""
    n = [min(max_rows or 64, x) for x in (1, 2, 5, 10, 64)]
    say("bound", max_rows, n)
    Trees(max_rows, [(150 + 37 * i, x) for i, x in enumerate(n)], 16, 6, 1).check(hip, max_rows)


@pytest.mark.parametrize("heads,kv", [(6, 1), (24, 4)])
def test_any_mask(hip, heads, kv):
    """Masks that are no trees: nothing, everything, bits past the rows, a row that does not see itself."""
    rng = np.random.default_rng(5)
    requests = [(0, 8), (33, 8), (95, 64), (0, 3), (70, 2)]
    m = rng.integers(0, 2 ** 63, 85, dtype=np.uint64) * 2 + rng.integers(0, 2, 85, dtype=np.uint64)
    m[:4] = [0, 2 ** 64 - 1, 2 ** 63, 1 << 7]
    m[8:10] = [0, 2 ** 64 - 1 - 2]
    m[80:85] = [0, 4, 0, 2, 1]
    b = Trees(8, requests, 16, heads, kv, masks_=m)
    got = b.check(hip)
    assert not got[0].any() and not got[2].any() and not got[80].any()  # nothing cached, nothing seen


def test_chain_is_causal_attention(hip):
    """A chain's masks are causal attention: both calls lie within the same bound of the same values."""
    for requests in ([(700, 5), (33, 1)], [(700, 40), (90, 64), (0, 33)], [(2000, 12)]):
        b = Trees(4, requests, 16, 24, 4)
        b.masks = np.concatenate([masks(list(range(-1, n - 1))) for _, n in requests])
        got = b.check(hip)
        op = b.op(hip, max_rows=64)
        b.d["out"].fill_(7.0)
        hip.paged_gqa_rows_device(op, torch.cuda.current_stream().cuda_stream)
        want, tol = b.expect()
        causal = b.d["out"].cpu().numpy()
        assert (np.abs(causal - want) <= tol).all() and (np.abs(causal - got) <= 2 * tol).all()


def test_a_hidden_node_without_finite_values(hip):
    """Values and keys of nodes that are no numbers reach the rows that see them, and no others."""
    for heads, kv, n in ((6, 1, 2), (6, 1, 5), (24, 4, 30)):
        def edit(b):
            for node in (1, n - 1):
                pos = 40 + node
                kind, slot, _, first = (int(x) for x in b.desc[0, pos // 16])
                raw = b.pool[kind][slot, pos - first]
                raw[b.blocks // 2:, :2] = np.frombuffer(np.float16(np.inf).tobytes(), np.uint8)
        b = Trees(9, [(40, n)], 16, heads, kv, edit=edit)
        t = b.tree_op(hip)
        hip.paged_gqa_tree_device(t, torch.cuda.current_stream().cuda_stream)
        got = b.d["out"].cpu().numpy()
        for t in range(n):
            sees = any(int(b.masks[t]) >> node & 1 for node in (1, n - 1))
            assert np.isnan(got[t]).all() if sees else np.isfinite(got[t]).all(), (n, t)


def test_two_streams_and_a_graph(hip):
    """A captured call, replayed over other lengths and masks, beside eager work; workspaces of their own."""
    a = Trees(11, [(300, 20), (50, 64)], 16, 6, 1)
    b = Trees(12, [(200, 33), (150, 10)], 16, 6, 1, max_pages=a.max_pages)
    ta, tb = a.tree_op(hip), b.tree_op(hip)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        hip.paged_gqa_tree_device(ta, s.cuda_stream)
    torch.cuda.synchronize()
    first = a.d["out"].clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        hip.paged_gqa_tree_device(ta, torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        a.d["out"].fill_(3.0)
        g.replay()
        with torch.cuda.stream(s):
            hip.paged_gqa_tree_device(tb, s.cuda_stream)
        torch.cuda.synchronize()
        assert torch.equal(a.d["out"], first)
    want, tol = b.expect()
    assert (np.abs(b.d["out"].cpu().numpy()[:b.M] - want) <= tol).all()
    # other masks and lengths in the same buffers
    a.masks[:] = 1
    a.d["masks"].copy_(dev(a.masks.view(np.int64)))
    g.replay()
    torch.cuda.synchronize()
    want, tol = a.expect()
    assert (np.abs(a.d["out"].cpu().numpy()[:a.M] - want) <= tol).all()


def test_workspace_serves_smaller_calls(hip):
    big = Trees(13, [(500, 64), (20, 30), (90, 12)], 16, 24, 4)
    t = big.tree_op(hip)
    for requests in ([(500, 3)], [(100, 64), (3, 1)], [(500, 12)]):
        b = Trees(14, requests, 16, 24, 4)
        op = b.tree_op(hip)
        op.bind_workspace(big.ws.data_ptr(), big.ws.numel())
        hip.paged_gqa_tree_device(op, torch.cuda.current_stream().cuda_stream)
        want, tol = b.expect()
        assert (np.abs(b.d["out"].cpu().numpy()[:b.M] - want) <= tol).all()
    t.bind_workspace(big.ws.data_ptr(), 16)
    with pytest.raises(ch.MemoryBudget):
        hip.paged_gqa_tree_device(t, None)


@pytest.mark.parametrize("heads,kv,most", [(6, 1, 2), (24, 4, 2), (8, 8, 16), (4, 2, 8)])
@pytest.mark.parametrize("cached", [30, 31, 32, 63, 95, 96])
def test_a_hidden_first_node(hip, heads, kv, most, cached):
    """At most 16 queries a KV head: rows that do not see node 0, which may be a full tile's last token."""
    say("hidden first node", heads, kv, most, cached)
    rng = np.random.default_rng(cached + heads)
    requests = [(cached, most), (cached + 1, most), (cached - 1, most)]
    free = rng.integers(0, 2 ** most, 3 * most, dtype=np.uint64)
    free[:most] &= np.uint64(2 ** most - 2)
    Trees(cached, requests, 16, heads, kv, masks_=free).check(hip, most)
    # several roots: every other node is one
    parent = [i - 1 if i % 2 else -1 for i in range(most)]
    Trees(cached + 1, requests, 16, heads, kv, masks_=np.concatenate([masks(parent)] * 3)).check(hip, most)


def test_no_rows_need_no_buffers(hip):
    """A step without nodes: addresses of empty buffers are null, as in the ragged batch's call."""
    b = Trees(15, [(20, 0), (5, 0)], 16, 6, 1)
    t = b.tree_op(hip)
    t.rows.rows, t.rows.query, t.rows.out, t.masks = 0, None, None, None
    t.bind_workspace(None, 0)
    hip.paged_gqa_tree_device(t, torch.cuda.current_stream().cuda_stream)
