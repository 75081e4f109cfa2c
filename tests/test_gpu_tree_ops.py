"""Plan of trees, commits, free slots and forks on the GPU: whole numbers and bytes, equal to the host's."""
import numpy as np
import pytest
import torch

import ctox_hip as ch
from tree_model import NO, flat, lines, masks, random_tree, starts

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)


def dev(a):
    a = np.ascontiguousarray(a)
    return torch.from_numpy(a.view({np.dtype(np.uint32): np.int32, np.dtype(np.uint64): np.int64}.get(a.dtype, a.dtype))).cuda()


def host(t):
    a = t.cpu().numpy()
    return a.view({np.dtype(np.int32): np.uint32, np.dtype(np.int64): np.uint64}.get(a.dtype, a.dtype))


def stream():
    return torch.cuda.current_stream().cuda_stream


# ---------------------------------------------------------------- plan
def run_plan(hip, forest, cached, pad=0, parents=None):
    nodes = [len(p) for p in forest]
    R, rows = len(forest), sum(nodes) + pad
    t = {"starts": dev(starts(nodes).astype(np.uint32)), "tokens": dev(np.array([a + n for a, n in zip(cached, nodes)], np.uint32)),
         "parents": dev(flat(forest, pad) if parents is None else parents), "masks": dev(np.full(max(rows, 1), 77, np.uint64)),
         "positions": dev(np.full(max(rows, 1), 99, np.uint32)), "depths": dev(np.full(R, 55, np.uint32))}
    hip.tree_plan_device(ch.TreePlan(*(t[k].data_ptr() for k in ("starts", "tokens", "parents", "masks", "positions", "depths")),
                                     requests=R, rows=rows), stream())
    return host(t["masks"]), host(t["positions"]), host(t["depths"])


@pytest.mark.parametrize("nodes,chain", [([1], 0), ([64], 1.0), ([64], 0), ([63, 2, 0, 1, 17], 0.5), ([5] * 300, 0.7),
                                         ([0], 0), ([0, 0, 3], 0), ([33, 0, 64], 0.9)])
def test_plan(hip, nodes, chain):
    say("plan", nodes[:5], len(nodes))
    rng = np.random.default_rng(len(nodes) + sum(nodes))
    forest = [random_tree(rng, n, 4, chain) for n in nodes]
    cached = [int(x) for x in rng.integers(0, 1 << 30, len(nodes))]
    m, pos, depths = run_plan(hip, forest, cached, pad=5)
    want = np.concatenate([masks(p) for p in forest] + [np.zeros(5, np.uint64)])
    assert np.array_equal(m, want)
    where = [a + len(line) - 1 for a, p in zip(cached, forest) for line in lines(p)]
    assert np.array_equal(pos, np.array(where + [99] * 5, np.uint32))
    assert depths.tolist() == [max((len(x) for x in lines(p)), default=0) for p in forest]


def test_plan_parents_that_are_none(hip):
    """A parent that is not in front of its node makes it a root; more than 64 rows are no tree."""
    parents = np.array([NO, 0, 5, 3, 1, 4, NO, 0xfffffff0], np.uint32)
    m, pos, depths = run_plan(hip, [[0] * 8], [10], parents=parents)
    assert m.tolist() == [1, 3, 4, 8, 0b10011, 0b110011, 64, 128] and depths.tolist() == [4]
    assert pos.tolist() == [10, 11, 10, 10, 12, 13, 10, 10]
    m, pos, depths = run_plan(hip, [[0] * 65, [-1, 0]], [0, 7])
    assert depths.tolist() == [NO, 2] and not m[:65].any() and m[65:67].tolist() == [1, 3]


# ---------------------------------------------------------------- pages
class Pages:
    """Tables of R requests over layers' pools, and what the calls make of them on the host."""

    def __init__(self, seed, tokens, nodes, page=16, layers=2, token_bytes=272, spare=9, max_pages=None, q2=0.3, gap=0):
        rng = self.rng = np.random.default_rng(seed)
        self.R, self.page, self.layers, self.token_bytes = len(tokens), page, layers, token_bytes
        self.tokens, self.nodes = np.array(tokens, np.uint32), nodes
        pages = [-(-t // page) for t in tokens]
        self.max_pages = max_pages or max(1, max(pages) + 1)
        # pages in front of the nodes may lie in the Q2 pool
        kinds = [[int(not (rng.random() < q2 and (p + 1) * page <= t - n)) for p in range(k)]
                 for k, t, n in zip(pages, tokens, nodes)]
        self.n4 = sum(sum(k) for k in kinds) + spare
        self.n2 = sum(len(k) - sum(k) for k in kinds) + 3
        slots = {1: iter(rng.permutation(self.n4)), 0: iter(rng.permutation(self.n2))}
        self.desc = np.full((self.R, self.max_pages, 4), 0xabcd, np.uint32)
        for r, ks in enumerate(kinds):
            for p, kind in enumerate(ks):
                self.desc[r, p] = (kind, next(slots[kind]), min(page, tokens[r] - p * page), p * page)
        self.page_bytes = page * token_bytes + gap
        self.pool = rng.integers(0, 256, (layers, self.n4 * self.page_bytes)).astype(np.uint8)
        self.starts = starts(nodes)
        self.d = {"pool": dev(self.pool), "desc": dev(self.desc), "starts": dev(self.starts.astype(np.uint32)),
                  "tokens": dev(self.tokens)}
        self.new = self.tokens.copy()

    def geometry(self):
        return dict(requests=self.R, page_tokens=self.page, max_pages=self.max_pages, q4_slots=self.n4)

    def pools(self):
        return [self.d["pool"][i].data_ptr() for i in range(self.layers)]

    def token(self, r, pos):
        at = int(self.desc[r, pos // self.page, 1]) * self.page_bytes + pos % self.page * self.token_bytes
        return slice(at, at + self.token_bytes)

    def commit(self, hip, kept, codes=None):
        """kept: per request a list of nodes, or None (ended)."""
        path = np.full(max(1, self.starts[-1]), NO, np.uint32)
        counts = np.array([NO if k is None else len(k) for k in kept], np.uint32)
        for r, k in enumerate(kept):
            if k:
                path[self.starts[r]:self.starts[r] + min(len(k), self.nodes[r])] = k[:self.nodes[r]]
        d = {"counts": dev(counts), "path": dev(path), "new": dev(np.full(self.R, 7, np.uint32)),
             "status": dev(np.full(self.R, 7, np.uint32))}
        op = ch.PagedCommit(self.pools(), self.d["desc"].data_ptr(), self.d["starts"].data_ptr(), self.d["tokens"].data_ptr(),
                            d["counts"].data_ptr(), d["path"].data_ptr(), d["new"].data_ptr(), d["status"].data_ptr(),
                            rows=len(path), token_bytes=self.token_bytes, q4_page_bytes=self.page_bytes, **self.geometry())
        hip.paged_commit_device(op, stream())
        codes = codes or [0] * self.R
        for r, k in enumerate(kept):
            if codes[r]:
                continue
            past = int(self.tokens[r]) - self.nodes[r]
            for j, node in enumerate(k or []):  # in order: a later token is never at an earlier one's new place
                self.pool[:, self.token(r, past + j)] = self.pool[:, self.token(r, past + node)]
            self.new[r] = 0 if k is None else past + len(k)
            for p in range(-(-int(self.tokens[r]) // self.page)):
                self.desc[r, p, 2] = max(0, min(self.page, int(self.new[r]) - p * self.page))
        assert host(d["status"]).tolist() == codes
        assert np.array_equal(host(d["new"]), self.new)
        self.same()
        self.d["tokens"] = d["new"]
        self.op = op, d
        return op

    def same(self):
        assert np.array_equal(host(self.d["desc"]), self.desc.reshape(host(self.d["desc"]).shape))
        assert np.array_equal(self.d["pool"].cpu().numpy(), self.pool)

    def free(self, hip, q2=True):
        d = {"q4": dev(np.full(max(1, self.n4), 7, np.uint32)), "q2": dev(np.full(self.n2, 7, np.uint32)), "counts": dev(np.full(2, 7, np.uint32))}
        op = ch.PagedFreeSlots(self.d["desc"].data_ptr(), self.d["tokens"].data_ptr(), d["q4"].data_ptr(),
                               d["q2"].data_ptr() if q2 else None, d["counts"].data_ptr(), q2_slots=self.n2 if q2 else 0,
                               **self.geometry())
        ws = torch.full((max(4, hip.paged_free_slots_workspace(op)),), 255, dtype=torch.uint8, device="cuda")
        op.bind_workspace(ws.data_ptr(), ws.numel())
        hip.paged_free_slots_device(op, stream())
        live = [self.desc[r, p] for r in range(self.R) for p in range(-(-int(self.new[r]) // self.page))]
        want = [sorted(set(range(n)) - {int(x[1]) for x in live if (x[0] != 0) == bool(kind)})
                for kind, n in ((1, self.n4), (0, self.n2 if q2 else 0))]
        assert host(d["counts"]).tolist() == [len(w) for w in want]
        assert host(d["q4"]).tolist()[:self.n4] == want[0] + [NO] * (self.n4 - len(want[0]))
        if q2:
            assert host(d["q2"]).tolist() == want[1] + [NO] * (self.n2 - len(want[1]))
        self.lists = want
        return d

    def fork(self, hip, pairs, lists, code=0, free=None, count=None):
        free = self.lists[0] if free is None else free
        d = {"s": dev(np.array([a for a, _ in pairs] + [0], np.uint32)), "t": dev(np.array([b for _, b in pairs] + [0], np.uint32)),
             "free": dev(np.array(free + [NO], np.uint32)), "count": dev(np.array([len(free) if count is None else count], np.uint32)),
             "status": dev(np.full(2, 7, np.uint32))}
        hip.paged_fork_device(ch.PagedFork(
            self.pools(), self.d["desc"].data_ptr(), self.d["tokens"].data_ptr(), d["s"].data_ptr(), d["t"].data_ptr(),
            d["free"].data_ptr(), d["count"].data_ptr(), d["status"].data_ptr(), forks=len(pairs),
            token_bytes=self.token_bytes, q4_page_bytes=self.page_bytes, **self.geometry()), stream())
        taken = 0
        for a, b in pairs if not code else []:
            t = int(self.new[a])
            for p in range(-(-t // self.page)):
                self.desc[b, p] = self.desc[a, p]
            if t % self.page:
                p, n = t // self.page, t % self.page * self.token_bytes
                old, new = int(self.desc[a, p, 1]) * self.page_bytes, free[taken] * self.page_bytes
                self.pool[:, new:new + n] = self.pool[:, old:old + n]
                self.desc[b, p, 1] = free[taken]
                taken += 1
            self.new[b] = t
        assert host(d["status"]).tolist() == [code, taken]
        assert np.array_equal(host(self.d["tokens"]), self.new)
        self.same()


def paths(rng, nodes, end=0.2):
    out = []
    for n in nodes:
        if rng.random() < end:
            out.append(None)
        else:
            out.append(sorted(int(x) for x in rng.choice(n, int(rng.integers(0, n + 1)), replace=False)) if n else [])
    return out


@pytest.mark.parametrize("page,layers,token_bytes,gap", [(16, 2, 1088, 0), (7, 3, 272, 0), (128, 1, 136, 4), (1, 2, 68, 0),
                                                        (24, 64, 272, 16)])
def test_commit_free_fork(hip, page, layers, token_bytes, gap):
    say("commit", page, layers, token_bytes)
    rng = np.random.default_rng(page)
    nodes = [64, 1, 0, 17, 33, 5, 64, 8]
    tokens = [n + int(x) for n, x in zip(nodes, [0, 0, 40, 129, 300, 1, 95, 16])]
    p = Pages(page, tokens, nodes, page, layers, token_bytes, spare=30, gap=gap)
    p.free(hip)
    kept = paths(rng, nodes, 0)
    kept[1] = kept[4] = None
    kept[0] = [0, 1, 2, 10, 63]
    kept[6] = list(range(64))
    p.commit(hip, kept)
    p.free(hip, q2=page != 7)
    p.fork(hip, [(0, 1), (3, 4), (3, 7)], p.lists)
    p.free(hip)
    p.fork(hip, [], p.lists)


def test_commit_of_many_requests(hip):
    rng = np.random.default_rng(3)
    nodes = [int(x) for x in rng.integers(0, 20, 700)]
    p = Pages(4, [n + int(x) for n, x in zip(nodes, rng.integers(0, 60, 700))], nodes, 8, 1, 136, spare=500)
    p.commit(hip, paths(rng, nodes))
    p.free(hip)
    ended = [r for r in range(700) if p.new[r] == 0][:40]
    going = [r for r in range(700) if r not in ended]
    p.fork(hip, [(int(rng.choice(going)), t) for t in ended], p.lists)
    p.free(hip)


def test_free_slots_of_large_tables(hip):
    """Tables that the one-launch form does not take, several thousand words of slots."""
    rng = np.random.default_rng(5)
    tokens = [int(x) for x in rng.integers(0, 4000, 40)]
    p = Pages(6, tokens, [0] * 40, 4, 1, 68, spare=20000, max_pages=1000)
    p.free(hip)
    p = Pages(7, [5], [0], 4, 1, 68, spare=300000)
    p.free(hip)


def test_commit_refuses_on_the_device(hip):
    """Codes a request; its neighbours are committed, it is left as it is."""
    nodes = [6, 6, 6, 6, 6, 3]
    for page in (4, 16):
        p = Pages(8, [20, 20, 20, 20, 20, 20], nodes, page, 2, 272, q2=0)
        p.desc[4, 19 // page, 0] = 0  # the page of the last token is a Q2 page
        p.d["desc"].copy_(dev(p.desc))
        p.commit(hip, [[0, 2, 1], [0, 6], [0] * 7, [0, 5], [0, 5], [2]], [2, 2, 1, 0, 2, 0])
    p = Pages(9, [10, 12], [4, 4], 16, 1, 272, max_pages=1)
    p.tokens[:] = p.new[:] = [17, 3]  # longer than its table; shorter than its rows
    p.d["tokens"].copy_(dev(p.tokens))
    p.commit(hip, [[0, 3], [0, 1]], [1, 1])


def test_fork_refuses_on_the_device(hip):
    p = Pages(10, [20, 37, 0, 5], [0] * 4, 16, 2, 272, q2=0, spare=4)
    p.free(hip)
    p.fork(hip, [(0, 2), (2, 3)], None, code=1)      # a target is a source
    p.fork(hip, [(0, 2), (1, 2)], None, code=1)      # one target twice
    p.fork(hip, [(0, 4)], None, code=1)
    p.fork(hip, [(9, 2)], None, code=1)
    p.fork(hip, [(0, 2), (1, 3)], None, code=2, count=1)
    p.fork(hip, [(0, 2), (1, 3)], None, code=4, free=[p.lists[0][0], p.n4])
    p.desc[1, 2, 0] = 0
    p.d["desc"].copy_(dev(p.desc))
    p.fork(hip, [(1, 2)], None, code=3)
    p.fork(hip, [(0, 2)], None)
    p.fork(hip, [(0, 2), (0, 3)], None, free=p.lists[0][1:])


def test_workspace_is_checked(hip):
    p = Pages(11, [20], [0])
    op = ch.PagedFreeSlots(p.d["desc"].data_ptr(), p.d["tokens"].data_ptr(), p.d["tokens"].data_ptr(), None,
                           p.d["tokens"].data_ptr(), q2_slots=0, **p.geometry())
    with pytest.raises(ch.MemoryBudget):
        hip.paged_free_slots_device(op, stream())


def test_fork_of_more_pages_than_the_pool_has(hip):
    """A count of free slots that is larger than the pool does not make room: nothing is changed."""
    p = Pages(14, [5, 0, 0, 0], [0] * 4, 16, 2, 272, q2=0, spare=1)
    assert p.n4 == 2
    p.free(hip)
    spare = p.lists[0][0]
    p.fork(hip, [(0, 1), (0, 2), (0, 3)], None, code=2, free=[spare, spare], count=9)
    p.fork(hip, [(0, 1), (0, 2), (0, 3)], None, code=2, free=[spare, spare], count=NO)
    p.fork(hip, [(0, 3)], None, free=[spare], count=1)
