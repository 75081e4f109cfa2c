"""The GatedDeltaNet token mixer over trees, and the state behind a path, against the recurrence in float64.

Every node's output is held to the sequential recurrence along its path (Q/src/reference.rs:230-297 behind the
convolution of :159-187 and the gates of Q/src/decoder.rs:881-902). Bound of the error, relative to the norm of an output
row: convolution, gates and norms 16 roundings of values of the row's size; k . S over 128 rows and the Gram sums
as many, each of products of unit vectors; a solve over d ancestors adds the errors of d terms of at most the
size of the largest delta. With e = 2^-24 that is (16 + 128 + 128 + 4 d + |log decays| + 16) e of the largest of |S_0|, |v|
and the deltas, taken as 512 e of the request's largest row; the state of a path likewise.
"""
import numpy as np
import pytest
import torch

import ctox_hip as ch
from tree_model import NO, flat, lines, random_tree, starts
from test_gpu_tree_ops import dev, host, stream

pytestmark = pytest.mark.gpu

E = 2.0 ** -24


def say(*a):
    print(*a, flush=True)


def block(s):
    """[.., heads][key][value] to the engine's order."""
    *lead, dk, dv = s.shape
    S = -(-dv // 16)
    full = np.zeros((*lead, 128, 16 * S), s.dtype)
    full[..., :dk, :dv] = s
    full = full.reshape(*lead, 8, 16, S, 16)
    n = len(lead)
    return np.ascontiguousarray(full.transpose(*range(n), n + 2, n + 1, n + 3, n)).reshape(*lead, S * 2048)


class Layer:
    def __init__(self, seed, nodes, heads=6, key_heads=2, dk=128, dv=128, K=4, blocked=False, chain=0.3, extra=5, pad=0,
                 parents=None, decay=1.0, s_std=0.1):
        rng = self.rng = np.random.default_rng(seed)
        self.H, self.KH, self.dk, self.dv, self.K, self.blocked = heads, key_heads, dk, dv, K, blocked
        self.nodes, R = nodes, len(nodes)
        self.forest = parents or [random_tree(rng, n, 4, chain) for n in nodes]
        self.starts = starts(nodes)
        self.M = int(self.starts[-1])
        self.C = 2 * key_heads * dk + heads * dv
        self.stride = self.C + 2 * heads + extra
        f = lambda *s, std=1.0: (rng.standard_normal(s) * std).astype(np.float32)
        self.proj = f(max(1, self.M) + pad, self.stride)
        self.w, self.windows = f(self.C, K, std=0.4), f(R, self.C, K)
        self.a_log = np.log(rng.uniform(0.05, 1.0, heads) * decay).astype(np.float32)
        self.dt = f(heads, std=0.5) - 2
        self.state = f(R, heads, dk, dv, std=s_std)
        self.kept = []
        for parent in self.forest:
            path = [0] if parent else []
            while path and rng.random() < 0.85:
                below = [i for i, p in enumerate(parent) if p == path[-1]]
                if not below:
                    break
                path.append(int(rng.choice(below)))
            self.kept.append(path)

    def expect(self):
        H, KH, dk, dv = self.H, self.KH, self.dk, self.dv
        out = np.zeros((self.M, H, dv))
        state, windows = self.state.astype(np.float64), self.windows.astype(np.float64)
        after, slid = state.copy(), windows.copy()
        for r, parent in enumerate(self.forest):
            S, win = {-1: state[r]}, {-1: windows[r]}
            for i, p in enumerate(parent):
                p = p if 0 <= p < i else -1
                row = self.proj[self.starts[r] + i].astype(np.float64)
                win[i] = np.concatenate([win[p][:, 1:], row[:self.C, None]], 1)
                y = (win[i] * self.w).sum(1)
                with np.errstate(over="ignore"):
                    y = y / (1 + np.exp(-y))
                q, k = (y[j * KH * dk:(j + 1) * KH * dk].reshape(KH, dk) for j in range(2))
                q, k = (np.repeat(x / np.sqrt((x * x).sum(1, keepdims=True) + 1e-6), H // KH, 0) for x in (q, k))
                v = y[2 * KH * dk:].reshape(H, dv)
                g = row[self.C:self.C + H] + self.dt
                ld = -np.exp(self.a_log.astype(np.float64)) * np.logaddexp(0, g)
                beta = 1 / (1 + np.exp(-row[self.C + H:self.C + 2 * H]))
                T = S[p] * np.exp(ld)[:, None, None]
                d = (v - np.einsum("hij,hi->hj", T, k)) * beta[:, None]
                S[i] = T + k[:, :, None] * d[:, None]
                out[self.starts[r] + i] = np.einsum("hij,hi->hj", S[i], q) / np.sqrt(dk)
            if self.kept[r]:
                after[r], slid[r] = S[self.kept[r][-1]], win[self.kept[r][-1]]
        return out, after, slid

    def op(self, hip, in_place=False, max_rows=0, gap=0):
        path, counts = np.full(max(1, self.M), NO, np.uint32), np.array([len(k) for k in self.kept], np.uint32)
        for r, k in enumerate(self.kept):
            path[self.starts[r]:self.starts[r] + len(k)] = k
        s = block(self.state).reshape(len(self.nodes), -1) if self.blocked else self.state.reshape(len(self.nodes), -1)
        self.floats = s.shape[1]
        s = np.concatenate([s, np.full((len(s), gap), 5, np.float32)], 1)
        w = np.concatenate([self.windows.reshape(len(s), -1), np.full((len(s), gap), 6, np.float32)], 1)
        d = self.d = {"proj": dev(self.proj), "w": dev(self.w), "win": dev(w), "a": dev(self.a_log), "dt": dev(self.dt),
                      "state": dev(s), "starts": dev(self.starts.astype(np.uint32)), "parents": dev(flat(self.forest, 1)),
                      "out": torch.full((len(self.proj), self.H, self.dv), 9.0, device="cuda"), "counts": dev(counts), "path": dev(path)}
        d["win2"] = d["win"] if in_place else torch.full_like(d["win"], 8)
        d["state2"] = d["state"] if in_place else torch.full_like(d["state"], 8)
        p = {k: v.data_ptr() for k, v in d.items()}
        op = ch.GdnTree(p["proj"], p["w"], p["win"], p["a"], p["dt"], p["state"], p["starts"], p["parents"], p["out"],
                        proj_stride=self.stride, a_off=self.C, b_off=self.C + self.H, requests=len(self.nodes), rows=self.M,
                        heads=self.H, key_heads=self.KH, key_dim=self.dk, value_dim=self.dv, kernel=self.K, d_counts=p["counts"],
                        d_path=p["path"], d_conv_out=p["win2"], d_state_out=p["state2"], max_rows=max_rows, blocked=self.blocked,
                        conv_stride=w.shape[1] if gap else 0, state_stride=s.shape[1] if gap else 0)
        self.ws = torch.full((max(16, hip.gdn_tree_workspace(op)),), 255, dtype=torch.uint8, device="cuda")
        op.bind_workspace(self.ws.data_ptr(), self.ws.numel())
        return op

    def compare(self):
        out, after, slid = self.expect()
        got = self.d["out"].cpu().numpy()
        assert (got[self.M:] == 9.0).all()
        for r, n in enumerate(self.nodes):
            a = int(self.starts[r])
            big = max(np.abs(self.state[r]).max() * 4, np.linalg.norm(out[a:a + n], axis=-1).max(initial=0), 1.0)
            assert np.linalg.norm(got[a:a + n] - out[a:a + n], axis=-1).max(initial=0) <= 512 * E * big, r
        state = self.d["state2"].cpu().numpy()[:, :self.floats]
        want = block(after).reshape(state.shape) if self.blocked else after.reshape(state.shape)
        assert np.abs(state - want).max() <= 512 * E * max(1.0, np.abs(want).max())
        assert np.array_equal(self.d["win2"].cpu().numpy()[:, :self.C * self.K].reshape(slid.shape), slid.astype(np.float32))

    def check(self, hip, **kw):
        op = self.op(hip, **kw)
        hip.gdn_tree_device(op, stream())
        hip.gdn_tree_commit_device(op, stream())
        self.compare()


@pytest.mark.parametrize("blocked", [False, True])
@pytest.mark.parametrize("nodes,chain", [([1], 0), ([16], 0.0), ([17], 0.5), ([64], 1.0), ([64], 0.0),
                                         ([3, 0, 33, 64, 1, 16, 32, 48], 0.4)])
def test_trees(hip, nodes, chain, blocked):
    say("delta", nodes, chain, blocked)
    Layer(len(nodes) + nodes[0], nodes, chain=chain, blocked=blocked, pad=2).check(hip)


@pytest.mark.parametrize("heads,key_heads,dk,dv", [(4, 4, 128, 64), (6, 2, 64, 128), (3, 1, 96, 80), (2, 1, 1, 1),
                                                   (2, 2, 17, 130), (48, 16, 128, 128)])
@pytest.mark.parametrize("K", [4, 1, 3, 8])
def test_shapes(hip, heads, key_heads, dk, dv, K):
    say("delta", heads, key_heads, dk, dv, K)
    for blocked in (False, True):
        Layer(dk + K, [20, 5, 33], heads, key_heads, dk, dv, K, blocked, chain=0.6).check(hip, gap=8)


@pytest.mark.parametrize("most,nodes", [(16, [16, 1, 9]), (32, [32, 17, 3]), (64, [64, 33]), (5, [5, 4])])
def test_bounds_and_batches(hip, most, nodes):
    """The kernels of each bound, with 64 value columns a workgroup and, in batches, 128."""
    say("delta", most)
    for count in (1, 15):
        Layer(most, nodes * count, 24, 8, chain=0.5, blocked=True).check(hip, max_rows=most, in_place=True)


def test_a_chain_is_the_fused_step(hip):
    """A chain's rows and its committed state are those of the row-by-row call."""
    L = Layer(5, [5], 48, 16, chain=1.0)
    L.kept = [[0, 1, 2, 3, 4]]
    L.check(hip)
    conv, state = dev(L.windows), dev(L.state)
    conv2, out = torch.zeros_like(conv), torch.zeros(5, 48, 128, device="cuda")
    ld, beta = torch.zeros(5, 48, device="cuda"), torch.zeros(5, 48, device="cuda")
    lib = ch.load_library()
    ch._check(lib.ctox_hip_gdn_fused_device(
        hip.handle, L.d["proj"].data_ptr(), L.stride, L.C, L.C + 48, L.d["w"].data_ptr(), conv.data_ptr(), conv2.data_ptr(), 4,
        L.d["a"].data_ptr(), L.d["dt"].data_ptr(), ld.data_ptr(), beta.data_ptr(), 0, state.data_ptr(), 5, 48, 16, 128, 128,
        out.data_ptr(), stream()))
    assert (out - L.d["out"]).abs().max() <= 1024 * E * out.abs().max().clamp(min=1)
    assert (state.flatten() - L.d["state2"].flatten()).abs().max() <= 1024 * E
    assert torch.equal(conv2.flatten(), L.d["win2"].flatten())


def test_strong_decays(hip):
    """Decays down to 0 in front of others: differences of their sums stay exact."""
    for decay, seed in ((30.0, 1), (1e4, 2)):
        Layer(seed, [64, 20], chain=0.9, decay=decay).check(hip)
    L = Layer(3, [40], chain=0.8)
    L.proj[5, L.C:L.C + L.H] = 3e38  # a decay of exactly 0 at one node
    with np.errstate(over="ignore"):
        L.check(hip)


def test_repeated_keys_and_forests(hip):
    """The same token again and again, and nodes whose parents are none."""
    L = Layer(4, [64], chain=1.0)
    L.proj[:] = L.proj[0]
    L.check(hip)
    p = [[-1, 0, -1, 2, 2, 9, 4, 6, 7, -1, 9]]
    Layer(6, [11], parents=p).check(hip)


def test_a_node_that_is_no_number_stays_with_its_descendants(hip):
    for n, blocked in ((12, False), (30, True), (64, False)):
        L = Layer(n, [n, 7], chain=0.2, blocked=blocked)
        bad = 3
        L.proj[bad, :L.C] = np.nan
        below = [i for i, line in enumerate(lines(L.forest[0])) if bad in line]
        path = next(x for x in reversed(lines(L.forest[0])) if bad not in x)
        L.kept[0] = path
        op = L.op(hip)
        hip.gdn_tree_device(op, stream())
        hip.gdn_tree_commit_device(op, stream())
        got = L.d["out"].cpu().numpy()[:L.M]
        want, after, _ = L.expect()
        assert np.isnan(got[below]).all()
        rest = [i for i in range(L.M) if i not in below]
        assert np.linalg.norm(got[rest] - want[rest], axis=-1).max() <= 512 * E * 8
        assert np.isfinite(L.d["state2"].cpu().numpy()).all()


def test_paths_that_name_no_nodes(hip):
    """Counts of 0 and of an ended request leave state and windows; a path ends at the first entry that is no node."""
    L = Layer(8, [9, 9, 9, 0], chain=0.5)
    L.kept = [[], [0, 1], lines(L.forest[2])[-1], []]
    op = L.op(hip)
    hip.gdn_tree_device(op, stream())
    counts, path = host(L.d["counts"]).copy(), host(L.d["path"]).copy()
    counts[:2] = [NO, 4]
    path[9:13] = [0, 1, 9, 2]
    L.forest[1][1] = 0
    L.d["counts"].copy_(dev(counts))
    L.d["path"].copy_(dev(path))
    hip.gdn_tree_commit_device(op, stream())
    L.compare()


def test_graph_of_both_calls(hip):
    L = Layer(9, [20, 40], 24, 8, blocked=True)
    op = L.op(hip)
    hip.gdn_tree_device(op, stream())
    hip.gdn_tree_commit_device(op, stream())
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        hip.gdn_tree_device(op, stream())
        hip.gdn_tree_commit_device(op, stream())
    for i in range(3):
        L.proj = (np.random.default_rng(i).standard_normal(L.proj.shape)).astype(np.float32)
        L.d["proj"].copy_(dev(L.proj))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        L.compare()


def test_workspace_is_checked(hip):
    L = Layer(10, [5])
    op = L.op(hip)
    op.bind_workspace(L.ws.data_ptr(), 16)
    for call in (hip.gdn_tree_device, hip.gdn_tree_commit_device):
        with pytest.raises(ch.MemoryBudget):
            call(op, stream())


@pytest.mark.parametrize("max_rows,nodes,over", [(0, [5, 70, 64, 20], [1]), (64, [65, 1], [0]), (16, [16, 17, 3, 40], [1, 3]),
                                                 (20, [32, 33, 7], [1]), (12, [12, 16, 64], [2])])
@pytest.mark.parametrize("batch", [False, True])
def test_more_nodes_than_the_bound(hip, max_rows, nodes, over, batch):
    """Requests past the bound (rounded up to 16, 32 or 64) are no trees of the call: rows of zeros, windows and
    states as they were; the others stand."""
    say("delta", max_rows, nodes, batch)
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    count = -(-cus // (6 * len(nodes))) if batch else 1  # (128 value columns a workgroup from a head a CU on)
    L = Layer(max_rows + 3, nodes * count, chain=0.5, blocked=batch)
    over = [r for r in range(len(L.nodes)) if r % len(nodes) in over]
    for r in over:  # paths that run into the rows past the bound
        L.kept[r] = max(lines(L.forest[r]), key=lambda x: x[-1])
    op = L.op(hip, max_rows=max_rows)
    hip.gdn_tree_device(op, stream())
    hip.gdn_tree_commit_device(op, stream())
    out, after, slid = L.expect()
    got, state = L.d["out"].cpu().numpy(), L.d["state2"].cpu().numpy()
    before = block(L.state) if L.blocked else L.state
    after = block(after) if L.blocked else after
    for r, n in enumerate(L.nodes):
        a = int(L.starts[r])
        windows = L.d["win2"].cpu().numpy()[r].reshape(slid[r].shape)
        if r in over:
            assert not got[a:a + n].any(), r
            assert np.array_equal(state[r], before[r].reshape(-1)) and np.array_equal(windows, L.windows[r]), r
            continue
        big = max(np.abs(L.state[r]).max() * 4, np.linalg.norm(out[a:a + n], axis=-1).max(), 1.0)
        assert np.linalg.norm(got[a:a + n] - out[a:a + n], axis=-1).max() <= 512 * E * big, r
        assert np.abs(state[r] - after[r].reshape(-1)).max() <= 512 * E * max(1.0, np.abs(after[r]).max()), r
        assert np.array_equal(windows, slid[r].astype(np.float32)), r


@pytest.mark.parametrize("heads,key_heads,dk,dv", [(2, 2, 17, 130), (3, 1, 96, 80), (6, 2, 64, 128), (4, 2, 128, 65)])
@pytest.mark.parametrize("K", [1, 3, 4, 5, 8])
@pytest.mark.parametrize("most", [16, 32, 64])
def test_shapes_of_batches(hip, heads, key_heads, dk, dv, K, most):
    """Enough heads that a workgroup takes 128 value columns: part-filled groups of them, short keys, all convolutions,
    both orders of the state."""
    say("delta", heads, key_heads, dk, dv, K, most)
    R = -(-torch.cuda.get_device_properties(0).multi_processor_count // heads)
    assert dv > 64  # (with fewer columns it takes 64 whatever the batch)
    rng = np.random.default_rng(most + K)
    nodes = [int(x) for x in rng.integers(0, 12, R)]
    nodes[0], nodes[R // 2], nodes[-1] = most, most - 1, most // 2 + 1
    for blocked in (False, True):
        Layer(dk + K, nodes, heads, key_heads, dk, dv, K, blocked, chain=0.6, pad=1).check(hip, max_rows=most, gap=8 if blocked else 0)
