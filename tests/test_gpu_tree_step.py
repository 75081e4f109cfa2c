"""Decode steps with trees of drafted tokens, the operators run together as a serving program runs them.

A small model of one attention and one GatedDeltaNet layer decodes three requests: per step page plan, tree plan,
rotary positions, append, tree attention, gated delta over the tree, logits, verification, commits of both kinds, free
slots; later a request ends and another is forked into its place. A twin decodes the tokens that were
committed one by one (trees of a single node). Queries, keys and values are rows of tables, so that both sides quantize the
same numbers: the caches have to be equal to the byte. What lies behind the attention differs by its roundings:
those of test_gpu_paged_attention_rows.py, below 1e-5 of an output here, through two products and a recurrence of
contractions (factor 20 at most): 2e-4 of the largest value for states and logits.
"""
import math

import numpy as np
import pytest
import torch

import ctox_hip as ch
from test_gpu_tree_ops import dev, host, stream
from tree_model import NO, lines, random_tree

pytestmark = pytest.mark.gpu

V, H, KV, HD, PAGE, PAGES = 50, 6, 1, 256, 4, 30
GH, GKH, DK, DV, K = 4, 2, 64, 64, 4
C, WIDE = 2 * GKH * DK + GH * DV, 2 * GKH * DK + GH * DV + 2 * GH
TOKEN = 2 * KV * HD // 64 * 34
MOST = 3 * 64


def say(*a):
    print(*a, flush=True)


class Model:
    """Weights, and R requests' caches and states with the buffers of a step."""

    def __init__(self, hip, R):
        self.hip, self.R, self.slots = hip, R, R * PAGES
        g = torch.Generator(device="cuda")
        g.manual_seed(5)
        f = lambda *s, std=1.0: torch.randn(*s, device="cuda", generator=g) * std
        self.tq, self.tk, self.tv = f(V, H, HD), f(V, KV, HD), f(V, KV * HD, std=0.7)
        self.tp, self.w1, self.w2 = f(V, WIDE), f(H * HD, WIDE, std=0.03).double(), f(GH * DV, V, std=0.4).double()
        self.conv_w, self.a_log, self.dt = f(C, K, std=0.4), f(GH, std=0.3) - 1, f(GH, std=0.3) - 2
        z = lambda *s, t=torch.int32: torch.zeros(s, dtype=t, device="cuda")
        self.q4, self.q2 = z(self.slots * PAGE, TOKEN, t=torch.uint8), z(PAGE, TOKEN, t=torch.uint8)
        self.desc, self.cached = z(R, PAGES, 4), z(R)
        self.free, self.free_counts = torch.arange(self.slots, dtype=torch.int32, device="cuda"), dev(np.array([self.slots, 0], np.uint32))
        self.windows, self.state = z(R, C, K, t=torch.float32), z(R, GH * DK * DV, t=torch.float32)
        self.b = {n: z(*s, t=t) for n, s, t in (
            ("added", (R,), torch.int32), ("starts", (R + 1,), torch.int32), ("tokens", (R,), torch.int32), ("pages", (R,), torch.int32),
            ("linear", (MOST,), torch.int32), ("slots", (MOST,), torch.int32), ("status", (4,), torch.int32), ("parents", (MOST,), torch.int32),
            ("masks", (MOST,), torch.int64), ("positions", (MOST,), torch.int32), ("depths", (R,), torch.int32),
            ("q", (MOST, H, HD), torch.float32), ("k", (MOST, KV, HD), torch.float32), ("v", (MOST, KV * HD), torch.float32),
            ("att", (MOST, H, HD), torch.float32), ("proj", (MOST, WIDE), torch.float32), ("core", (MOST, GH, DV), torch.float32),
            ("node", (MOST,), torch.int32), ("u", (MOST,), torch.float32), ("s", (R,), torch.float32), ("counts", (R,), torch.int32),
            ("path", (MOST,), torch.int32), ("next", (R,), torch.int32), ("codes", (R,), torch.int32), ("fork", (2,), torch.int32))}

    def p(self, name):
        return self.b[name].data_ptr()

    def bind(self, op, name):
        n = getattr(self.hip, name + "_workspace")(op)
        ws = torch.full((max(16, n),), 255, dtype=torch.uint8, device="cuda")
        op.bind_workspace(ws.data_ptr(), ws.numel())
        return ws

    def step(self, forest, tokens, draft=None, u=None, s=None):
        """One target pass over the trees; returns (paths, next tokens, target logits)."""
        hip, R, b, st = self.hip, self.R, self.b, stream()
        nodes = [len(x) for x in forest]
        M = sum(nodes)
        b["added"].copy_(dev(np.array(nodes, np.uint32)))
        b["parents"][:M] = dev(np.array([p & NO for x in forest for p in x], np.uint32))
        b["node"][:M] = dev(np.array(tokens, np.uint32))
        hip.paged_plan_device(ch.PagedPlan(
            self.cached.data_ptr(), self.p("added"), self.desc.data_ptr(), self.free.data_ptr(), self.p("starts"), self.p("tokens"),
            self.p("pages"), self.p("linear"), self.p("slots"), self.p("status"), requests=R, page_tokens=PAGE, max_pages=PAGES,
            free_count=int(self.free_counts[0]), q4_slots=self.slots, max_rows=MOST), st)
        assert b["status"].tolist()[0] == 0
        hip.tree_plan_device(ch.TreePlan(self.p("starts"), self.p("tokens"), self.p("parents"), self.p("masks"), self.p("positions"),
                                         self.p("depths"), requests=R, rows=MOST), st)
        at = b["node"][:M].long()
        b["q"][:M], b["k"][:M], b["v"][:M] = self.tq[at], self.tk[at], self.tv[at]
        hip.rope_axes_device(ch.RopeAxes(self.p("q"), self.p("positions"), MOST, H, HD, 64, 1e4, d_k=self.p("k"), k_heads=KV,
                                         d_row_count=self.p("starts") + 4 * R), st)
        hip.kv_append_q4_device(self.q4.data_ptr(), self.p("k"), self.p("v"), self.p("slots"), MOST, KV * HD, PAGE, self.slots,
                                PAGE * TOKEN, stream=st)
        params = ch.PagedGqaParams(H, KV, HD, 0, PAGE, PAGES, 2 * KV * HD, TOKEN // 34 * 18, TOKEN, PAGE * (TOKEN // 34 * 18), PAGE * TOKEN,
                                   1 / math.sqrt(HD))
        att = ch.PagedGqaTree(self.p("q"), self.p("att"), self.q2.data_ptr(), self.q4.data_ptr(), self.desc.data_ptr(),
                              self.p("starts"), self.p("tokens"), self.p("masks"), rows=MOST, requests=R, params=params)
        w0 = self.bind(att, "paged_gqa_tree")
        hip.paged_gqa_tree_device(att, st)
        b["proj"][:M] = (self.tp[at] + b["att"][:M].flatten(1).double() @ self.w1).float()
        delta = ch.GdnTree(self.p("proj"), self.conv_w.data_ptr(), self.windows.data_ptr(), self.a_log.data_ptr(), self.dt.data_ptr(),
                           self.state.data_ptr(), self.p("starts"), self.p("parents"), self.p("core"), proj_stride=WIDE, a_off=C,
                           b_off=C + GH, requests=R, rows=MOST, heads=GH, key_heads=GKH, key_dim=DK, value_dim=DV, kernel=K,
                           d_counts=self.p("counts"), d_path=self.p("path"), d_conv_out=self.windows.data_ptr(),
                           d_state_out=self.state.data_ptr())
        w1 = self.bind(delta, "gdn_tree")
        hip.gdn_tree_device(delta, st)
        logits = (b["core"][:M].flatten(1).double() @ self.w2).float()
        if draft is None:  # single nodes: each is kept
            b["counts"].copy_(b["added"])
            b["path"][:M] = 0
        else:
            b["u"][:M], b["s"][:] = dev(u), dev(s)
            ver = ch.VerifyTree(logits.data_ptr(), self.p("node"), self.p("parents"), self.p("starts"), self.p("counts"), self.p("path"),
                                self.p("next"), requests=R, rows=M, vocab=V, max_children=4, temperature=0.8, d_draft=draft.data_ptr(),
                                d_accept_draws=self.p("u"), d_sample_draws=self.p("s"))
            w2 = self.bind(ver, "verify_tree")
            hip.verify_tree_device(ver, st)
        hip.gdn_tree_commit_device(delta, st)
        self.commit()
        counts, path, nxt, starts = (host(b[n]).tolist() for n in ("counts", "path", "next", "starts"))
        return [path[a:a + c] for a, c in zip(starts, counts)], nxt, logits

    def commit(self, rows=MOST):
        geometry = dict(requests=self.R, page_tokens=PAGE, max_pages=PAGES, q4_slots=self.slots)
        new = torch.zeros_like(self.cached)
        self.hip.paged_commit_device(ch.PagedCommit(
            [self.q4.data_ptr()], self.desc.data_ptr(), self.p("starts"), self.p("tokens"), self.p("counts"), self.p("path"),
            new.data_ptr(), self.p("codes"), rows=rows, token_bytes=TOKEN, q4_page_bytes=PAGE * TOKEN, **geometry), stream())
        assert not self.b["codes"].any()
        self.cached = new
        op = ch.PagedFreeSlots(self.desc.data_ptr(), new.data_ptr(), self.free.data_ptr(), None, self.free_counts.data_ptr(),
                               q2_slots=0, **geometry)
        ws = self.bind(op, "paged_free_slots")
        self.hip.paged_free_slots_device(op, stream())
        torch.cuda.synchronize()

    def end_and_fork(self, source, target):
        """Request `target` ends; `source` goes on in its place too."""
        R = self.R
        self.b["starts"].zero_()
        self.b["tokens"].copy_(self.cached)
        self.b["counts"].zero_()
        self.b["counts"][target] = -1
        self.commit()
        pair = dev(np.array([source, target], np.uint32))
        self.hip.paged_fork_device(ch.PagedFork(
            [self.q4.data_ptr()], self.desc.data_ptr(), self.cached.data_ptr(), pair.data_ptr(), pair.data_ptr() + 4, self.free.data_ptr(), self.free_counts.data_ptr(), self.p("fork"),
            requests=R, forks=1, page_tokens=PAGE, max_pages=PAGES, q4_slots=self.slots, token_bytes=TOKEN,
            q4_page_bytes=PAGE * TOKEN), stream())
        assert self.b["fork"].tolist()[0] == 0
        self.windows[target], self.state[target] = self.windows[source], self.state[source]
        self.b["counts"].zero_()
        self.b["tokens"].copy_(self.cached)
        self.commit()  # (the list of free slots, with the fork's page)

    def cache(self, r):
        t = torch.arange(int(self.cached[r]), device="cuda")
        return self.q4[self.desc[r, t // PAGE, 1].long() * PAGE + t % PAGE]


def test_steps_equal_plain_decoding(hip):
    R = 3
    tree, twin = Model(hip, R), Model(hip, R)
    rng = np.random.default_rng(3)
    bigram = (rng.standard_normal((V, V)) * 1.5).astype(np.float32)
    root, sent, accepted = [1, 2, 3], [[], [], []], 0
    for step in range(9):
        say("step", step, host(tree.cached).tolist())
        if step == 6:  # request 0 ends, request 2 goes on twice
            tree.end_and_fork(2, 0)
            twin.end_and_fork(2, 0)
            root[0], sent[0] = root[2], list(sent[2])
        forest = [random_tree(rng, int(n), 4, 0.4) for n in rng.integers(0 if step == 4 else 1, 20, R)]
        tokens, draft = [], []
        for r, parent in enumerate(forest):
            mine = [root[r]] * len(parent)
            for u in range(len(parent)):
                kids = [i for i, p in enumerate(parent) if p == u]
                q = np.exp(bigram[mine[u]].astype(np.float64) / 0.8)
                for i, t in zip(kids, rng.choice(V, len(kids), replace=False, p=q / q.sum())):
                    mine[i] = int(t)
            tokens += mine
            draft += [bigram[t] for t in mine]
        M = len(tokens)
        # (the target's logits lie near the draft's, so that paths are accepted)
        d = dev(np.array(draft, np.float32).reshape(M, V))
        before = [int(x) for x in host(tree.cached)]
        paths, nxt, logits = tree.step(forest, tokens, d, rng.random(M).astype(np.float32), rng.random(R).astype(np.float32))
        base = np.concatenate([[0], np.cumsum([len(x) for x in forest])])
        for r, parent in enumerate(forest):
            assert int(tree.cached[r]) == before[r] + len(paths[r])
            if not parent:
                continue
            assert paths[r] == lines(parent)[paths[r][-1]]  # a path from the root down
            sent[r] += [tokens[base[r] + i] for i in paths[r]]
            accepted += len(paths[r]) - 1
            root[r] = nxt[r]
        # the twin: the committed tokens, one a step
        while any(int(twin.cached[r]) < len(sent[r]) for r in range(R)):
            at = [int(x) for x in host(twin.cached)]
            now = [r for r in range(R) if at[r] < len(sent[r])]
            _, _, last = twin.step([[-1] if r in now else [] for r in range(R)], [sent[r][at[r]] for r in now])
            for i, r in enumerate(now):  # the logits behind the last committed token
                if at[r] + 1 == len(sent[r]) and forest[r]:
                    mine = logits[base[r] + paths[r][-1]]
                    assert (mine - last[i]).abs().max() <= 2e-4 * last[i].abs().max()
        for r in range(R):
            assert torch.equal(tree.cache(r), twin.cache(r))
            assert (tree.state[r] - twin.state[r]).abs().max() <= 2e-4 * max(1.0, float(twin.state[r].abs().max()))
            assert (tree.windows[r] - twin.windows[r]).abs().max() <= 2e-4 * max(1.0, float(twin.windows[r].abs().max()))
    assert accepted
    # the forks share their full pages and hold nothing else together
    shared = int(tree.desc.shape[0])
    live = [[int(tree.desc[r, p, 1]) for p in range(-(-int(tree.cached[r]) // PAGE))] for r in range(shared)]
    free = host(tree.free).tolist()[:int(tree.free_counts[0])]
    assert sorted(set(sum(live, [])) | set(free)) == list(range(tree.slots)) and not set(sum(live, [])) & set(free)
    assert not set(live[1]) & set(live[0] + live[2])
