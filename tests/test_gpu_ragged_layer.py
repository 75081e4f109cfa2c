"""An attention layer's run over ragged batches, with the operators as they are used together.

Fused q/gate|k|v projection, per-head norm and rotary positions, page plan,
append to the Q4 pool, attention over the mixed pages, the heads' gates, output
projection with its residual. Every operator is held to its own bound, in float64
from what the device gave it; the gate is values / (1 + exp(-g)): the exponent's
argument (|g| 2^-24), exp and quotient (2 ulps each), sum and product, at most
(|g| + 10) 2^-24 of the result.
"""
import math

import numpy as np
import pytest
import torch

import test_gpu_paged_attention_rows as attention
import test_gpu_ragged_ops as ragged
import test_gpu_rows_matmul as matmul
from oracle import paged_kv as pk

pytestmark = pytest.mark.gpu

H, KV, HD, HIDDEN = 10, 2, 256, 448
WIDE = 2 * H * HD + 2 * KV * HD            # [head][q | gate], k, v
CV, BLOCKS = KV * HD, 2 * KV * HD // 64
T4, T2 = BLOCKS * 34, BLOCKS * 18
THETA, EPS, RD, AXES = 1e7, 1e-6, 64, 3


def say(*a):
    print(*a, flush=True)


class Layer:
    """Weights, cache and buffers of one layer for batches of R requests and at most `most` rows."""

    def __init__(self, hip, seed, R, most, page=16, max_pages=12):
        import ctox_hip as ch
        self.hip, self.R, self.most, self.page, self.max_pages = hip, R, most, page, max_pages
        rng = self.rng = np.random.default_rng(seed)
        self.wide, self.wide64 = matmul.build(hip, rng, [1, 0, 1], [2 * H * HD, CV, CV], HIDDEN)
        self.down, self.down64 = matmul.build(hip, rng, [1], [HIDDEN], H * HD, s_in=False, s_out=False)
        slots = R * max_pages
        self.q4_slots = slots
        self.free = [int(x) for x in rng.permutation(slots)]
        self.desc = np.zeros((R, max_pages, 4), np.int64)
        self.cached = np.zeros(R, np.int64)
        self.plan = ragged.Plan([0] * R, [0] * R, page, max_pages, self.free, most, slots, self.desc)
        self.plan.t["positions"].zero_()
        z = lambda *s, t=torch.float32: torch.zeros(s, dtype=t, device="cuda")
        self.q4, self.q2 = z(slots * page * T4, t=torch.uint8), z(slots * page * T2, t=torch.uint8)
        self.q2_next = 0
        self.x, self.y, self.proj = z(most, HIDDEN), z(most, HIDDEN), z(most, WIDE)
        self.q, self.k, self.raw, self.out = z(most, H, HD), z(most, KV, HD), z(most, H, HD), z(most, H, HD)
        self.pos = z(most, AXES, t=torch.int32)
        self.wq, self.wk = (rng.standard_normal((2, HD)) * 0.2).astype(np.float32)
        self.dwq, self.dwk = ragged.dev(self.wq), ragged.dev(self.wk)
        self.axis = [i % AXES for i in range(RD // 2)]
        starts = self.plan.t["row_starts"].data_ptr()
        p = self.proj.data_ptr()
        self.rope = ch.RopeAxes(d_q=p, d_k=p + 4 * 2 * H * HD, d_positions=self.pos.data_ptr(), rows=most, q_heads=H,
                                k_heads=KV, head_dim=HD, rotary_dim=RD, theta=THETA, eps=EPS, axes=AXES,
                                axis_of_pair=self.axis, q_strides=(WIDE, 2 * HD), k_strides=(WIDE, HD),
                                d_q_out=self.q.data_ptr(), d_k_out=self.k.data_ptr(), d_q_norm=self.dwq.data_ptr(),
                                d_k_norm=self.dwk.data_ptr(), d_row_count=starts + 4 * R)
        params = ch.PagedGqaParams(H, KV, HD, 0, page, max_pages, 2 * CV, T2, T4, page * T2, page * T4, 1 / math.sqrt(HD))
        self.att = ch.PagedGqaRows(self.q.data_ptr(), self.raw.data_ptr(), self.q2.data_ptr(), self.q4.data_ptr(),
                                   self.plan.t["descriptors"].data_ptr(), starts, self.plan.t["tokens"].data_ptr(), most,
                                   R, params, most)
        n = hip.paged_gqa_rows_workspace(self.att)
        self.ws = z(n, t=torch.uint8)
        self.att.bind_workspace(self.ws.data_ptr(), n)
        n = max(self.wide.rows_workspace(most), self.down.rows_workspace(most))
        self.mws = z(n, t=torch.uint8)

    def step(self):
        """The layer on the current stream; nothing here knows the batch's lengths."""
        from ctox_hip import _check, load_library
        hip, s, most = self.hip, torch.cuda.current_stream().cuda_stream, self.most
        ws = (self.mws.data_ptr(), self.mws.numel())
        hip.paged_plan_device(self.plan.op, s)
        self.wide.dispatch_rows(self.x.data_ptr(), most, self.proj.data_ptr(), *ws, stream=s)
        torch.mul(self.plan.t["positions"][:most, None], torch.arange(1, AXES + 1, device="cuda", dtype=torch.int32)
                  if self.mult is None else self.mult, out=self.pos)
        hip.rope_axes_device(self.rope, s)
        hip.kv_append_q4_device(self.q4.data_ptr(), self.k.data_ptr(), self.proj.data_ptr() + 4 * (WIDE - CV),
                                self.plan.t["slots"].data_ptr(), most, CV, self.page, self.q4_slots, self.page * T4,
                                key_stride=CV, value_stride=WIDE, stream=s)
        self.raw.zero_()
        hip.paged_gqa_rows_device(self.att, s)
        torch.add(self.raw, 0.0, out=self.out)
        _check(load_library().ctox_hip_attention_gate_device(hip.handle, self.out.data_ptr(), self.proj.data_ptr(), most, H,
                                                             HD, WIDE, s))
        self.down.dispatch_rows(self.out.data_ptr(), most, self.y.data_ptr(), *ws, d_residual=self.x.data_ptr(), stream=s)

    mult = None

    def load(self, added, x):
        """A step's inputs."""
        t = self.plan.t
        self.added = np.array(added)
        t["cached"].copy_(ragged.dev(self.cached.astype(np.int32)))
        t["added"].copy_(ragged.dev(self.added.astype(np.int32)))
        free = self.free + [self.q4_slots] * (self.q4_slots - len(self.free))
        t["free_slots"].copy_(ragged.dev(np.array(free, np.int32)))
        t["descriptors"].copy_(ragged.dev(self.desc.astype(np.int32)))
        self.x.copy_(ragged.dev(x))

    def rows(self):
        return self.rng.standard_normal((self.most, HIDDEN)).astype(np.float32)

    def get(self, n):
        return getattr(self, n).cpu().numpy()

    def check(self):
        """Every operator of the step just run against float64; then the host's books."""
        n = int(self.added.sum())
        want = ragged.plan_ref(self.cached.tolist(), self.added.tolist(), self.desc, self.free, self.page, self.max_pages,
                               self.most, self.q4_slots)
        starts, positions, slots, _, desc, need = want
        assert self.plan.get("status")[0] == 0 and self.plan.get("slots")[:n].tolist() == slots
        assert (self.plan.get("descriptors").reshape(desc.shape) == desc).all()
        x, proj = self.get("x"), self.get("proj")
        matmul.check(proj, *matmul.expect(self.wide64, x, None), False)
        # rotary positions
        pos = np.array(positions)[:, None] * np.arange(1, AXES + 1)
        q = proj[:n, :2 * H * HD].reshape(n, H, 2 * HD)
        k = proj[:n, 2 * H * HD:2 * H * HD + CV].reshape(n, KV, HD)
        for got, src, w in ((self.get("q"), q[..., :HD], self.wq), (self.get("k"), k, self.wk)):
            y, mag = ragged.rope64(src.astype(np.float64), w.astype(np.float64), pos.astype(np.float64),
                                   np.array(self.axis), RD, THETA, EPS)
            assert (np.abs(got[:n] - y) <= 26 * 2.0 ** -24 * mag).all()
        # appended bytes
        pool = self.get("q4").reshape(self.q4_slots, self.page, T4)
        kk, v = self.get("k").reshape(-1, CV), proj[:, WIDE - CV:]
        for t, s in enumerate(slots):
            row = pk.quantize_values(np.concatenate([kk[t], v[t]]), pk.Q4)
            assert pool[s // self.page, s % self.page].tobytes() == row, t
        # attention over what the pools hold
        b = attention.Batch.__new__(attention.Batch)
        b.requests, b.page, b.H, b.KV = list(zip(self.cached.tolist(), self.added.tolist())), self.page, H, KV
        b.n, b.tokens, b.blocks, b.max_pages = self.added.tolist(), (self.cached + self.added).tolist(), BLOCKS, self.max_pages
        b.pool = {1: pool.reshape(*pool.shape[:2], BLOCKS, 34),
                  0: self.get("q2").reshape(self.q4_slots, self.page, BLOCKS, 18)}
        b.desc, b.q, b.M, b.starts = desc, self.get("q"), n, np.array(starts)
        y, tol = b.expect()
        raw = self.get("raw")
        assert (np.abs(raw[:n] - y) <= tol).all() and (raw[n:] == 0).all()
        # gates, output projection
        g = proj[:, :2 * H * HD].reshape(-1, H, 2 * HD)[..., HD:].astype(np.float64)
        y = raw / (1.0 + np.exp(-g))
        out = self.get("out")
        assert (np.abs(out - y) <= (np.abs(g) + 10) * 2.0 ** -24 * np.abs(y) + 2.0 ** -140).all()
        matmul.check(self.get("y"), *matmul.expect(self.down64, out.reshape(self.most, -1), x), False)
        self.desc, self.free, self.cached = desc, self.free[need:], self.cached + self.added

    def demote(self, r, page):
        """A full page of request r to two bits."""
        kind, slot, tokens, _ = (int(v) for v in self.desc[r, page])
        assert kind == 1 and tokens == self.page
        self.hip.kv_demote_device(self.q4.data_ptr() + slot * self.page * T4,
                                  self.q2.data_ptr() + self.q2_next * self.page * T2, tokens, BLOCKS)
        torch.cuda.synchronize()
        self.desc[r, page, :2] = (0, self.q2_next)
        self.q2_next += 1
        self.free.append(slot)


BATCHES = [[40, 0, 17, 1, 0], [1, 30, 1, 0, 0], [1, 1, 1, 1, 1], [0, 61, 15, 16, 3], [0, 0, 0, 0, 0], [70, 1, 1, 1, 12]]


def test_prompts_chunks_and_single_tokens(hip):
    """Prompts, chunks behind them, single tokens and requests that add nothing, with pages demoted between."""
    say("case layer steps")
    m = Layer(hip, 3, 5, 97)
    for i, added in enumerate(BATCHES):
        m.load(added, m.rows())
        m.step()
        torch.cuda.synchronize()
        m.check()
        if i == 1:
            m.demote(0, 0)
            m.demote(2, 0)
        if i == 3:
            m.demote(1, 2)


def test_captured_once_for_all_lengths(hip):
    """One captured step replays every batch, with eager work between, and gives the eager bits."""
    say("case layer graph")
    m = Layer(hip, 4, 5, 97)
    m.mult = torch.arange(1, AXES + 1, device="cuda", dtype=torch.int32)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    m.load(BATCHES[0], m.rows())
    torch.cuda.synchronize()
    # The gate is one of the entry points that wait for the device when the stream differs from the last call's, so
    # the capturing stream has to have been the last one.
    with torch.cuda.stream(side):
        m.step()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        m.step()
    for i, added in enumerate(BATCHES):
        x, pool = m.rows(), m.q4.clone()
        both = []
        for how in (graph.replay, m.step):
            m.q4.copy_(pool)
            m.load(added, x)
            for t in (m.proj, m.q, m.k, m.raw, m.out, m.y):
                t.fill_(3.0)
            torch.cuda.synchronize()
            how()
            torch.cuda.synchronize()
            n = sum(added)
            both.append([t.clone() for t in (m.proj, m.q[:n], m.k[:n], m.raw, m.out, m.y, m.q4)])
        for a, b in zip(*both):
            assert torch.equal(a, b)
        m.check()
        if i == 1:
            m.demote(0, 1)


def test_two_layers_on_two_streams(hip):
    """Layers with buffers of their own run at the same time on streams of their own."""
    say("case layer streams")
    layers = [Layer(hip, 5, 5, 97), Layer(hip, 6, 5, 97)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for added in BATCHES[:3]:
        for m, add in zip(layers, (added, added[::-1])):
            m.load(add, m.rows())
        torch.cuda.synchronize()
        for m, s in zip(layers, streams):
            with torch.cuda.stream(s):
                m.step()
        torch.cuda.synchronize()
        for m in layers:
            m.check()
