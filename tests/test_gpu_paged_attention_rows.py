"""GPU parity of the ragged batch's attention over the paged cache.

Against the formula in float64 over the values that the pages stand for.
Tolerance, with e = 2^-24, S = max over visible tokens of scale sum |q k|, and
Y = sum p |v|:
  * a score: the query keeps 21 bits or more (8 e), a 64-dim block is at most 128
    rounded sums, four blocks and the scale 8 more: |ds| <= 144 e S; the
    exponent's argument and 2^x add 4 e max(1, 2 S);
  * a probability is off by a factor within 1 +- 2 |ds| or so, in numerator and
    denominator: 4 (144 e S + 4 e max(1, 2 S));
  * P s_v keeps 21 bits (8 e), a sum over T tokens rounds at most 2 T times (two
    parts), the denominator T times, joins and the end 64 times.
So |out - exact| <= Y e (4 (144 S + 4 max(1, 2 S)) + 8 + 3 T + 64).
"""
import math

import numpy as np
import pytest
import torch

from oracle import paged_kv as pk

pytestmark = pytest.mark.gpu

Q2, Q4 = 0, 1
BB = {Q2: 18, Q4: 34}
HD = 256


def say(*a):
    print(*a, flush=True)


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


class Batch:
    """Requests (cached, new) with random pages; pages chosen by `q2` lie in the Q2 pool."""

    def __init__(self, seed, requests, page, heads, kv_heads, q2=lambda r, p: False, max_pages=None, pad=0,
                 k_scale=2.4, v_scale=1.5, edit=None):
        rng = np.random.default_rng(seed)
        self.requests, self.page, self.H, self.KV = requests, page, heads, kv_heads
        self.n = [b for _, b in requests]
        self.tokens = [a + b for a, b in requests]
        cv = kv_heads * HD
        self.blocks = 2 * cv // 64
        pages = [-(-t // page) for t in self.tokens]
        self.max_pages = max(1, max(pages)) if max_pages is None else max_pages
        kinds = [[Q2 if q2(r, p) else Q4 for p in range(pages[r])] for r in range(len(requests))]
        self.pool, self.slots = {}, {}
        for kind in (Q2, Q4):
            count = sum(k == kind for ks in kinds for k in ks) + 2
            raw = rng.integers(0, 256, (count, page, self.blocks, BB[kind])).astype(np.uint8)
            s = np.abs(rng.standard_normal(raw.shape[:3])) * 0.3 + 1.0
            s[..., :self.blocks // 2] *= k_scale
            s[..., self.blocks // 2:] *= v_scale
            raw[..., :2] = s.astype(np.float16).view(np.uint8).reshape(*raw.shape[:3], 2)
            self.pool[kind], self.slots[kind] = raw, iter(rng.permutation(count))
        self.desc = np.zeros((len(requests), self.max_pages, 4), np.uint32)
        for r, ks in enumerate(kinds):
            for p, kind in enumerate(ks):
                self.desc[r, p] = (kind, next(self.slots[kind]), min(page, self.tokens[r] - p * page), p * page)
        M = sum(self.n)
        self.M = M
        self.q = rng.standard_normal((M + pad, heads, HD)).astype(np.float32)
        self.starts = np.concatenate([[0], np.cumsum(self.n)]).astype(np.int32)
        if edit:
            edit(self)

    def token_values(self, r):
        """(K, V [tokens][KV][HD] float64, present [tokens]) of request r from its pages."""
        T = self.tokens[r]
        out, present = np.zeros((T, self.blocks * 64)), np.zeros(T, bool)
        for p in range(min(self.max_pages, -(-T // self.page))):
            kind, slot, count, first = (int(x) for x in self.desc[r, p])
            for j in range(p * self.page, min((p + 1) * self.page, T)):
                if first <= j < first + count:
                    present[j] = True
                    raw = self.pool[kind][slot, j - first]
                    out[j] = pk.dequantize_bytes(raw.tobytes(), kind)
        half = self.blocks * 32
        return out[:, :half].reshape(T, self.KV, HD), out[:, half:].reshape(T, self.KV, HD), present

    def expect(self):
        want = np.zeros((self.M, self.H, HD))
        tol = np.zeros((self.M, self.H, HD))
        G, e = self.H // self.KV, 2.0 ** -24
        for r, (cached, n) in enumerate(self.requests):
            if n == 0:
                continue
            K, V, present = self.token_values(r)
            j = np.arange(self.tokens[r])
            for h in range(self.H):
                k, v = K[:, h // G], V[:, h // G]
                for t in range(n):
                    at = self.starts[r] + t
                    see = present & (j <= cached + t)
                    if not see.any():
                        continue
                    q = self.q[at, h].astype(np.float64)
                    s = k[see] @ q / 16.0
                    S = (np.abs(k[see]) @ np.abs(q) / 16.0).max()
                    p = np.exp(s - s.max())
                    p /= p.sum()
                    want[at, h] = p @ v[see]
                    tol[at, h] = (p @ np.abs(v[see])) * e * (4 * (144 * S + 4 * max(1, 2 * S)) + 72 + 3 * see.sum())
        return want, tol

    def op(self, hip, rows=None, max_rows=0, share=None):
        import ctox_hip as ch
        b4, b2 = self.blocks * 34, self.blocks * 18
        if not hasattr(self, "d"):
            self.d = {n: dev(v) for n, v in dict(
                q=self.q, q2=self.pool[Q2].reshape(-1), q4=self.pool[Q4].reshape(-1), desc=self.desc.view(np.int32),
                starts=self.starts, tokens=np.array(self.tokens, np.int32)).items()}
            self.d["out"] = torch.full(self.q.shape, 7.0, device="cuda")
        d = self.d
        params = ch.PagedGqaParams(self.H, self.KV, HD, 0, self.page, self.max_pages, self.blocks * 64, b2, b4,
                                   self.page * b2, self.page * b4, 1.0 / math.sqrt(HD))
        op = ch.PagedGqaRows(d["q"].data_ptr(), d["out"].data_ptr(), d["q2"].data_ptr(), d["q4"].data_ptr(),
                             d["desc"].data_ptr(), d["starts"].data_ptr(), d["tokens"].data_ptr(),
                             self.q.shape[0] if rows is None else rows, len(self.requests), params, max_rows)
        n = hip.paged_gqa_rows_workspace(op)
        self.ws = torch.full((n + 64,), 0xEE, dtype=torch.uint8, device="cuda")
        op.bind_workspace(self.ws.data_ptr(), n)
        return op

    def run(self, hip, **kw):
        op = self.op(hip, **kw)
        hip.paged_gqa_rows_device(op, torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert bool((self.ws[-64:] == 0xEE).all())
        return self.d["out"].cpu().numpy()

    def check(self, got):
        want, tol = self.expect()
        assert (got[self.M:] == 7.0).all()
        err = np.abs(got[:self.M].astype(np.float64) - want)
        bad = ~(err <= tol)
        assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:5].tolist(), float(np.nanmax(err / np.maximum(tol, 1e-30))))


def old(r, p):
    return p % 3 == 1


@pytest.mark.parametrize("heads,kv_heads", [(24, 4), (4, 4), (8, 1), (2, 2)])
@pytest.mark.parametrize("page", [16, 24, 7, 128])
def test_one_request_many_rows(hip, page, heads, kv_heads):
    say(f"case rows attention page={page} heads={heads}/{kv_heads}")
    b = Batch(page + heads, [(150, 43)], page, heads, kv_heads, q2=old)
    b.check(b.run(hip))


@pytest.mark.parametrize("cached,new", [(0, 17), (0, 1), (0, 64), (127, 20), (128, 20), (129, 20), (255, 3), (256, 1),
                                        (0, 300), (1000, 18), (513, 129)])
def test_lengths(hip, cached, new):
    say(f"case rows attention cached={cached} new={new}")
    b = Batch(cached + new, [(cached, new)], 16, 6, 1, q2=lambda r, p: p % 4 == 2 and 16 * p + 16 < cached)
    b.check(b.run(hip))


@pytest.mark.parametrize("page", [16, 24])
def test_ragged_batch(hip, page):
    say(f"case rows attention ragged page={page}")
    b = Batch(5, [(40, 1), (0, 70), (300, 0), (513, 2), (7, 30), (0, 0), (260, 3), (90, 90)], page, 12, 2, q2=old, pad=6)
    b.check(b.run(hip))


@pytest.mark.parametrize("page", [16, 8, 20])
@pytest.mark.parametrize("count", [1, 3, 40])
def test_single_tokens(hip, page, count):
    say(f"case rows attention decode page={page} requests={count}")
    rng = np.random.default_rng(count)
    b = Batch(count + page, [(int(x), 1) for x in rng.integers(0, 700, count)], page, 24, 4, q2=old, pad=2)
    b.check(b.run(hip, max_rows=1))


def test_long_decode_in_several_runs_per_wave(hip):
    """A context whose ranges exceed 64 tiles a wave: descriptors are read again."""
    say("case rows attention long decode")
    b = Batch(3, [(24000, 1)] * 24, 16, 8, 8, q2=lambda r, p: p > 8)
    # the same pages for every request: only the first needs the reference
    b.desc[1:] = b.desc[0]
    b.q[1:] = b.q[0]
    got = b.run(hip, max_rows=1)
    assert (got[1:] == got[0]).all()
    b.requests, b.M, b.n = b.requests[:1], 1, [1]
    b.check(got[:1])


def test_a_join_of_many_parts(hip):
    say("case rows attention split")
    b = Batch(9, [(5000, 40)], 16, 6, 1, q2=lambda r, p: p < 250)
    b.check(b.run(hip))


def test_absent_tokens_and_rows_that_see_nothing(hip):
    say("case rows attention holes")

    def edit(b):
        b.desc[0, 0, 2] = 0                # the first pages are gone: rows 0.. of request 0 see nothing
        b.desc[0, 1, 2] = 0
        b.desc[1, 3, 2] = 5                # a page that holds less than it should
        b.desc[2, 0] = (Q4, 0, 16, 16)     # a page of other tokens
        b.desc[3, :, 2] = 0                # nothing at all, one row
        b.desc[4, :, 2] = 0
    b = Batch(13, [(0, 60), (80, 40), (10, 1), (30, 1), (30, 30)], 16, 6, 1, edit=edit, pad=1)
    got = b.run(hip)
    b.check(got)
    assert (got[:32] == 0).all() and (got[101] == 0).all() and (got[102:132] == 0).all()


def test_what_is_masked_does_not_count(hip):
    """Infinities and NaN in later tokens of the chunk, past the end of the last page and in no page."""
    say("case rows attention non-finite masked")
    for kind in (0x7c00, 0x7e00, 0xfc00):
        def edit(b):
            raw = np.array([kind & 255, kind >> 8], np.uint8)
            last = int(b.desc[0, 6, 1])
            b.pool[Q4][last, 2:, :, :2] = raw        # tokens 98 .. (the chunk's rows 18 ..) and past the end
            b.pool[Q4][last, 2:, :, 2:] = 255
            spare = set(range(b.pool[Q4].shape[0])) - {int(s) for s in b.desc[:, :, 1].reshape(-1)}
            for s in spare:
                b.pool[Q4][s, :, :, :2] = raw
        b = Batch(17, [(80, 22), (37, 1)], 16, 6, 1, edit=edit)
        got = b.run(hip)
        clean = Batch(17, [(80, 22), (37, 1)], 16, 6, 1)
        want, tol = clean.expect()
        keep = np.r_[0:18, 22]
        err = np.abs(got[keep].astype(np.float64) - want[keep])
        assert (err <= tol[keep]).all(), kind


def test_non_finite_queries_stay_in_their_rows(hip):
    say("case rows attention non-finite queries")
    b = Batch(19, [(60, 30), (20, 1)], 16, 4, 2)
    want, tol = b.expect()
    b.q[5, 1, 7], b.q[11, 2, 200], b.q[30, 0, 3] = np.nan, np.inf, np.nan
    got = b.run(hip)
    for r, h in ((5, 1), (11, 2), (30, 0)):
        assert np.isnan(got[r, h]).all()
        got[r, h], want[r, h] = 0, 0
    assert (np.abs(got - want) <= tol).all()


@pytest.mark.parametrize("k_scale,v_scale", [(30.0, 1.0), (1e-3, 1e-4), (2.0, 3000.0)])
def test_peaked_flat_and_scaled(hip, k_scale, v_scale):
    say(f"case rows attention scales {k_scale} {v_scale}")
    b = Batch(23, [(200, 25), (333, 1)], 16, 6, 1, q2=old, k_scale=k_scale, v_scale=v_scale)
    b.check(b.run(hip))


def test_value_scales_that_grow_and_shrink(hip):
    say("case rows attention value scales over six orders")

    def edit(b):
        for kind in (Q2, Q4):
            raw = b.pool[kind]
            rng = np.random.default_rng(kind)
            mag = 10.0 ** rng.uniform(-3, 3, raw.shape[:3])
            raw[..., b.blocks // 2:, :2] = mag[..., b.blocks // 2:].astype(np.float16).view(np.uint8).reshape(
                *raw.shape[:2], b.blocks // 2, 2)
    b = Batch(29, [(700, 25), (300, 2)], 16, 6, 1, q2=old, edit=edit)
    b.check(b.run(hip))


def test_growing_scores_move_the_maximum(hip):
    say("case rows attention growing scores")

    def edit(b):
        s = np.zeros((b.tokens[0],))
        for p in range(-(-b.tokens[0] // b.page)):
            slot = int(b.desc[0, p, 1])
            raw = b.pool[Q4]
            v = np.float16(0.02 * 1.35 ** p)
            raw[slot, :, :b.blocks // 2, :2] = np.array([v]).view(np.uint8)
    b = Batch(31, [(360, 40)], 16, 6, 1, edit=edit)
    b.check(b.run(hip))


def test_agrees_with_the_attention_of_one_sequence(hip):
    import ctox_hip as ch
    say("case rows attention against paged_gqa")
    b = Batch(37, [(500, 5)], 16, 24, 4, q2=old)
    got = b.run(hip)
    b4, b2 = b.blocks * 34, b.blocks * 18
    out = torch.empty(5, 24, HD, device="cuda")
    params = ch.PagedGqaParams(24, 4, HD, 505, 16, b.max_pages, b.blocks * 64, b2, b4, 16 * b2, 16 * b4, 1 / 16.0)
    hip.paged_gqa_device(b.d["q"].data_ptr(), b.d["q2"].data_ptr(), b.d["q4"].data_ptr(), b.d["desc"].data_ptr(), params, 5,
                         out.data_ptr())
    torch.cuda.synchronize()
    _, tol = b.expect()
    assert (np.abs(out.cpu().numpy() - got) <= 2 * tol).all()


def test_repeats_replays_and_other_lengths(hip):
    """One captured call, replayed for batches of other lengths with eager work in between."""
    say("case rows attention graph")
    cases = [[(40, 1), (0, 50), (100, 9)], [(0, 0), (200, 3), (77, 57)], [(10, 20), (30, 20), (250, 20)]]
    first = Batch(41, cases[0], 16, 6, 1, max_pages=20, q2=old)
    hold = first.op(hip, max_rows=60)
    big = {n: torch.zeros(max(v.numel(), 1 << 16), dtype=v.dtype, device="cuda") for n, v in first.d.items()}
    big["q2"] = torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")
    big["q4"] = torch.zeros(1 << 21, dtype=torch.uint8, device="cuda")
    big["q"], big["out"] = (torch.zeros(64 * 6 * HD, device="cuda") for _ in range(2))
    hold.query, hold.out = big["q"].data_ptr(), big["out"].data_ptr()
    hold.q2_pages, hold.q4_pages = big["q2"].data_ptr(), big["q4"].data_ptr()
    hold.descriptors, hold.row_starts, hold.tokens = (big[n].data_ptr() for n in ("desc", "starts", "tokens"))
    hold.rows = 64
    ws = torch.empty(hip.paged_gqa_rows_workspace(hold), dtype=torch.uint8, device="cuda")
    hold.bind_workspace(ws.data_ptr(), ws.numel())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        hip.paged_gqa_rows_device(hold, torch.cuda.current_stream().cuda_stream)
    for seed, c in enumerate(cases):
        b = Batch(seed, c, 16, 6, 1, max_pages=20, q2=old)
        b.op(hip)
        for n in ("q", "q2", "q4", "desc", "starts", "tokens"):
            big[n][:b.d[n].numel()] = b.d[n].reshape(-1)
        outs = []
        for how in ("eager", "replay", "replay"):
            big["out"].fill_(7.0)
            ws.fill_(0xFF)
            torch.cuda.synchronize()
            if how == "eager":
                hip.paged_gqa_rows_device(hold, torch.cuda.current_stream().cuda_stream)
            else:
                graph.replay()
            torch.cuda.synchronize()
            outs.append(big["out"].clone())
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
        b.check(outs[0].cpu().numpy().reshape(64, 6, HD))


def test_refusals_with_a_backend(hip):
    import ctox_hip as ch
    say("case rows attention refusals")
    b = Batch(43, [(20, 20)], 16, 6, 1)
    for kind, edit in ((ch.MemoryBudget, lambda o: o.bind_workspace(o.workspace, o.workspace_bytes - 1)),
                       (ch.MemoryBudget, lambda o: o.bind_workspace(None, o.workspace_bytes)),
                       (ch.MemoryBudget, lambda o: o.bind_workspace(o.workspace + 8, o.workspace_bytes)),
                       (ch.ShapeError, lambda o: setattr(o, "query", o.query + 4)),
                       (ch.ShapeError, lambda o: setattr(o, "out", o.out + 8)),
                       (ch.ShapeError, lambda o: setattr(o, "tokens", None))):
        op = b.op(hip)
        edit(op)
        with pytest.raises(kind):
            hip.paged_gqa_rows_device(op)
    op = b.op(hip, rows=0)
    hip.paged_gqa_rows_device(op)
    torch.cuda.synchronize()
    assert bool((b.d["out"] == 7.0).all())


@pytest.mark.parametrize("heads,kv_heads,most", [(16, 1, 1), (32, 2, 1), (34, 2, 1), (33, 1, 1), (80, 2, 1), (24, 4, 2),
                                                 (24, 4, 3), (2, 1, 8), (2, 1, 9), (6, 6, 16), (6, 6, 17), (5, 1, 6)])
def test_few_queries_at_the_limits(hip, heads, kv_heads, most):
    """Requests of up to `most` rows around 16 and 32 queries a KV head, and groups that reach them alone."""
    say(f"case rows attention few heads={heads}/{kv_heads} most={most}")
    rows = [most, 1, 0, max(1, most - 1), most, 1]
    b = Batch(heads + most, list(zip([0, 31, 40, 333, 1000, 0], rows)), 16, heads, kv_heads, q2=old, pad=3)
    b.check(b.run(hip, max_rows=most))


@pytest.mark.parametrize("most", [1, 5, 40])
def test_pages_past_four_gibibytes(hip, most):
    """Pages at the far end of pools of more than 2^32 bytes."""
    say(f"case rows attention far pages most={most}")
    b = Batch(most, [(200, most), (31, 1)], 16, 12, 2, q2=old)
    op = b.op(hip, max_rows=most)
    pools = {}
    for kind, name in ((Q2, "q2"), (Q4, "q4")):
        near = b.d[name]
        page = 16 * b.blocks * BB[kind]
        skip = (2 ** 32 + 5 * page) // page + 1
        pools[name] = torch.empty(skip * page + near.numel(), dtype=torch.uint8, device="cuda")
        pools[name][skip * page:] = near
        b.desc[..., 1] += np.where((b.desc[..., 0] == kind) & (b.desc[..., 2] > 0), skip, 0).astype(np.uint32)
    b.d["desc"].copy_(dev(b.desc.view(np.int32)))
    op.q2_pages, op.q4_pages = pools["q2"].data_ptr(), pools["q4"].data_ptr()
    hip.paged_gqa_rows_device(op, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    for kind, name in ((Q2, "q2"), (Q4, "q4")):  # (the reference reads the near copies)
        skip = (2 ** 32 + 5 * 16 * b.blocks * BB[kind]) // (16 * b.blocks * BB[kind]) + 1
        b.desc[..., 1] -= np.where((b.desc[..., 0] == kind) & (b.desc[..., 2] > 0), skip, 0).astype(np.uint32)
    b.check(b.d["out"].cpu().numpy())


# (name, heads, KV heads, requests, max_rows): one batch for each of the three kernels
KERNELS = [("128 queries", 6, 1, [(80, 40), (21, 30)], 0), ("32 queries", 6, 1, [(80, 5), (21, 3)], 5),
           ("16 queries", 6, 1, [(80, 2), (21, 1)], 2)]


@pytest.mark.parametrize("name,heads,kv_heads,requests,most", KERNELS)
@pytest.mark.parametrize("holes", [False, True])
def test_queries_below_the_normal_range(hip, name, heads, kv_heads, requests, most, holes):
    """Rows whose largest value is an f32 subnormal, beside ordinary ones, over masked and absent tokens: all
    scores are 0 to within any step, so they get the mean of what they see."""
    say(f"case rows attention subnormal queries {name} holes={holes}")

    def edit(b):
        for i, size in enumerate((1e-42, 1e-39, 3e-45, 1e-37)):
            b.q[i::5] *= np.float32(size)
        if holes:
            b.desc[0, 1, 2] = 0
            b.desc[1, 0, 2] = 5
    b = Batch(47, requests, 16, heads, kv_heads, q2=old, edit=edit, pad=2)
    b.check(b.run(hip, max_rows=most))


def value_scales(b, r, at, scale):
    """V scales of the tokens `at` of request r."""
    for j in at:
        kind, slot, _, first = (int(x) for x in b.desc[r, j // b.page])
        b.pool[kind][slot, j - first, b.blocks // 2:, :2] = np.array([scale], np.float16).view(np.uint8)


def look_at(b, r, token, rows, score):
    """Queries of request r's rows that give `token` about that score (natural units) and others a small one."""
    G = b.H // b.KV
    k, _, _ = b.token_values(r)
    for t in rows:
        for h in range(b.H):
            x = k[token, h // G]
            b.q[b.starts[r] + t, h] = (x * (score * 16.0 / (x @ x))).astype(np.float32)


@pytest.mark.parametrize("name,heads,kv_heads,requests,most", KERNELS)
@pytest.mark.parametrize("large", [1e3, 6e4])
@pytest.mark.parametrize("small", [1e-3, 6e-5])
def test_large_values_out_of_sight(hip, name, heads, kv_heads, requests, most, large, small):
    """The chunk's last token is of a large value scale: rows before it do not see it, and keep their bits."""
    say(f"case rows attention large value masked {name} {large} {small}")

    def edit(b):
        for r, (cached, n) in enumerate(requests):
            value_scales(b, r, range(cached + n), small)
            value_scales(b, r, [cached + n - 1], large)
    b = Batch(53, requests, 16, heads, kv_heads, q2=old, edit=edit)
    b.check(b.run(hip, max_rows=most))


@pytest.mark.parametrize("name,heads,kv_heads,requests,most", KERNELS)
@pytest.mark.parametrize("token,others", [(3, range(4, 120)), (70, range(0, 64)), (3, range(40, 120)), (70, range(64, 70))])
@pytest.mark.parametrize("small,large,score", [(1e-3, 1e3, 16.0), (1e-3, 6e4, 20.0), (6e-5, 6e4, 25.0), (0.0, 1.0, 16.0),
                                               (0.0, 6e-8, 10.0), (3e-7, 6e4, 40.0)])
def test_small_values_of_a_peak(hip, name, heads, kv_heads, requests, most, token, others, small, large, score):
    """Probability 1 - tiny on a token of small (or no) values, tiny ones on tokens of large values: before, behind
    and beside it in its tile, and in later tiles alone."""
    say(f"case rows attention peak {name} {token} {others} {small} {large} {score}")

    def edit(b):
        n = sum(requests[0])
        value_scales(b, 0, range(n), small)
        value_scales(b, 0, [j for j in others if j < n], large)
        look_at(b, 0, token, range(requests[0][1]), score)
    b = Batch(59, requests, 16, heads, kv_heads, q2=old, edit=edit)
    b.check(b.run(hip, max_rows=most))


@pytest.mark.parametrize("name,heads,kv_heads,requests,most", KERNELS)
def test_a_peak_that_comes_late(hip, name, heads, kv_heads, requests, most):
    """Large values first, then a token of small ones whose score is far above: what was summed shrinks to nothing."""
    say(f"case rows attention late peak {name}")

    def edit(b):
        n = sum(requests[0])
        value_scales(b, 0, range(n), 1e-3)
        value_scales(b, 0, range(48), 6e4)
        look_at(b, 0, 66, range(requests[0][1]), 60.0)
    b = Batch(61, requests, 16, heads, kv_heads, q2=old, edit=edit)
    b.check(b.run(hip, max_rows=most))


@pytest.mark.parametrize("heads,kv_heads", [(24, 4), (6, 1), (4, 4), (34, 1), (1024, 512)])
def test_a_workspace_for_many_rows_serves_fewer(hip, heads, kv_heads):
    """Its size does not fall with rows, requests or max_rows."""
    import ctox_hip as ch
    say(f"case rows attention workspace {heads}/{kv_heads}")
    b4, b2 = 2 * kv_heads * 4 * 34, 2 * kv_heads * 4 * 18
    params = ch.PagedGqaParams(heads, kv_heads, HD, 0, 16, 8, 2 * kv_heads * HD, b2, b4, 16 * b2, 16 * b4, 1 / 16.0)

    def size(rows, requests, most):
        return hip.paged_gqa_rows_workspace(ch.PagedGqaRows(*[1 << 16] * 7, rows=rows, requests=requests, params=params,
                                                            max_rows=most))
    rows = [0, 1, 2, 3, 5, 6, 16, 17, 32, 33, 100, 500, 511, 512, 513, 2000, 2700, 2731, 4096, 10923, 100000]
    requests = [1, 2, 3, 32, 511, 512, 513, 4096]
    most = [1, 2, 3, 5, 6, 16, 17, 32, 33, 500, 0]
    got = np.array([[[size(r, q, x) for x in most] for q in requests] for r in rows])
    for axis in range(3):
        assert (np.diff(got, axis=axis) >= 0).all(), axis


def test_one_workspace_for_a_prompt_and_its_chunks(hip):
    say("case rows attention workspace reuse")
    big = Batch(67, [(0, 700)], 16, 4, 4)
    hold = big.op(hip)
    need, ws = hold.workspace_bytes, big.ws
    for requests, most in (([(0, 700)], 0), ([(300, 40)], 0), ([(700, 1)], 1), ([(100, 9)], 9), ([(90, 600)], 0)):
        b = Batch(71, requests, 16, 4, 4, q2=old)
        op = b.op(hip, max_rows=most)
        op.bind_workspace(ws.data_ptr(), need)
        hip.paged_gqa_rows_device(op, torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert bool((ws[-64:] == 0xEE).all())
        b.check(b.d["out"].cpu().numpy())


def check_some(b, got, picks):
    """The rows (request, row, head) of `picks` against float64, all others finite, rows past the end untouched."""
    G, e, last = b.H // b.KV, 2.0 ** -24, None
    assert (got[b.M:] == 7.0).all() and np.isfinite(got[:b.M]).all()
    for r, t, h in sorted(picks):
        if r != last:
            last, (K, V, present) = r, b.token_values(r)
        see = present & (np.arange(b.tokens[r]) <= b.requests[r][0] + t)
        k, v, q = K[see, h // G], V[see, h // G], b.q[b.starts[r] + t, h].astype(np.float64)
        s, S = k @ q / 16.0, (np.abs(k) @ np.abs(q) / 16.0).max()
        p = np.exp(s - s.max())
        p /= p.sum()
        tol = (p @ np.abs(v)) * e * (4 * (144 * S + 4 * max(1, 2 * S)) + 72 + 3 * see.sum())
        assert (np.abs(got[b.starts[r] + t, h] - p @ v) <= tol).all(), (r, t, h)


@pytest.mark.parametrize("count", [65, 257, 300, 512, 513, 1025, 4096])
@pytest.mark.parametrize("kind", ["one row", "few rows", "mixed"])
def test_many_requests(hip, count, kind):
    """More requests than a workgroup's lanes (256 or 512) and than are cut (512), a third of them without rows, one of a
    long context: its token axis is cut up to 512 requests."""
    say(f"case rows attention requests={count} {kind}")
    rng = np.random.default_rng(count)
    most = {"one row": 1, "few rows": 4, "mixed": 40}[kind]
    rows = rng.integers(1, most + 1, count) if kind != "mixed" else np.where(np.arange(count) % 37 == 5, 40, 1)
    rows[rng.permutation(count)[:count // 3]] = 0
    cached = rng.integers(0, 30, count)
    for r in (count - 3, count // 2):
        rows[r], cached[r] = max(1, most), 2500
    b = Batch(count, list(zip(cached.tolist(), rows.tolist())), 16, 6, 1, q2=old, pad=2)
    got = b.run(hip, max_rows=most)
    picks = [(r, t, h) for r in (*rng.permutation(count)[:60].tolist(), 0, count - 3, count // 2, count - 1)
             for t in range(b.n[r]) for h in (0, 5)]
    check_some(b, got, picks)


def test_a_prompt_whose_tiles_fill_the_chip(hip):
    """Two workgroups a CU or more from query tiles alone: token ranges are not cut and nothing is joined."""
    say("case rows attention uncut prompt")
    b = Batch(73, [(30, 2075), (5, 1), (0, 33)], 16, 32, 16, q2=lambda r, p: p % 4 == 1, pad=3)
    got = b.run(hip)
    rng = np.random.default_rng(5)
    picks = [(0, int(t), int(h)) for t in (*range(3), *range(2070, 2075), *rng.integers(0, 2075, 40))
             for h in rng.permutation(32)[:8]]
    check_some(b, got, picks + [(1, 0, h) for h in range(32)] + [(2, t, h) for t in (0, 31, 32) for h in range(32)])


def test_one_prompt_alone_whose_tiles_fill_the_chip(hip):
    say("case rows attention uncut prompt of one request")
    b = Batch(79, [(0, 1100)], 24, 120, 60, q2=lambda r, p: p % 4 == 1)
    got = b.run(hip)
    rng = np.random.default_rng(7)
    check_some(b, got, [(0, int(t), int(h)) for t in (0, 1, 62, 63, 64, 1098, 1099, *rng.integers(0, 1100, 20))
                        for h in rng.permutation(120)[:6]])


@pytest.mark.parametrize("name,heads,kv_heads,requests,most", KERNELS)
@pytest.mark.parametrize("kind", [0x7c00, 0x7e00])
def test_non_finite_values_of_a_hardly_weighted_token(hip, name, heads, kv_heads, requests, most, kind):
    """A probability below f32's range is not 0: the rows that see a token of infinite values get no numbers, the rows
    before it keep theirs."""
    say(f"case rows attention non-finite value {name} {kind:x}")
    n = sum(requests[0])

    def edit(b):
        look_at(b, 0, 3, range(requests[0][1]), 400.0)
        value_scales(b, 0, [n - 1], 0.5)
    clean = Batch(83, requests, 16, heads, kv_heads, q2=old, edit=edit)
    want, tol = clean.expect()
    b = Batch(83, requests, 16, heads, kv_heads, q2=old, edit=edit)
    value_scales(b, 0, [n - 1], np.uint16(kind).view(np.float16))
    got = b.run(hip, max_rows=most)
    last = requests[0][1] - 1
    assert not np.isfinite(got[last]).any()
    keep = [i for i in range(b.M) if i != last]
    assert (np.abs(got[keep] - want[keep]) <= tol[keep]).all()


@pytest.mark.parametrize("name,heads,kv_heads,requests,most", KERNELS)
def test_more_rows_than_tokens_and_rows_in_front(hip, name, heads, kv_heads, requests, most):
    """Requests whose lengths say fewer tokens than rows (the first rows see nothing), or none; rows that lie before the
    first request's are left alone."""
    say(f"case rows attention short {name}")
    n = [r[1] for r in requests]
    b = Batch(89, [(0, n[0]), (0, n[1]), (40, n[1])], 16, heads, kv_heads, q2=old, pad=5)
    op = b.op(hip, max_rows=most)
    short = n[0] // 2
    b.d["tokens"].copy_(dev(np.array([short, 0, b.tokens[2]], np.int32)))
    b.d["starts"].add_(3)
    hip.paged_gqa_rows_device(op, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    got = b.d["out"].cpu().numpy()
    assert (got[:3] == 7.0).all() and (got[b.M + 3:] == 7.0).all()
    got, q = got[3:b.M + 3], b.q[3:b.M + 3].astype(np.float64)
    assert (got[:n[0] - short] == 0).all() and (got[n[0]:n[0] + n[1]] == 0).all()
    G, e = heads // kv_heads, 2.0 ** -24
    for r, first, tokens in ((0, 0, short), (2, n[0] + n[1], b.tokens[2])):
        K, V, _ = b.token_values(r)
        for t in range(max(0, n[r if r == 0 else 1] - tokens), n[r if r == 0 else 1]):
            seen = tokens - n[r if r == 0 else 1] + t + 1
            for h in range(heads):
                k, v, x = K[:seen, h // G], V[:seen, h // G], q[first + t, h]
                s, S = k @ x / 16.0, (np.abs(k) @ np.abs(x) / 16.0).max()
                p = np.exp(s - s.max())
                p /= p.sum()
                tol = (p @ np.abs(v)) * e * (4 * (144 * S + 4 * max(1, 2 * S)) + 72 + 3 * seen)
                assert (np.abs(got[first + t, h] - p @ v) <= tol).all(), (r, t, h)
