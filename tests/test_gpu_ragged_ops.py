"""GPU parity of the ragged batch's rotary positions, page plan and K/V append.

* Rotary positions against the formula in float64. Tolerance: an output is
  a cos - b sin of two normed values. Norm: a sum of squares of up to 1024
  terms in a tree of at most 16 levels and 4 serial steps, halved by the root,
  then three products, a quotient and a root (16 half ulps); sincospif within
  2 ulps each (4 halves), the product and the sum (2): 22 half ulps, plus
  the turn's rounding to 32 bits, 2 pi 2^-25 <= 4 half ulps: 26 half ulps
  (2^-24) of |a| + |b|.
* The plan and the appended bytes are whole numbers: equal.
"""
import math

import numpy as np
import pytest
import torch

from oracle import paged_kv as pk

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


# ---------------------------------------------------------------- rope
def rope64(x, w, pos, axis, rd, theta, eps):
    """x [rows][heads][hd] float64 -> (expected, |a| + |b| of every output)."""
    hd, half = x.shape[-1], rd // 2
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * (1.0 + w)
    ang = pos[:, axis] * theta ** (-2.0 * np.arange(half) / rd)
    c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
    y, m = x.copy(), np.abs(x)
    a, b = x[..., :half], x[..., half:rd]
    y[..., :half], y[..., half:rd] = a * c - b * s, b * c + a * s
    m[..., :half] = m[..., half:rd] = np.abs(a) + np.abs(b)
    return y, m


def rope_case(hip, rows, qh, kh, hd, rd, axes, far, norm=True, in_place=False, offset=0, pad=0, heads_first=False,
              count=None):
    import ctox_hip
    rng = np.random.default_rng(rows * 31 + hd + rd + axes)
    theta, eps = 1e7, 1e-6
    row = (2 * qh + kh) * hd + pad
    proj = rng.standard_normal(rows * row + offset).astype(np.float32)
    pos = rng.integers(0, far, (rows, axes)).astype(np.uint32)
    pos[0] = far - 1
    axis = np.array([i % axes for i in range(rd // 2)])
    wq, wk = (rng.standard_normal((2, hd)) * 0.2).astype(np.float32)
    x = proj[offset:].reshape(rows, row)
    q = x[:, :2 * qh * hd].reshape(rows, qh, 2 * hd)[..., :hd].astype(np.float64)
    k = x[:, 2 * qh * hd:(2 * qh + kh) * hd].reshape(rows, kh, hd).astype(np.float64)
    d, dp = dev(proj), dev(pos.view(np.int32))
    dwq, dwk = dev(wq), dev(wk)
    base = d.data_ptr() + 4 * offset
    dcount = dev(np.array([rows if count is None else count], np.int32))
    kw = dict(d_q=base, d_k=base + 4 * 2 * qh * hd, d_positions=dp.data_ptr(), rows=rows, q_heads=qh, k_heads=kh,
              head_dim=hd, rotary_dim=rd, theta=theta, eps=eps, axes=axes, axis_of_pair=axis.tolist(),
              q_strides=(row, 2 * hd), k_strides=(row, hd), d_row_count=dcount.data_ptr())
    if norm:
        kw.update(d_q_norm=dwq.data_ptr(), d_k_norm=dwk.data_ptr())
    if not in_place:
        oq = torch.full((qh, rows, hd) if heads_first else (rows, qh, hd), 7.0, device="cuda")
        ok = torch.full((rows, kh, hd), 7.0, device="cuda")
        kw.update(d_q_out=oq.data_ptr(), d_k_out=ok.data_ptr())
        if heads_first:
            kw.update(q_out_strides=(hd, rows * hd))
    hip.rope_axes_device(ctox_hip.RopeAxes(**kw), torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    if in_place:
        y = d.cpu().numpy()
        rest = np.ones_like(y, bool)
        rest[offset:].reshape(rows, row)[:, :2 * qh * hd].reshape(rows, qh, 2 * hd)[..., :hd] = False
        rest[offset:].reshape(rows, row)[:, 2 * qh * hd:(2 * qh + kh) * hd] = False
        assert np.array_equal(y[rest], proj[rest])  # gates and padding untouched
        y = y[offset:].reshape(rows, row)
        gq = y[:, :2 * qh * hd].reshape(rows, qh, 2 * hd)[..., :hd]
        gk = y[:, 2 * qh * hd:(2 * qh + kh) * hd].reshape(rows, kh, hd)
    else:
        gq = (oq.transpose(0, 1) if heads_first else oq).cpu().numpy()
        gk = ok.cpu().numpy()
    n = rows if count is None else count
    for got, src, w in ((gq, q, wq), (gk, k, wk)):
        want, mag = rope64(src, w.astype(np.float64) if norm else None, pos.astype(np.float64), axis, rd, theta, eps)
        err = np.abs(got[:n] - want[:n])
        assert (err <= 26 * 2.0 ** -24 * mag[:n]).all(), float((err / np.maximum(mag[:n], 1e-30)).max() * 2 ** 24)
        if not in_place:
            assert (got[n:] == 7.0).all()


@pytest.mark.parametrize("rows,qh,kh,hd,rd,axes,far", [
    (1, 24, 4, 256, 64, 1, 1), (1, 24, 4, 256, 64, 3, 2 ** 31 - 1), (7, 24, 4, 256, 64, 3, 262144),
    (513, 3, 1, 256, 256, 4, 100000), (33, 5, 2, 128, 128, 2, 5000), (5, 2, 2, 64, 32, 1, 40),
    (9, 2, 1, 40, 40, 1, 1000),                                # a head of ten lanes
    (6, 2, 1, 100, 30, 3, 1000), (4, 1, 1, 2, 2, 1, 9), (3, 2, 1, 1024, 512, 2, 77), (3, 2, 2, 300, 44, 1, 77),
])
def test_rope_axes_matches_float64(hip, rows, qh, kh, hd, rd, axes, far):
    say(f"case rope rows={rows} heads={qh}/{kh} hd={hd} rd={rd} axes={axes} far={far}")
    rope_case(hip, rows, qh, kh, hd, rd, axes, far)


@pytest.mark.parametrize("kw", [dict(norm=False), dict(in_place=True), dict(in_place=True, norm=False, offset=1),
                                dict(offset=2, pad=3), dict(heads_first=True), dict(count=4), dict(count=0)])
@pytest.mark.parametrize("hd,rd", [(256, 64), (96, 30)])
def test_rope_axes_forms(hip, kw, hd, rd):
    say(f"case rope forms {kw} hd={hd}")
    rope_case(hip, 6, 3, 2, hd, rd, 3, 30000, **kw)


def test_rope_axes_of_one_axis_is_the_partial_rope(hip):
    import ctox_hip
    say("case rope against partial_rope")
    rng = np.random.default_rng(3)
    q0, k0 = rng.standard_normal((5, 6, 256)).astype(np.float32), rng.standard_normal((5, 2, 256)).astype(np.float32)
    qa, ka, qb, kb = dev(q0), dev(k0), dev(q0), dev(k0)
    pos = dev(np.arange(11, 16, dtype=np.int32))
    hip.partial_rope_device(qa.data_ptr(), ka.data_ptr(), 5, 6, 2, 256, 64, 11, 1e4)
    hip.rope_axes_device(ctox_hip.RopeAxes(d_q=qb.data_ptr(), d_k=kb.data_ptr(), d_positions=pos.data_ptr(), rows=5,
                                           q_heads=6, k_heads=2, head_dim=256, rotary_dim=64, theta=1e4))
    torch.cuda.synchronize()
    # The older entry point forms its angle in 32 bits: position 15 * 2^-24 plus its powf.
    for a, b in ((qa, qb), (ka, kb)):
        assert float((a - b).abs().max()) <= 2.0 ** -24 * (15 * 8 + 26) * 2 * float(b.abs().max())


# ---------------------------------------------------------------- plan
def plan_ref(cached, added, desc, free, page, max_pages, max_rows, q4_slots):
    """The bookkeeping of one request after the other."""
    R = len(cached)
    code, need, rows = 0, 0, 0
    for r in range(R):
        total = cached[r] + added[r]
        if total > max_pages * page:
            return 1
        need += -(-total // page) - -(-cached[r] // page)
        rows += added[r]
        if added[r] and cached[r] % page:
            d = desc[r, cached[r] // page]
            if d[0] == 0 or d[3] != cached[r] // page * page or d[1] >= q4_slots:
                code = 4
    if rows > max_rows:
        return 2
    if need > len(free):
        return 3
    if code:
        return code
    if any(s >= q4_slots for s in free[:need]):
        return 5
    desc, take = desc.copy(), iter(free)
    starts, positions, slots, pages = [0], [], [], []
    for r in range(R):
        for pos in range(cached[r], cached[r] + added[r]):
            p = pos // page
            if pos % page == 0:
                desc[r, p] = (1, next(take), 0, pos)
            desc[r, p, 2] = pos % page + 1
            positions.append(pos)
            slots.append(int(desc[r, p, 1]) * page + pos % page)
        starts.append(len(positions))
        pages.append(-(-(cached[r] + added[r]) // page))
    return starts, positions, slots, pages, desc, need


class Plan:
    def __init__(self, cached, added, page, max_pages, free, max_rows, q4_slots, desc):
        import ctox_hip
        R = len(cached)
        self.t = {n: dev(np.array(v, np.int32).reshape(-1)) for n, v in (("cached", cached), ("added", added),
                                                                        ("free_slots", np.array(list(free) or [0])))}
        self.t["descriptors"] = dev(desc.astype(np.int32))
        for n, k in (("row_starts", R + 1), ("tokens", R), ("page_counts", R), ("positions", max(1, max_rows)),
                     ("slots", max(1, max_rows)), ("status", 4)):
            self.t[n] = torch.full((k,), -7, dtype=torch.int32, device="cuda")
        self.op = ctox_hip.PagedPlan(**{f"d_{n}": v.data_ptr() for n, v in self.t.items()}, requests=R,
                                     page_tokens=page, max_pages=max_pages, free_count=len(free), q4_slots=q4_slots,
                                     max_rows=max_rows)

    def get(self, n):
        return self.t[n].cpu().numpy()


def plan_case(hip, cached, added, page, max_pages=None, spare=3, max_rows=None, seed=0, free=None, q4_slots=None,
              break_desc=None):
    rng = np.random.default_rng(seed)
    R = len(cached)
    most = max(-(-(a + n) // page) for a, n in zip(cached, added))
    max_pages = most + 1 if max_pages is None else max_pages
    held = [-(-a // page) for a in cached]
    need = sum(-(-(a + n) // page) - h for a, n, h in zip(cached, added, held))
    perm = rng.permutation(sum(held) + need + spare)
    desc = rng.integers(0, 1000, (R, max_pages, 4))
    at = 0
    for r in range(R):
        for p in range(min(held[r], max_pages)):
            desc[r, p] = (1, perm[at], min(page, cached[r] - p * page), p * page)
            at += 1
    if break_desc:
        break_desc(desc)
    free = perm[at:] if free is None else free
    q4_slots = len(perm) if q4_slots is None else q4_slots
    max_rows = sum(added) + 4 if max_rows is None else max_rows
    p = Plan(cached, added, page, max_pages, free, max_rows, q4_slots, desc)
    want = plan_ref(cached, added, desc, free, page, max_pages, max_rows, q4_slots)
    for again in range(2):  # the same inputs again: the same plan
        hip.paged_plan_device(p.op, torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        check_plan(p, want, cached, added, page, desc, max_rows)
    return p


def check_plan(p, want, cached, added, page, desc, max_rows):
    R = len(cached)
    if isinstance(want, int):
        assert p.get("status")[0] == want
        assert (p.get("status")[1:] == 0).all()
        assert (p.get("row_starts") == 0).all() and (p.get("slots")[:max_rows] == -1).all()
        assert p.get("tokens").tolist() == list(cached) and (p.get("descriptors") == desc).all()
        assert p.get("page_counts").tolist() == [-(-a // page) for a in cached]
        return
    starts, positions, slots, pages, d, need = want
    assert p.get("status").tolist() == [0, need, len(positions), sum(pages)]
    assert p.get("row_starts").tolist() == starts
    assert p.get("tokens").tolist() == [a + n for a, n in zip(cached, added)]
    assert p.get("page_counts").tolist() == pages
    n = len(positions)
    assert p.get("positions")[:n].tolist() == positions and (p.get("positions")[n:] == -7).all()
    assert p.get("slots")[:n].tolist() == slots and (p.get("slots")[n:max_rows] == -1).all()
    assert (p.get("descriptors") == d).all()


@pytest.mark.parametrize("cached,added,page", [
    ([0], [1], 16), ([0], [0], 16), ([15, 16, 17], [1, 1, 1], 16), ([5, 0, 30, 7], [0, 40, 2, 0], 8),
    ([100, 3], [1, 700], 24), ([0, 0, 0], [16, 15, 17], 16), ([1000], [5000], 1), ([31], [1], 128),
])
def test_plan_matches_the_bookkeeping(hip, cached, added, page):
    say(f"case plan cached={cached} added={added} page={page}")
    plan_case(hip, cached, added, page)


@pytest.mark.parametrize("requests", [63, 511, 513, 1025, 4096])
def test_plan_of_many_requests(hip, requests):
    say(f"case plan requests={requests}")
    rng = np.random.default_rng(requests)
    added = rng.integers(0, 40, requests) * (rng.random(requests) < 0.7)
    plan_case(hip, rng.integers(0, 300, requests).tolist(), added.tolist(), 16, seed=requests)


def broken(word, value):
    def f(desc):
        desc[1, 0, word] = value
    return f


@pytest.mark.parametrize("cached,added,kw", [
    ([16, 5], [30, 10], dict(max_pages=2)), ([16, 5], [30, 10], dict(max_rows=39)),
    ([16, 5], [30, 10], dict(free=[9], q4_slots=40)), ([16, 5], [30, 10], dict(break_desc=broken(0, 0))),
    ([16, 5], [30, 10], dict(break_desc=broken(3, 16))), ([16, 5], [30, 10], dict(break_desc=broken(1, 5000))),
    ([0, 5], [40, 0], dict(free=[0, 1, 2, 3], q4_slots=2)),
])
def test_plan_that_cannot_be_placed(hip, cached, added, kw):
    say(f"case plan refused {sorted(kw)}")
    p = plan_case(hip, cached, added, 16, **kw)
    assert p.get("status")[0] != 0


# ---------------------------------------------------------------- append
def append_case(hip, rows, cv, page, slots, seed=0, key_pad=0, value_pad=0, offset=0, edit=None):
    rng = np.random.default_rng(seed)
    tb = 2 * cv // 64 * 34
    n = 6
    k = (rng.standard_normal((rows, cv + key_pad)) * 2).astype(np.float32)
    v = (rng.standard_normal((rows, cv + value_pad)) * 2).astype(np.float32)
    if edit:
        edit(k, v)
    page_bytes = page * tb + 8
    pool = rng.integers(0, 256, n * page_bytes).astype(np.uint8)
    dk, dv = dev(np.concatenate([np.zeros(offset, np.float32), k.reshape(-1)])), dev(v)
    dp, ds = dev(pool), dev(np.array(slots, np.uint32).view(np.int32))
    hip.kv_append_q4_device(dp.data_ptr(), dk.data_ptr() + 4 * offset, dv.data_ptr(), ds.data_ptr(), rows, cv, page, n,
                            page_bytes, key_stride=cv + key_pad, value_stride=cv + value_pad,
                            stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    want = pool.copy()
    for t, s in enumerate(slots):
        if s < n * page:
            at = s // page * page_bytes + s % page * tb
            want[at:at + tb] = np.frombuffer(pk.quantize_values(np.concatenate([k[t, :cv], v[t, :cv]]), pk.Q4), np.uint8)
    got = dp.cpu().numpy()
    bad = np.nonzero(got != want)[0]
    assert bad.size == 0, (bad[:8], got[bad[:8]], want[bad[:8]])


def special(k, v):
    k[0, :64] = 0.0
    k[0, 64:128] = 3.25
    v[0, :64] = 1e-30                                          # the f16 scale underflows to zero
    k[1, :64] = 4.0 * ((np.arange(64) % 15 + 0.5 - 7.5) / 7.5)  # rounding ties
    k[1, 0] = 4.0
    v[1, :64] = np.float32(7000.0) * v[1, :64]
    k[2, :64] = np.float32(1e-40)                              # denormal maximum


@pytest.mark.parametrize("rows,cv,page", [(1, 1024, 16), (40, 1024, 16), (40, 256, 24), (40, 64, 7), (40, 192, 16),
                                          (5, 1280, 8), (7, 2048, 16), (3, 4160, 4)])
def test_append_matches_oracle(hip, rows, cv, page):
    say(f"case append rows={rows} cv={cv} page={page}")
    rng = np.random.default_rng(rows + cv)
    slots = rng.permutation(6 * page)[:rows]
    slots = np.concatenate([slots, np.full(rows - len(slots), 0xffffffff)]).astype(np.int64)
    if rows > 4:
        slots[3] = 0xffffffff
        slots[4] = 6 * page  # past the pool
    append_case(hip, rows, cv, page, slots.tolist(), edit=special if rows >= 3 and cv >= 128 else None)


@pytest.mark.parametrize("kw", [dict(key_pad=256, value_pad=4), dict(key_pad=1), dict(offset=1), dict(value_pad=3)])
def test_append_strides_and_alignment(hip, kw):
    say(f"case append {kw}")
    append_case(hip, 9, 256, 8, [40, 3, 17, 0xffffffff, 5, 6, 7, 8, 47], **kw)


# ---------------------------------------------------------------- streams and graphs
def test_plan_append_and_rope_replay_in_a_graph(hip):
    """A captured step replays on new lengths and rows, with other work in between."""
    import ctox_hip
    say("case ragged graph")
    rng = np.random.default_rng(8)
    R, page, max_pages, cv, max_rows = 5, 8, 12, 128, 64
    slots_all = 60
    desc0 = np.zeros((R, max_pages, 4), np.int64)
    free = rng.permutation(slots_all)
    p = Plan([0] * R, [0] * R, page, max_pages, free, max_rows, slots_all, desc0)
    tb = 2 * cv // 64 * 34
    pool = torch.zeros(slots_all * page * tb, dtype=torch.uint8, device="cuda")
    k, v = torch.zeros(max_rows, cv, device="cuda"), torch.zeros(max_rows, cv, device="cuda")
    pos = p.t["positions"]
    pos.zero_()
    rope = ctox_hip.RopeAxes(d_q=k.data_ptr(), d_positions=pos.data_ptr(), rows=max_rows, q_heads=1, head_dim=cv,
                             rotary_dim=32, theta=1e4, d_row_count=p.t["row_starts"].data_ptr() + 4 * R)

    def step(stream):
        hip.paged_plan_device(p.op, stream)
        hip.rope_axes_device(rope, stream)
        hip.kv_append_q4_device(pool.data_ptr(), k.data_ptr(), v.data_ptr(), p.t["slots"].data_ptr(), max_rows, cv,
                                page, slots_all, page * tb, stream=stream)

    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(torch.cuda.current_stream().cuda_stream)
    for it in range(3):
        added = rng.integers(0, 13, R)
        kk, vv = rng.standard_normal((2, max_rows, cv)).astype(np.float32)
        out = []
        for how in ("graph", "eager"):
            p.t["cached"].zero_()
            p.t["added"].copy_(dev(added.astype(np.int32)))
            p.t["descriptors"].zero_()
            pool.zero_()
            k.copy_(dev(kk))
            v.copy_(dev(vv))
            torch.cuda.synchronize()
            if how == "graph":
                graph.replay()
            else:
                step(torch.cuda.current_stream().cuda_stream)
            torch.cuda.synchronize()
            out.append([t.clone() for t in (pool, k, p.t["slots"], p.t["row_starts"], p.t["descriptors"])])
        for a, b in zip(*out):
            assert torch.equal(a, b)
        assert int(out[0][3][-1]) == int(added.sum()) and bool(out[0][0].any())
        n = int(added.sum())
        assert torch.equal(out[0][1][n:], dev(kk)[n:])  # rows behind the last request


def test_append_past_four_gibibytes(hip):
    """A slot at the far end of a pool of more than 2^32 bytes."""
    say("case append far slot")
    rng = np.random.default_rng(12)
    cv, page = 256, 16
    tb = 2 * cv // 64 * 34
    slots = 2 ** 32 // (page * tb) + 4
    k, v = rng.standard_normal((2, 2, cv)).astype(np.float32)
    dk, dv = dev(k), dev(v)
    pool = torch.empty(slots * page * tb, dtype=torch.uint8, device="cuda")
    pool[:2 * page * tb] = 9
    pool[-2 * page * tb:] = 9
    ds = dev(np.array([slots * page - 1, slots * page - page], np.uint32).view(np.int32))
    hip.kv_append_q4_device(pool.data_ptr(), dk.data_ptr(), dv.data_ptr(), ds.data_ptr(), 2, cv, page, slots, page * tb,
                            stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert bool((pool[:2 * page * tb] == 9).all())
    want = np.full((2 * page, tb), 9, np.uint8)
    for t, at in ((0, 2 * page - 1), (1, page)):
        want[at] = np.frombuffer(pk.quantize_values(np.concatenate([k[t], v[t]]), pk.Q4), np.uint8)
    assert np.array_equal(pool[-2 * page * tb:].cpu().numpy().reshape(2 * page, tb), want)


@pytest.mark.parametrize("hd,rd", [(256, 64), (96, 30)])
def test_rope_axes_of_keys_alone(hip, hd, rd):
    import ctox_hip
    say(f"case rope keys alone hd={hd}")
    rng = np.random.default_rng(hd)
    x = rng.standard_normal((11, 3, hd)).astype(np.float32)
    pos = rng.integers(0, 5000, (11, 1)).astype(np.uint32)
    dx, dp = dev(x), dev(pos.view(np.int32))
    hip.rope_axes_device(ctox_hip.RopeAxes(d_q=None, d_k=dx.data_ptr(), d_positions=dp.data_ptr(), rows=11, q_heads=0,
                                           k_heads=3, head_dim=hd, rotary_dim=rd, theta=1e4),
                         torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    want, mag = rope64(x.astype(np.float64), None, pos.astype(np.float64), np.zeros(rd // 2, int), rd, 1e4, 1e-6)
    assert (np.abs(dx.cpu().numpy() - want) <= 26 * 2.0 ** -24 * mag).all()
