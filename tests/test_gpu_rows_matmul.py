"""GPU parity of the packed products for any number of activation rows.

Against the formula in float64 over the same packed blocks. Tolerance of an
f32 result, with A = sum |w| |x s_in| (the magnitude that rounds):
  * x s_in is one rounding (2^-24) and, in two f16 parts, 2^-23 more (lo rounds
    a value below 2^-11 |x| by half its step) plus an absolute 2^-40 of the row's
    largest value X, which weighs at most 2^-40 X sum |w|;
  * a 64-column block's sum: 128 products, at most 128 f32 roundings of partial
    sums (2^-24 each of a value <= the block's share of A): the units add 16 at a time in an
    unspecified order, so all 128 are counted;
  * blocks: one multiply and one add a block, K / 64 <= 272 terms, and at most
    64 partial sums of a split;
  * 1 / L, exponent, bias, s_out: 6 more.
All roundings of one sign would give (2 + 128 + 2 K / 64 + 64 + 6) 2^-24 A; SiLU's
derivative is below 1.1 and its expf and quotient add 6 ulps of the result. An f16
result adds half a step (2^-11 of the value, 2^-25 below the normal range).
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

Q2, Q4 = 0, 1
BYTES = {Q2: 18, Q4: 34}


def say(*a):
    print(*a, flush=True)


def pack(rng, dtype, rows, cols, scale_edit=None):
    w = rng.integers(0, 256, (rows, cols // 64, BYTES[dtype])).astype(np.uint8)
    s = np.abs(rng.standard_normal((rows, cols // 64)) * 0.02).astype(np.float16)
    if scale_edit:
        scale_edit(s)
    w[..., :2] = s.view(np.uint8).reshape(rows, cols // 64, 2)
    return w


def values(w, dtype):
    bits, L = (2, 3) if dtype == Q2 else (4, 15)
    s = w[..., :2].copy().view(np.float16).astype(np.float64)
    c = np.stack([(w[..., 2:] >> (bits * i)) & (2 ** bits - 1) for i in range(8 // bits)], -1)
    return (s * (2.0 * c.reshape(*w.shape[:-1], 64) - L) / L).reshape(w.shape[0], -1)


def build(hip, rng, dtypes, rows_each, cols, s_in=True, s_out=True, bias=False, silu=False, scale_edit=None):
    """A resident matrix of one or several segments, and its float64 weights."""
    import ctox_hip as ch
    parts = [pack(rng, d, r, cols, scale_edit) for d, r in zip(dtypes, rows_each)]
    rows = sum(rows_each)
    segs, at, off = [], 0, 0
    for i, (d, r, p) in enumerate(zip(dtypes, rows_each, parts)):
        segs.append(ch.QuantSegment(i, at, at + r, ch.TensorDType(d), off, p.size))
        at, off = at + r, off + p.size
    si = rng.uniform(0.5, 1.5, cols).astype(np.float16) if s_in else None
    so = rng.uniform(0.5, 1.5, rows).astype(np.float32) if s_out else None
    bi = (rng.standard_normal(rows) * 0.1).astype(np.float32) if bias else None
    mixed = len(dtypes) > 1
    m = hip.prepare(ch.FusedMatVec(
        ch.TensorDType.MixedQ2Q4B64 if mixed else ch.TensorDType(dtypes[0]), np.concatenate([p.reshape(-1) for p in parts]),
        rows, cols, segments=segs if mixed else (), s_in=None if si is None else ch.ScaleSlice.F16Le(si),
        s_out=None if so is None else ch.ScaleSlice.F32(so), bias=bi,
        activation=ch.Activation.Silu if silu else ch.Activation.Identity))
    W = np.concatenate([values(p, d) for p, d in zip(parts, dtypes)])
    return m, dict(W=W, s_in=si, s_out=so, bias=bi, silu=silu)


def expect(d, x, residual):
    """(float64 result, bound of an f32 result's error)."""
    cols = x.shape[1]
    xs = x.astype(np.float64)
    if d["s_in"] is not None:
        xs = xs * d["s_in"].astype(np.float64)
    y = xs @ d["W"].T
    mag = np.abs(xs) @ np.abs(d["W"]).T
    top = np.abs(xs).max(1, keepdims=True) * np.abs(d["W"]).sum(1)
    tol = (2 + 128 + cols // 32 + 64 + 6) * 2.0 ** -24 * mag + 2.0 ** -40 * top
    if d["bias"] is not None:
        y = y + d["bias"]
        tol += 2.0 ** -24 * np.abs(d["bias"])
    if d["s_out"] is not None:
        y, tol = y * d["s_out"], tol * np.abs(d["s_out"])
    if d["silu"]:
        y = y / (1.0 + np.exp(-y))
        tol = 1.1 * tol + 6 * 2.0 ** -23 * np.abs(y)
    if residual is not None:
        y = y + residual.astype(np.float64)
        tol += 2.0 ** -24 * np.abs(y)
    return y, tol


def run(m, x, residual=None, y_half=False, x_pad=0, y_pad=0, r_pad=0, in_place=False, guard=3):
    import ctox_hip as ch
    T = ch.TensorDType
    rows, cols = x.shape
    n = m.rows
    xt = T.F16 if x.dtype == np.float16 else T.F32
    yt, ydt = (T.F16, torch.float16) if y_half else (T.F32, torch.float32)
    dx = torch.full((rows, cols + x_pad), math.nan, dtype=torch.from_numpy(x).dtype, device="cuda")
    dx[:, :cols] = torch.from_numpy(x).cuda()
    y = torch.full((rows + guard, n + y_pad), 7.0, dtype=ydt, device="cuda")
    dr = None
    if residual is not None:
        if in_place:
            y[:rows, :n] = torch.from_numpy(residual).cuda().to(ydt)
            dr = y
        else:
            dr = torch.full((rows, n + r_pad), math.nan, dtype=ydt, device="cuda")
            dr[:, :n] = torch.from_numpy(residual).cuda().to(ydt)
    need = m.rows_workspace(rows, xt)
    ws = torch.full((need + 64,), 0xAA, dtype=torch.uint8, device="cuda")
    m.dispatch_rows(dx.data_ptr(), rows, y.data_ptr(), ws.data_ptr(), need, None if dr is None else dr.data_ptr(), xt, yt,
                    cols + x_pad, n + y_pad, n + y_pad if in_place else n + r_pad,
                    torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    got = y.cpu().numpy()
    assert (got[rows:] == 7.0).all() and (got[:, n:] == 7.0).all()
    assert bool((ws[need:] == 0xAA).all())
    return got[:rows, :n]


def check(got, want, tol, half):
    if half:
        tol = tol + 2.0 ** -11 * np.abs(want) + 2.0 ** -25 + 2.0 ** -11 * tol
    err = np.abs(got.astype(np.float64) - want)
    assert (err <= tol).all(), (float((err / tol).max()), np.argwhere(err > tol)[:4].tolist())


@pytest.mark.parametrize("rows", [1, 2, 16, 31, 32, 33, 64, 65, 96, 129, 300])
@pytest.mark.parametrize("dtype", [Q2, Q4])
def test_rows_match_float64(hip, dtype, rows):
    say(f"case rows product dtype={dtype} rows={rows}")
    rng = np.random.default_rng(rows * 2 + dtype)
    n, cols = (200, 1088) if rows % 2 else (256, 640)
    m, d = build(hip, rng, [dtype], [n], cols)
    x = rng.standard_normal((rows, cols)).astype(np.float32)
    check(run(m, x), *expect(d, x, None), False)


@pytest.mark.parametrize("n,cols", [(1, 64), (15, 64), (17, 128), (127, 960), (129, 1024), (257, 1152), (513, 2112)])
@pytest.mark.parametrize("dtype", [Q2, Q4])
def test_odd_matrix_sizes(hip, dtype, n, cols):
    say(f"case rows product sizes dtype={dtype} n={n} cols={cols}")
    rng = np.random.default_rng(n + cols)
    m, d = build(hip, rng, [dtype], [n], cols, bias=True)
    for rows in (1, 37):
        x = rng.standard_normal((rows, cols)).astype(np.float32)
        check(run(m, x), *expect(d, x, None), False)


@pytest.mark.parametrize("kw", [
    dict(bias=True), dict(silu=True), dict(bias=True, silu=True), dict(s_in=False), dict(s_out=False),
    dict(s_in=False, s_out=False, bias=True),
])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("half", [False, True])
def test_epilogues_and_types(hip, kw, residual, half):
    say(f"case rows product epilogue {kw} residual={residual} half={half}")
    rng = np.random.default_rng(17)
    t = np.float16 if half else np.float32
    for rows, n in ((40, 144), (130, 272)):
        m, d = build(hip, rng, [Q4], [n], 704, **kw)
        x = rng.standard_normal((rows, 704)).astype(t)
        r = rng.standard_normal((rows, n)).astype(t) if residual else None
        check(run(m, x, r, y_half=half), *expect(d, x, r), half)


def test_types_apart_strides_and_residual_in_place(hip):
    say("case rows product strides")
    rng = np.random.default_rng(23)
    m, d = build(hip, rng, [Q2], [200], 320, bias=True)
    x = rng.standard_normal((70, 320)).astype(np.float32)
    xh = x.astype(np.float16)
    r = rng.standard_normal((70, 200)).astype(np.float16)
    check(run(m, x, r, y_half=True, x_pad=5, y_pad=3, r_pad=9), *expect(d, x, r), True)
    check(run(m, xh, r.astype(np.float32), x_pad=1, y_pad=1, r_pad=2), *expect(d, xh, r), False)
    check(run(m, x, r.astype(np.float32), y_pad=7, in_place=True), *expect(d, x, r), False)


def test_mixed_segments(hip):
    say("case rows product mixed segments")
    rng = np.random.default_rng(29)
    for half in (False, True):
        m, d = build(hip, rng, [Q4, Q2, Q4], [64, 37, 150], 384, s_in=not half, bias=True, silu=True)
        for rows in (3, 90):
            x = rng.standard_normal((rows, 384)).astype(np.float16 if half else np.float32)
            r = rng.standard_normal((rows, 251)).astype(x.dtype)
            check(run(m, x, r, y_half=half), *expect(d, x, r), half)


def test_large_shape_with_every_tile_shape(hip):
    """Enough workgroups for the 128 x 256 tiles, and a K split of a long K."""
    say("case rows product large")
    rng = np.random.default_rng(31)
    m, d = build(hip, rng, [Q4], [17408 // 2], 1024)
    x = rng.standard_normal((2050, 1024)).astype(np.float32)
    pick = rng.permutation(2050)[:97]
    got = run(m, x)
    check(got[pick], *expect(d, x[pick], None), False)
    m, d = build(hip, rng, [Q2], [96], 17408)
    x = rng.standard_normal((20, 17408)).astype(np.float32)
    check(run(m, x), *expect(d, x, None), False)


def test_magnitudes(hip):
    """Rows of very different size, a row of zeros, outliers, scales down to f16 subnormals."""
    say("case rows product magnitudes")
    rng = np.random.default_rng(37)

    def edit(s):
        s[0], s[1, 1], s[2] = 0, 6e-8, 60000
    m, d = build(hip, rng, [Q4], [48], 256, scale_edit=edit, s_in=False)
    x = (rng.standard_normal((9, 256)) * 10.0 ** np.array([-42, -38, -30, -6, 0, 3, 12, 30, 0])[:, None]).astype(np.float32)
    x[8] = 0
    x[4, 7] = 1e6
    want, tol = expect(d, x, None)
    tol = tol + 2.0 ** -149 * (np.abs(d["W"]).sum(1) + 1)  # results below f32's normal range
    got = run(m, x)
    check(got, want, tol, False)
    assert (got[:, 0] == 0).all() and (got[8] == 0).all()


def test_non_finite_rows_stay_in_their_rows(hip):
    say("case rows product non-finite")
    rng = np.random.default_rng(41)
    for half in (False, True):
        m, d = build(hip, rng, [Q4], [80], 192, s_in=False)
        x = rng.standard_normal((70, 192)).astype(np.float16 if half else np.float32)
        x[3, 5], x[40, 100], x[69, 191] = np.nan, np.inf, -np.inf
        got = run(m, x, y_half=half)
        bad = [3, 40, 69]
        assert np.isnan(got[3]).all()
        for r, c in ((40, 100), (69, 191)):
            sign = np.sign(x[r, c].astype(np.float64) * d["W"][:, c])
            assert (got[r] == sign * np.inf).all()
        rest = [i for i in range(70) if i not in bad]
        check(got[rest], *expect(d, x[rest], None), half)


def test_agrees_with_the_matvec_of_few_rows(hip):
    say("case rows product against dispatch")
    rng = np.random.default_rng(43)
    m, d = build(hip, rng, [Q4], [160], 1024, bias=True, silu=True)
    x = rng.standard_normal((5, 1024)).astype(np.float32)
    dx, y = torch.from_numpy(x).cuda(), torch.empty(5, 160, device="cuda")
    m.dispatch(dx.data_ptr(), 5, y.data_ptr())
    torch.cuda.synchronize()
    want, tol = expect(d, x, None)
    check(run(m, x), want, tol, False)
    # the matvec keeps 21 bits below a block's largest value: 2^-20 of sum |w| X is its bound
    assert (np.abs(y.cpu().numpy() - want) <= tol + 2.0 ** -20 * np.abs(x).max() * 1.5 * 1.5 * np.abs(d["W"]).sum(1)).all()


def test_repeats_and_graph_replays_are_the_same(hip):
    say("case rows product graph")
    import ctox_hip as ch
    rng = np.random.default_rng(47)
    m, d = build(hip, rng, [Q4], [300], 2048, silu=True)
    rows = 50
    x = torch.zeros(rows, 2048, device="cuda")
    y = torch.zeros(rows, 300, device="cuda")
    ws = torch.empty(m.rows_workspace(rows), dtype=torch.uint8, device="cuda")

    def call():
        m.dispatch_rows(x.data_ptr(), rows, y.data_ptr(), ws.data_ptr(), ws.numel(),
                        stream=torch.cuda.current_stream().cuda_stream)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for it in range(3):
        xn = rng.standard_normal((rows, 2048)).astype(np.float32)
        x.copy_(torch.from_numpy(xn))
        call()
        torch.cuda.synchronize()
        eager = y.clone()
        y.zero_()
        ws.fill_(0xFF)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, eager)
        check(eager.cpu().numpy(), *expect(d, xn, None), False)


def test_refusals_with_a_matrix(hip):
    import ctox_hip as ch
    say("case rows product refusals")
    rng = np.random.default_rng(53)
    m, _ = build(hip, rng, [Q4], [64], 128)
    t = torch.zeros(64 * 128, device="cuda")
    ws = torch.empty(m.rows_workspace(8), dtype=torch.uint8, device="cuda")
    p, w = t.data_ptr(), ws.data_ptr()
    m.dispatch_rows(p, 0, p, 0, 0)  # nothing to do
    for kind, kw in ((ch.MemoryBudget, dict(workspace_bytes=ws.numel() - 1)), (ch.MemoryBudget, dict(d_workspace=w + 4)),
                     (ch.MemoryBudget, dict(d_workspace=None)), (ch.ShapeError, dict(x_stride=127)),
                     (ch.ShapeError, dict(y_stride=63)), (ch.ShapeError, dict(d_residual=p, residual_stride=60)),
                     (ch.ShapeError, dict(d_x=p + 2)), (ch.ShapeError, dict(d_x=None)), (ch.ShapeError, dict(d_y=None)),
                     (ch.ShapeError, dict(d_residual=p + 1)), (ch.ShapeError, dict(d_y=p, d_residual=p, residual_stride=65)),
                     (ch.ShapeError, dict(rows=2 ** 20 + 1)), (ch.UnsupportedDType, dict(x_dtype=0)),
                     (ch.UnsupportedDType, dict(y_dtype=2))):
        args = dict(d_x=p, rows=8, d_y=p + 4096, d_workspace=w, workspace_bytes=ws.numel())
        args.update(kw)
        with pytest.raises(kind):
            m.dispatch_rows(**args)
    other = ch.HipBackend(0)
    m.backend = other
    with pytest.raises(ch.InvalidState):
        m.dispatch_rows(p, 8, p + 4096, w, ws.numel())
    m.backend = hip
    other.close()


@pytest.mark.parametrize("dtypes,n,cols", [([Q4], [16], 5120), ([Q2], [96], 17408), ([Q4], [1500], 4096), ([Q2, Q4], [64, 700], 2048),
                                           ([Q4], [40], 448)])
def test_a_workspace_for_many_rows_serves_fewer(hip, dtypes, n, cols):
    import ctox_hip as ch
    say(f"case rows product workspace {dtypes} {n} {cols}")
    rng = np.random.default_rng(59)
    m, d = build(hip, rng, dtypes, n, cols, s_in=False)
    for xt in (ch.TensorDType.F32, ch.TensorDType.F16):
        sizes = [m.rows_workspace(r, xt) for r in [*range(0, 1100), *range(1100, 20000, 37), *range(20000, 2 ** 20, 9973)]]
        assert all(a <= b for a, b in zip(sizes, sizes[1:]))
    most = 700
    ws = torch.full((m.rows_workspace(most) + 64,), 0xAA, dtype=torch.uint8, device="cuda")
    x = rng.standard_normal((most, cols)).astype(np.float32)
    dx, y = torch.from_numpy(x).cuda(), torch.empty(most, sum(n), device="cuda")
    for rows in (most, 1, 17, 64, 200, 333):
        y.fill_(7.0)
        m.dispatch_rows(dx.data_ptr(), rows, y.data_ptr(), ws.data_ptr(), ws.numel() - 64,
                        stream=torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        check(y[:rows].cpu().numpy(), *expect(d, x[:rows], None), False)
        assert bool((y[rows:] == 7.0).all()) and bool((ws[-64:] == 0xAA).all())


# (rows of x, outputs) of a workgroup's tile, split K or not, parts of an activation -> a call that gets them:
# rows and outputs that leave the last tiles part-filled.
TILED = [((32, 128), False, 1, (33, 72, 128)), ((32, 128), False, 2, (33, 72, 128)), ((32, 128), True, 1, (33, 72, 2112)),
         ((32, 128), True, 2, (33, 72, 2112)), ((64, 128), False, 1, (300, 17000, 128)),
         ((64, 128), False, 2, (300, 17000, 128)), ((64, 128), True, 1, (6000, 72, 17408)),
         ((64, 128), True, 2, (33, 10250, 17408)), ((128, 128), False, 1, (1500, 12300, 192)),
         ((128, 128), False, 2, (1500, 12300, 192)), ((128, 128), True, 1, (4100, 1500, 17408)),
         ((128, 128), True, 2, (9000, 520, 17408)), ((128, 256), False, 1, (4100, 17000, 128)),
         ((128, 256), False, 2, (4100, 17000, 128)), ((128, 256), True, 1, (2050, 5000, 17408)),
         ((128, 256), True, 2, (2050, 5000, 17408))]


@pytest.mark.parametrize("dtype", [Q2, Q4])
@pytest.mark.parametrize("tile,split,parts,size", TILED)
def test_every_tile_shape(hip, dtype, tile, split, parts, size):
    import ctox_hip as ch
    say(f"case rows product tile={tile} split={split} parts={parts} dtype={dtype} {size}")
    rows, n, cols = size
    rng = np.random.default_rng(rows + n + cols + dtype)
    m, d = build(hip, rng, [dtype], [n], cols, s_in=parts == 2, bias=True)
    half = parts == 1
    got = m.rows_tiling(rows, ch.TensorDType.F16 if half else ch.TensorDType.F32)
    assert got[:2] == tile and (got[2] > 1) == split
    x = rng.standard_normal((rows, cols), dtype=np.float32).astype(np.float16 if half else np.float32)
    pick = np.unique(np.r_[0, 31, rows - 1 - np.arange(5), rng.integers(0, rows, 40)] % rows)
    y = run(m, x)
    check(y[pick], *expect(d, x[pick], None), False)
    m.close()


@pytest.mark.parametrize("dtype", [Q2, Q4])
def test_f16_activations_below_the_normal_range(hip, dtype):
    say(f"case rows product f16 subnormals dtype={dtype}")
    rng = np.random.default_rng(61)
    m, d = build(hip, rng, [dtype], [70], 256, s_in=False, bias=False)
    x = (rng.standard_normal((40, 256)) * 10.0 ** rng.uniform(-7.5, -4, (40, 1))).astype(np.float16)
    x[7] = np.uint16(1).view(np.float16)
    check(run(m, x), *expect(d, x, None), False)


@pytest.mark.parametrize("kinds", [("F32", "F16Le"), ("F16Le", "F16Le"), ("F32", "F32")])
@pytest.mark.parametrize("half", [False, True])
def test_scale_types_of_mixed_segments(hip, kinds, half):
    import ctox_hip as ch
    say(f"case rows product scales {kinds} half={half}")
    rng = np.random.default_rng(67)
    cols, rows_each, dtypes = 448, (41, 90), (Q2, Q4)
    parts = [pack(rng, d, r, cols) for d, r in zip(dtypes, rows_each)]
    types = dict(F32=np.float32, F16Le=np.float16)
    si = rng.uniform(0.5, 1.5, cols).astype(types[kinds[0]])
    so = rng.uniform(0.5, 1.5, 131).astype(types[kinds[1]])
    bias = (rng.standard_normal(131) * 0.1).astype(np.float32)
    segs = [ch.QuantSegment(0, 0, 41, ch.TensorDType(Q2), 0, parts[0].size),
            ch.QuantSegment(1, 41, 131, ch.TensorDType(Q4), parts[0].size, parts[1].size)]
    m = hip.prepare(ch.FusedMatVec(ch.TensorDType.MixedQ2Q4B64, np.concatenate([p.reshape(-1) for p in parts]), 131, cols,
                                   segments=segs, s_in=getattr(ch.ScaleSlice, kinds[0])(si),
                                   s_out=getattr(ch.ScaleSlice, kinds[1])(so), bias=bias, activation=ch.Activation.Silu))
    d = dict(W=np.concatenate([values(p, t) for p, t in zip(parts, dtypes)]), s_in=si.astype(np.float64), s_out=so.astype(np.float64),
             bias=bias, silu=True)
    for rows in (5, 80):
        x = rng.standard_normal((rows, cols)).astype(np.float16 if half else np.float32)
        check(run(m, x, y_half=half), *expect(d, x, None), half)
