"""Refusals of the ragged-batch entry points. Every check of an argument runs
before the backend handle is read, so all of them are reached without a GPU:
the calls pass no backend, and a call that is in order ends at that."""
import ctypes

import pytest

import ctox_hip
from ctox_hip import PagedPlan, RopeAxes

P = 0x10000  # an address that no check reads


def call(name, *args):
    lib = ctox_hip.load_library()
    with pytest.raises(ctox_hip.ShapeError) as e:
        ctox_hip._check(getattr(lib, name)(None, *args))
    return str(e.value)


def rope(**over):
    kw = dict(d_q=P, d_positions=P, rows=3, q_heads=4, head_dim=256, rotary_dim=64, theta=1e7, d_k=P, k_heads=2,
              d_q_norm=P, d_k_norm=P)
    kw.update(over)
    return call("ctox_hip_rope_axes_device", ctypes.byref(RopeAxes(**kw)), None)


def test_rope_axes_in_order_without_a_backend():
    assert rope() == "null argument"
    assert rope(axis_of_pair=[0, 1] * 16, axes=2) == "null argument"
    assert rope(d_k=None, k_heads=0, d_k_norm=None) == "null argument"
    # heads outermost: [heads][rows][head_dim]
    assert rope(q_out_strides=(256, 3 * 256), d_q_out=2 * P) == "null argument"


@pytest.mark.parametrize("over,says", [
    (dict(rotary_dim=0), "rotary"), (dict(rotary_dim=63), "rotary"), (dict(rotary_dim=258), "rotary"),
    (dict(head_dim=1024, rotary_dim=514), "rotary"), (dict(theta=0.0), "theta"), (dict(theta=float("nan")), "theta"),
    (dict(head_dim=1028), "heads or axes"), (dict(axes=0), "heads or axes"), (dict(axes=5), "heads or axes"),
    (dict(q_heads=0, k_heads=0), "heads or axes"), (dict(eps=0.0), "epsilon"), (dict(eps=float("inf")), "epsilon"),
    (dict(axis_of_pair=[0] * 31 + [1]), "axis 1 of 1"), (dict(d_q=None), "null"), (dict(d_k=None), "null"),
    (dict(q_strides=(1 << 30, 256)), "stride"), (dict(d_q_out=2 * P, q_out_strides=(1024, 255)), "overlap"),
    (dict(d_q_out=2 * P, q_out_strides=(256, 256)), "overlap"),
    (dict(d_q_out=P, q_strides=(2048, 512), q_out_strides=(1024, 256)), "in place"),
])
def test_rope_axes_refuses(over, says):
    assert says in rope(**over)


def plan(**over):
    kw = {f"d_{n}": P for n in ("cached", "added", "descriptors", "free_slots", "row_starts", "tokens", "page_counts",
                                "positions", "slots", "status")}
    kw.update(requests=3, page_tokens=16, max_pages=8, free_count=5, q4_slots=40, max_rows=64)
    kw.update(over)
    return call("ctox_hip_paged_plan_device", ctypes.byref(PagedPlan(**kw)), None)


def test_plan_in_order_without_a_backend():
    assert plan() == "null argument"


@pytest.mark.parametrize("over,says", [
    (dict(requests=0), "requests"), (dict(requests=4097), "requests"), (dict(page_tokens=0), "geometry"),
    (dict(max_pages=0), "geometry"), (dict(max_pages=1 << 28), "geometry"), (dict(q4_slots=1 << 28), "geometry"),
    (dict(requests=4096, max_pages=1 << 20, page_tokens=1), "geometry"), (dict(max_rows=1 << 31), "geometry"),
])
def test_plan_refuses(over, says):
    assert says in plan(**over)


def append(**over):
    kw = dict(pages=P, keys=P, key_stride=1024, values=P, value_stride=1024, slots=P, rows=5, cv=1024, page=16,
              q4_slots=9, page_bytes=16 * 1088)
    kw.update(over)
    return call("ctox_hip_kv_append_q4_device", *kw.values(), None)


def test_append_in_order_without_a_backend():
    assert append() == "null argument"


@pytest.mark.parametrize("over,says", [
    (dict(cv=0), "multiple of 64"), (dict(cv=96), "multiple of 64"), (dict(page=0), "fit"), (dict(page=17), "fit"),
    (dict(page_bytes=16 * 1088 + 2), "fit"), (dict(q4_slots=1 << 28), "fit"), (dict(rows=1 << 31), "too large"),
    (dict(key_stride=1 << 30), "too large"),
])
def test_append_refuses(over, says):
    assert says in append(**over)


def test_rope_axes_needs_one_axis_per_pair():
    with pytest.raises(ctox_hip.ShapeError):
        RopeAxes(d_q=P, d_positions=P, rows=1, q_heads=1, head_dim=64, rotary_dim=64, theta=1e4, axis_of_pair=[0] * 31)


def rows_product(**over):
    kw = dict(x=P, y=P, residual=None, rows=4, x_stride=0, y_stride=0, residual_stride=0, x_dtype=4, y_dtype=3,
              workspace=P, workspace_bytes=1 << 20)
    kw.update(over)
    lib, op = ctox_hip.load_library(), ctox_hip._MatrixRows(*kw.values())
    with pytest.raises(ctox_hip.EngineError) as e:
        ctox_hip._check(lib.ctox_hip_matrix_dispatch_rows(None, None, ctypes.byref(op), None))
    return str(e.value)


@pytest.mark.parametrize("over,says", [
    (dict(), "null argument"), (dict(x_dtype=1), "dtypes"), (dict(y_dtype=5), "dtypes"), (dict(rows=(1 << 20) + 1), "2^20"),
    (dict(x_stride=1 << 30), "stride"), (dict(y_stride=1 << 31), "stride"), (dict(residual_stride=1 << 40), "stride"),
])
def test_rows_product_refuses(over, says):
    assert says in rows_product(**over)


def test_rows_workspace_refuses():
    lib, n = ctox_hip.load_library(), ctypes.c_size_t()
    for args, kind in (((None, 5, 4), ctox_hip.ShapeError), ((None, 5, 0), ctox_hip.UnsupportedDType),
                       ((None, (1 << 20) + 1, 4), ctox_hip.ShapeError)):
        with pytest.raises(kind):
            ctox_hip._check(lib.ctox_hip_matrix_rows_workspace(*args, ctypes.byref(n)))


def attention(params=None, **over):
    p = dict(query_heads=24, key_value_heads=4, head_dim=256, tokens=0, page_tokens=16, page_count=8,
             combined_values=2048, q2_token_bytes=576, q4_token_bytes=1088, q2_page_bytes=16 * 576,
             q4_page_bytes=16 * 1088, scale=0.0625)
    p.update(params or {})
    kw = dict(d_query=P, d_out=P, d_q2_pages=P, d_q4_pages=P, d_descriptors=P, d_row_starts=P, d_tokens=P, rows=9,
              requests=3)
    kw.update(over)
    lib, op, n = ctox_hip.load_library(), ctox_hip.PagedGqaRows(params=ctox_hip.PagedGqaParams(*p.values()), **kw), ctypes.c_size_t()
    said = []
    for f, args in (("ctox_hip_paged_gqa_rows_workspace", (ctypes.byref(n),)), ("ctox_hip_paged_gqa_rows_device", (None,))):
        with pytest.raises(ctox_hip.EngineError) as e:
            ctox_hip._check(getattr(lib, f)(None, ctypes.byref(op), *args))
        said.append(str(e.value))
    assert said[0] == said[1]
    return said[0]


@pytest.mark.parametrize("params,over,says", [
    ({}, {}, "null argument"), (dict(head_dim=128), {}, "head_dim 256"), (dict(key_value_heads=0), {}, "contract"),
    (dict(query_heads=22), {}, "contract"), (dict(page_tokens=0), {}, "contract"), (dict(page_count=0), {}, "contract"),
    (dict(scale=float("inf")), {}, "contract"), (dict(combined_values=1024), {}, "geometry"),
    (dict(q4_page_bytes=16 * 1088 - 4), {}, "geometry"), (dict(q2_page_bytes=16 * 576 + 2), {}, "geometry"),
    ({}, dict(requests=0), "requests"), ({}, dict(requests=4097), "requests"), ({}, dict(rows=(1 << 20) + 1), "rows"),
])
def test_attention_refuses(params, over, says):
    assert says in attention(params, **over)


@pytest.mark.parametrize("make", [
    lambda: RopeAxes(d_q=P, d_positions=P, rows=1, q_heads=1, head_dim=64, rotary_dim=64, theta=1e4,
                     axis_of_pair=[0] * 31 + [256]),
    lambda: RopeAxes(d_q=P, d_positions=P, rows=1, q_heads=1, head_dim=64, rotary_dim=64, theta=1e4,
                     axis_of_pair=[0] * 31 + [-1]),
    lambda: RopeAxes(d_q=P, d_positions=P, rows=2 ** 32 + 1, q_heads=1, head_dim=64, rotary_dim=64, theta=1e4),
    lambda: RopeAxes(d_q=P, d_positions=P, rows=1, q_heads=1, head_dim=64, rotary_dim=64, theta=1e4, q_strides=(-64, 64)),
    lambda: PagedPlan(*[P] * 10, requests=2 ** 32 + 3, page_tokens=16, max_pages=8, free_count=5, q4_slots=40, max_rows=64),
    lambda: PagedPlan(*[P] * 10, requests=3, page_tokens=16, max_pages=8, free_count=-1, q4_slots=40, max_rows=64),
    lambda: ctox_hip.PagedGqaRows(*[P] * 7, rows=-1, requests=3, params=ctox_hip.PagedGqaParams()),
    lambda: ctox_hip.PagedGqaRows(*[P] * 7, rows=9, requests=2 ** 32 + 3, params=ctox_hip.PagedGqaParams()),
    lambda: ctox_hip.PagedGqaRows(*[P] * 7, rows=9, requests=3, params=ctox_hip.PagedGqaParams(), max_rows=2 ** 32),
])
def test_numbers_that_do_not_fit_are_refused(make):
    """A field takes its value or refuses it; none is taken modulo the field's size."""
    with pytest.raises(ctox_hip.ShapeError):
        make()


def test_a_field_set_later_is_checked_too():
    op = ctox_hip.PagedGqaRows(*[P] * 7, rows=9, requests=3, params=ctox_hip.PagedGqaParams())
    with pytest.raises(ctox_hip.ShapeError):
        op.requests = 2 ** 32 + 3
    op.requests = 2 ** 32 - 1
    assert op.requests == 2 ** 32 - 1 and op.query == P


def unbound(cls):
    """A handle without a device: every check of these calls comes before it is read."""
    x = object.__new__(cls)
    x.handle = x.backend = None
    return x


@pytest.mark.parametrize("over", [dict(rows=2 ** 64 + 1), dict(component_values=-64), dict(page_tokens=2 ** 32 + 16),
                                  dict(q4_slots=2 ** 32 + 9), dict(q4_page_bytes=-4), dict(key_stride=-1024),
                                  dict(value_stride=2 ** 64 + 1024)])
def test_append_numbers_that_do_not_fit_are_refused(over):
    kw = dict(d_q4_pages=P, d_keys=P, d_values=P, d_slots=P, rows=5, component_values=1024, page_tokens=16, q4_slots=9,
              q4_page_bytes=16 * 1088)
    kw.update(over)
    with pytest.raises(ctox_hip.ShapeError, match="does not fit"):
        unbound(ctox_hip.HipBackend).kv_append_q4_device(**kw)


@pytest.mark.parametrize("over", [dict(rows=2 ** 64 + 4), dict(x_stride=-1), dict(y_stride=2 ** 64), dict(residual_stride=-5),
                                  dict(workspace_bytes=-1)])
def test_rows_product_numbers_that_do_not_fit_are_refused(over):
    kw = dict(d_x=P, rows=4, d_y=P, d_workspace=P, workspace_bytes=1 << 20)
    kw.update(over)
    m = unbound(ctox_hip.HipMatrix)
    m.backend = unbound(ctox_hip.HipBackend)
    with pytest.raises(ctox_hip.ShapeError, match="does not fit"):
        m.dispatch_rows(**kw)
    if "rows" in over:
        with pytest.raises(ctox_hip.ShapeError, match="does not fit"):
            m.rows_workspace(over["rows"])


def test_rows_tiling_refuses():
    lib, t = ctox_hip.load_library(), (ctypes.c_uint32 * 3)()
    for args, kind in (((5, 4, 0, None), ctox_hip.ShapeError), ((5, 1, 0, t), ctox_hip.UnsupportedDType),
                       ((0, 4, 0, t), ctox_hip.ShapeError), (((1 << 20) + 1, 4, 0, t), ctox_hip.ShapeError),
                       ((5, 4, 0, t), ctox_hip.ShapeError)):
        with pytest.raises(kind):
            ctox_hip._check(lib.ctox_hip_matrix_rows_tiling(None, *args))


def test_more_rows_than_a_launch_holds_are_refused():
    """A grid holds less than 2^32 threads along its first axis; the calls' workgroups of 256 or 512 reach it."""
    assert rope(rows=(1 << 24) - 1) == "null argument"
    assert "rows" in rope(rows=1 << 24)
    assert append(rows=(1 << 24) - 1) == "null argument"
    assert "too large" in append(rows=1 << 24)
    wide = dict(query_heads=8192, key_value_heads=8192, combined_values=8192 * 512, q2_token_bytes=8192 * 144,
                q4_token_bytes=8192 * 272, q2_page_bytes=16 * 8192 * 144, q4_page_bytes=16 * 8192 * 272)
    assert attention(wide, rows=100000) == "null argument"
    assert "rows" in attention(wide, rows=1 << 17)
