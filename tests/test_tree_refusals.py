"""Refusals of the entry points for trees of drafted tokens. Every check of an argument runs before the backend
handle is read, so all of them are reached without a GPU: the calls pass no backend, and a call that is in order
ends at that."""
import ctypes

import pytest

import ctox_hip as ch

P = 0x10000  # an address that no check reads


def call(name, op, kind=ch.ShapeError, bytes_out=False):
    lib = ch.load_library()
    args = (ctypes.byref(ctypes.c_size_t()),) if bytes_out else (None,)
    with pytest.raises(kind) as e:
        ch._check(getattr(lib, name)(None, ctypes.byref(op), *args))
    return str(e.value)


def plan(**over):
    kw = {f"d_{n}": P for n in ("row_starts", "tokens", "parents", "masks", "positions", "depths")}
    kw.update(requests=3, rows=20)
    kw.update(over)
    return call("ctox_hip_tree_plan_device", ch.TreePlan(**kw))


@pytest.mark.parametrize("over,says", [
    ({}, "null argument"), (dict(requests=0), "requests"), (dict(requests=4097), "requests"), (dict(rows=1 << 24), "2^24"),
    (dict(d_parents=None), "null"), (dict(d_depths=None), "null"),
])
def test_plan_refuses(over, says):
    assert says in plan(**over)


def attention(bytes_out=False, name=None, kind=ch.ShapeError, d_masks=P, **over):
    params = dict(query_heads=24, key_value_heads=4, head_dim=256, tokens=0, page_tokens=16, page_count=8,
                  combined_values=2048, q2_token_bytes=576, q4_token_bytes=1088, q2_page_bytes=9216,
                  q4_page_bytes=17408, scale=0.0625)
    kw = dict(rows=20, requests=3, max_rows=0)
    for k, v in over.items():
        (params if k in params else kw)[k] = v
    op = ch.PagedGqaTree(P, P, P, P, P, P, P, d_masks, params=ch.PagedGqaParams(*params.values()), **kw)
    name = "ctox_hip_paged_gqa_tree_" + ("workspace" if bytes_out else "device")
    return call(name, op, kind, bytes_out)


@pytest.mark.parametrize("over,says", [
    ({}, "null argument"), (dict(max_rows=64), "null argument"), (dict(max_rows=65), "65 nodes"),
    (dict(requests=0), "requests"), (dict(rows=(1 << 20) + 1), "too many"), (dict(combined_values=2047), "geometry"),
    (dict(query_heads=23), "contract"),
])
def test_attention_refuses(over, says):
    assert says in attention(**over)
    assert says in attention(bytes_out=True, **over)


def test_attention_needs_masks_and_head_dim():
    assert "null" in attention(d_masks=None)
    assert "8-byte" in attention(d_masks=P + 4)
    assert "head_dim" in attention(kind=ch.UnsupportedOperation, head_dim=128)


def verify(kind=ch.ShapeError, bytes_out=False, **over):
    kw = {f"d_{n}": P for n in ("target", "draft", "tokens", "parents", "row_starts", "accept_draws", "sample_draws",
                                "counts", "path", "next")}
    kw.update(requests=3, rows=20, vocab=1000, max_children=4, temperature=1.0)
    kw.update(over)
    return call("ctox_hip_verify_tree_" + ("workspace" if bytes_out else "device"), ch.VerifyTree(**kw), kind, bytes_out)


@pytest.mark.parametrize("over,says", [
    ({}, "null argument"), (dict(temperature=0.0, d_accept_draws=None, d_sample_draws=None), "null argument"),
    (dict(requests=0), "requests"), (dict(requests=4097), "requests"), (dict(rows=65536), "2^16"),
    (dict(vocab=0), "vocabulary"), (dict(vocab=1 << 31), "vocabulary"), (dict(max_children=0), "children"),
    (dict(max_children=65), "children"), (dict(draft_vocab=500), "inverse"), (dict(draft_vocab=0), "inverse"),
    (dict(draft_vocab=1001, d_draft_inverse=P), "inverse"), (dict(target_stride=999), "logit rows"),
    (dict(draft_stride=999), "logit rows"), (dict(target_stride=1 << 30), "logit rows"),
])
def test_verify_refuses(over, says):
    assert says in verify(**over)
    assert says in verify(bytes_out=True, **over)


@pytest.mark.parametrize("t", [-0.5, float("nan"), float("inf")])
def test_verify_refuses_temperatures(t):
    assert "temperature" in verify(kind=ch.InvalidArtifact, temperature=t)


@pytest.mark.parametrize("name", ["target", "tokens", "parents", "row_starts", "accept_draws", "sample_draws", "counts",
                                  "path", "next"])
def test_verify_needs_its_pointers(name):
    assert "null" in verify(**{f"d_{name}": None})


GEOMETRY = dict(requests=3, max_pages=8, page_tokens=16, q4_slots=40, token_bytes=1088, q4_page_bytes=17408)


def commit(pools=(P, 2 * P), **over):
    kw = {f"d_{n}": P for n in ("descriptors", "row_starts", "tokens", "counts", "path", "new_tokens", "status")}
    kw.update(GEOMETRY, rows=20)
    kw.update(over)
    return call("ctox_hip_paged_commit_device", ch.PagedCommit(list(pools), **kw))


def fork(pools=(P, 2 * P), **over):
    kw = {f"d_{n}": P for n in ("descriptors", "tokens", "sources", "targets", "free_slots", "free_count", "status")}
    kw.update(GEOMETRY, forks=2)
    kw.update(over)
    return call("ctox_hip_paged_fork_device", ch.PagedFork(list(pools), **kw))


@pytest.mark.parametrize("over,says", [
    ({}, "null argument"), (dict(requests=0), "requests"), (dict(requests=4097), "requests"), (dict(pools=()), "layers"),
    (dict(pools=(P,) * 65), "layers"), (dict(pools=(P, None)), "null"), (dict(pools=(P, P + 2)), "alignment"),
    (dict(page_tokens=0), "geometry"), (dict(max_pages=0), "geometry"), (dict(max_pages=1 << 28), "geometry"),
    (dict(q4_slots=1 << 28), "geometry"), (dict(token_bytes=0), "page"), (dict(token_bytes=1090), "page"),
    (dict(q4_page_bytes=17404), "page"), (dict(q4_page_bytes=17410), "page"),
])
def test_pools_refuse(over, says):
    assert says in commit(**over)
    assert says in fork(**over)


def test_fork_and_commit_refuse():
    assert "too many" in fork(forks=4097)
    assert "too many" in commit(rows=1 << 31)
    assert "null" in fork(d_sources=None) and "null" in commit(d_path=None)


def free(bytes_out=False, **over):
    kw = {f"d_{n}": P for n in ("descriptors", "tokens", "q4_free", "q2_free", "counts")}
    kw.update(requests=3, max_pages=8, page_tokens=16, q4_slots=40, q2_slots=20)
    kw.update(over)
    return call("ctox_hip_paged_free_slots_" + ("workspace" if bytes_out else "device"), ch.PagedFreeSlots(**kw),
                bytes_out=bytes_out)


@pytest.mark.parametrize("over,says", [
    ({}, "null argument"), (dict(requests=0), "requests"), (dict(page_tokens=0), "geometry"),
    (dict(q4_slots=(1 << 24) + 1), "geometry"), (dict(q2_slots=(1 << 24) + 1), "geometry"), (dict(max_pages=0), "geometry"),
])
def test_free_slots_refuses(over, says):
    assert says in free(**over)
    assert says in free(bytes_out=True, **over)


def delta(commit=False, bytes_out=False, **over):
    kw = {f"d_{n}": P for n in ("proj", "conv_w", "conv_in", "a_log", "dt_bias", "state_in", "row_starts", "parents", "out",
                                "counts", "path", "conv_out", "state_out")}
    kw.update(proj_stride=20000, a_off=19000, b_off=19100, requests=3, rows=20, heads=48, key_heads=16, key_dim=128,
              value_dim=128, kernel=4)
    kw.update(over)
    name = "ctox_hip_gdn_tree_" + ("workspace" if bytes_out else "commit_device" if commit else "device")
    return call(name, ch.GdnTree(**kw), bytes_out=bytes_out)


@pytest.mark.parametrize("over,says", [
    ({}, "null argument"), (dict(requests=0), "requests"), (dict(rows=1 << 24), "2^24"), (dict(max_rows=65), "65 nodes"),
    (dict(heads=0), "shapes"), (dict(key_heads=0), "shapes"), (dict(heads=47), "shapes"), (dict(key_dim=0), "shapes"),
    (dict(key_dim=129), "shapes"), (dict(value_dim=0), "shapes"), (dict(kernel=0), "shapes"), (dict(kernel=9), "shapes"),
    (dict(proj_stride=10239), "channels"), (dict(a_off=19953), "channels"), (dict(b_off=1 << 40), "channels"),
    (dict(conv_stride=40959), "states"), (dict(state_stride=786431), "states"), (dict(state_stride=1 << 31), "states"),
    (dict(blocked=True, state_stride=786434), "16-byte"),
])
def test_delta_refuses(over, says):
    for how in (dict(), dict(commit=True), dict(bytes_out=True)):
        assert says in delta(**how, **over)


def test_numbers_that_do_not_fit_their_field_are_refused():
    with pytest.raises(ch.ShapeError):
        delta(rows=1 << 32)
    with pytest.raises(ch.ShapeError):
        verify(vocab=-1)
    op = ch.TreePlan(P, P, P, P, P, P, 1, 1)
    with pytest.raises(ch.ShapeError):
        op.rows = 1 << 32
