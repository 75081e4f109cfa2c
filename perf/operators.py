"""Operators that take a prompt chunk of a ragged batch through an attention layer.

A case is a dict of plain values whose "op" names the operator:

  project    y = act((x * s_in . W^T + bias) * s_out) + residual, W resident in
             packed Q2 / Q4 blocks, any number of rows, x and y f32 or f16
  rope       (1 + w) RMS norm of each q / k head, then rotary positions on one
             to four axes, read from a fused projection's rows
  plan       page descriptors and the slot map of a batch's new tokens, from
             the requests' lengths
  attention  append of a ragged batch's new K / V rows to the paged mixed
             Q2 / Q4 cache, then causal attention of those rows over it

`run` computes the plain forms with elementary torch operations in 32 bits
(angles in 64); where `own` is set it calls the library. `exact` evaluates the
same inputs in float64.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda"
EPS = 1e-6
Q2, Q4 = 0, 1
BLOCK_BYTES = {Q2: 18, Q4: 34}
BITS = {Q2: 2, Q4: 4}
LEVELS = {Q2: 3, Q4: 15}  # value = scale * (2 code - LEVELS) / LEVELS
HD = 256
SINK, RECENT = 128, 256   # tokens that the cache keeps in Q4 pages at either end
_backend = None


def _ctox():
    path = os.path.join(ROOT, "ctox-llm_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import ctox_hip
    return ctox_hip


def hip():
    """The process's backend handle, as a serving program holds one per GPU."""
    global _backend
    if _backend is None:
        _backend = _ctox().HipBackend(0)
    return _backend


def _stream():
    return torch.cuda.current_stream().cuda_stream


def listed():
    return [
        # The q|k|v projections of sixteen rows: two requests' draft verifications in one pass.
        {"name": "project_qkv_rows16", "op": "project", "dtype": Q4, "rows": 14336, "columns": 5120, "batch": 16,
         "half": False, "s_in": True, "bias": False, "silu": False, "residual": False},
        # A gate projection with bias and SiLU for a chunk of an odd number of tokens.
        {"name": "project_gate_rows777", "op": "project", "dtype": Q4, "rows": 17408, "columns": 5120, "batch": 777,
         "half": False, "s_in": True, "bias": True, "silu": True, "residual": False},
        # The down projection of a 4096-token prompt, added to the residual stream: the largest product.
        {"name": "project_down_rows4096", "op": "project", "dtype": Q2, "rows": 5120, "columns": 17408, "batch": 4096,
         "half": False, "s_in": True, "bias": False, "silu": False, "residual": True},
        # The output projection of a 2048-token chunk with f16 activations, as a half-precision host holds them.
        {"name": "project_out_half_rows2048", "op": "project", "dtype": Q4, "rows": 5120, "columns": 6144,
         "batch": 2048, "half": True, "s_in": False, "bias": False, "silu": False, "residual": True},
        # q / k norms and rotary of a decode batch, text positions on one axis.
        {"name": "rope_text_rows16", "op": "rope", "rows": 16, "heads": 24, "kv_heads": 4, "rotary": 64, "axes": 1,
         "far": 262144},
        # The same for a chunk of video tokens, positions in time, height and width.
        {"name": "rope_video_rows4096", "op": "rope", "rows": 4096, "heads": 24, "kv_heads": 4, "rotary": 64, "axes": 3,
         "far": 16384},
        # The plan of one decode step of eight requests.
        {"name": "plan_decode_8", "op": "plan", "requests": 8, "added": 1, "cached": 30000, "page": 16},
        # The plan of a large ragged step: 512 requests, prompts and decodes mixed.
        {"name": "plan_mixed_512", "op": "plan", "requests": 512, "added": 257, "cached": 9000, "page": 16},
        # A decode step of 32 requests with contexts of up to 8192 tokens.
        {"name": "attention_decode_32", "op": "attention", "requests": 32, "new": 1, "cached": 8192, "page": 16,
         "heads": 24, "kv_heads": 4, "ragged": True},
        # A 4096-token prompt from an empty cache.
        {"name": "attention_prompt_4096", "op": "attention", "requests": 1, "new": 4096, "cached": 0, "page": 16,
         "heads": 24, "kv_heads": 4, "ragged": False},
        # A 512-token chunk behind 32768 cached tokens.
        {"name": "attention_chunk_32k", "op": "attention", "requests": 1, "new": 512, "cached": 32768, "page": 16,
         "heads": 24, "kv_heads": 4, "ragged": False},
        # A mixed step: requests of 0 to 601 new rows, pages of 24 tokens that end inside any tile.
        {"name": "attention_mixed_6", "op": "attention", "requests": 6, "new": 601, "cached": 5003, "page": 24,
         "heads": 24, "kv_heads": 4, "ragged": True},
    ]


def _log_int(rng, lo, hi, multiple=1):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / multiple)) * multiple))


def draw(rng):
    op = rng.choice(["project", "project", "project", "rope", "plan", "attention", "attention", "attention"])
    if op == "project":
        rows, columns = _log_int(rng, 64, 17408), _log_int(rng, 256, 17408, 64)
        most = min(4096, 5120 * 17408 * 4096 // (rows * columns))
        half = rng.random() < 0.3
        return {"op": op, "dtype": rng.choice([Q2, Q4]), "rows": rows, "columns": columns,
                "batch": _log_int(rng, 1, most), "half": half, "s_in": rng.random() < (0.3 if half else 0.7),
                "bias": rng.random() < 0.4, "silu": rng.random() < 0.3, "residual": rng.random() < 0.5}
    if op == "rope":
        heads, kv_heads = rng.choice([(24, 4), (16, 4), (8, 2), (4, 1)])
        return {"op": op, "rows": _log_int(rng, 1, 4096), "heads": heads, "kv_heads": kv_heads,
                "rotary": rng.choice([64, 64, 128, 256, 32]), "axes": rng.choice([1, 2, 3, 3, 4]),
                "far": _log_int(rng, 64, 1000000)}
    if op == "plan":
        return {"op": op, "requests": _log_int(rng, 1, 512), "added": _log_int(rng, 1, 257),
                "cached": _log_int(rng, 1, 9000), "page": rng.choice([16, 16, 8, 24, 128])}
    heads, kv_heads = rng.choice([(24, 4), (24, 4), (16, 4), (8, 2), (8, 8)])
    requests, page, ragged = _log_int(rng, 1, 32), rng.choice([16, 16, 128, 24, 7]), rng.random() < 0.7
    new = _log_int(rng, 1, 2048 if requests == 1 else 512)
    # The plain form's scores stay within 2^28 values, its keys and values within 2^28.
    most = min(32768, 2 ** 28 // (requests * new * heads), 2 ** 28 // (requests * kv_heads * HD * 2))
    return {"op": op, "requests": requests, "new": new, "cached": _log_int(rng, 1, max(1, most - new)), "page": page,
            "heads": heads, "kv_heads": kv_heads, "ragged": ragged}


# ---------------------------------------------------------------- lengths
def _lengths(c):
    """(cached, new) of every request. Ragged batches spread both from nothing to the case's
    largest along a fixed sequence; every sixth request or so has no new rows."""
    R, most = c["requests"], c.get("new", c.get("added"))
    if not c.get("ragged", True):
        return [c["cached"]] * R, [most] * R
    cached, new = [], []
    for r in range(R):
        f, g = (0.618034 * r) % 1.0, (0.754878 * r) % 1.0
        cached.append(int(round(c["cached"] * (1.0 - f))))
        n = 1 if most == 1 else int(round(most * (1.0 - g) ** 3))
        new.append(0 if r % 6 == 5 and most > 1 else max(n, 0))
    return cached, new


def _q2_pages(cached, page):
    """Whether each of a request's pages was demoted: past the sink, wholly older than the recent window."""
    sink = -(-SINK // page) * page
    return [p * page >= sink and (p + 1) * page <= cached - RECENT for p in range(-(-cached // page))]


# ---------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 7919 + 29)
    return g


def _randn(g, *shape, std=1.0):
    return torch.randn(*shape, device=DEV, generator=g) * std


def _blocks(g, dtype, rows, blocks, scales):
    """Packed rows [rows][blocks][block bytes]: uniform codes and the given f16 scales."""
    w = torch.randint(0, 256, (rows, blocks, BLOCK_BYTES[dtype]), dtype=torch.uint8, device=DEV, generator=g)
    w[:, :, :2] = scales.half().view(torch.uint8).view(rows, blocks, 2)
    return w


def _cache_rows(g, dtype, rows, cv):
    """Token rows of a page pool [rows][token bytes]: normed keys, values of varying size."""
    n = cv // 64
    k = 2.4 + 0.35 * _randn(g, rows, n)
    v = 1.5 * torch.exp(0.3 * _randn(g, rows, n))
    return _blocks(g, dtype, rows, 2 * n, torch.cat([k.abs(), v], 1)).flatten(1)


def _inputs(c, seed):
    """The tensors that a case starts from."""
    g, op = _gen(seed), c["op"]
    if op == "project":
        M, N, K = c["batch"], c["rows"], c["columns"]
        t = torch.float16 if c["half"] else torch.float32
        i = {"w": _blocks(g, c["dtype"], N, K // 64, _randn(g, N, K // 64, std=0.02).abs()),
             "s_out": (0.75 + 0.5 * torch.rand(N, device=DEV, generator=g)).half(),
             "s_in": (0.75 + 0.5 * torch.rand(K, device=DEV, generator=g)).half() if c["s_in"] else None,
             "bias": _randn(g, N, std=0.1) if c["bias"] else None}
        x = _randn(g, M, K)
        if c["dtype"] == Q2:  # a down projection reads silu(gate) * up
            x = x * torch.sigmoid(x) * _randn(g, M, K)
        i["x"] = x.to(t)
        i["residual"] = _randn(g, M, N).to(t) if c["residual"] else None
        return i
    if op == "rope":
        T, H, KV, axes = c["rows"], c["heads"], c["kv_heads"], c["axes"]
        half = c["rotary"] // 2
        # Pairs go to the axes in turn, the last eighth to the first axis alone.
        axis = [0 if p >= half - half // 8 else p % axes for p in range(half)]
        return {"proj": _randn(g, T, (2 * H + 2 * KV) * HD), "q_norm": _randn(g, HD, std=0.1),
                "k_norm": _randn(g, HD, std=0.1), "axis": axis,
                "positions": torch.randint(0, c["far"], (T, axes), dtype=torch.int32, device=DEV, generator=g)}
    cached, new = _lengths(c)
    page, R = c["page"], c["requests"]
    pages = [-(-(a + n) // page) for a, n in zip(cached, new)]
    held = [-(-a // page) for a in cached]
    max_pages = max(1, max(pages))
    if op == "plan":
        max_pages += 3
        total, take = sum(held), sum(pages) - sum(held)
        perm = torch.randperm(total + take + 7, device=DEV, generator=g).to(torch.int32)
        desc = np.zeros((R, max_pages, 4), np.int32)
        at = 0
        for r in range(R):
            n = held[r]
            first = np.arange(n) * page
            desc[r, :n, 0], desc[r, :n, 3] = 1, first
            desc[r, :n, 2] = np.minimum(page, cached[r] - first)
            at += n
        desc = torch.from_numpy(desc).to(DEV)
        desc[..., 1][desc[..., 2] > 0] = perm[:total]
        rows = sum(new) + 5
        return {"cached": torch.tensor(cached, dtype=torch.int32, device=DEV),
                "added": torch.tensor(new, dtype=torch.int32, device=DEV), "descriptors": desc,
                "free": perm[total:].contiguous(), "max_rows": rows, "q4_slots": total + take + 7,
                "row_starts": torch.empty(R + 1, dtype=torch.int32, device=DEV),
                "tokens": torch.empty(R, dtype=torch.int32, device=DEV),
                "page_counts": torch.empty(R, dtype=torch.int32, device=DEV),
                "positions": torch.zeros(rows, dtype=torch.int32, device=DEV),
                "slots": torch.empty(rows, dtype=torch.int32, device=DEV),
                "status": torch.empty(4, dtype=torch.int32, device=DEV)}
    # attention
    H, KV, cv = c["heads"], c["kv_heads"], c["kv_heads"] * HD
    n2 = sum(sum(_q2_pages(a, page)) for a in cached)
    n4 = sum(pages) - n2
    slots4 = torch.randperm(n4 + 1, device=DEV, generator=g).cpu().numpy()
    slots2 = torch.randperm(n2 + 1, device=DEV, generator=g).cpu().numpy()
    desc = np.zeros((R, max_pages, 4), np.int32)
    slot_map, at = [], {Q2: 0, Q4: 0}
    for r in range(R):
        total = cached[r] + new[r]
        old = _q2_pages(cached[r], page)
        for p in range(pages[r]):
            kind = Q2 if p < len(old) and old[p] else Q4
            desc[r, p] = (kind, (slots2 if kind == Q2 else slots4)[at[kind]], min(page, total - p * page), p * page)
            at[kind] += 1
        pos = np.arange(cached[r], total)
        slot_map.append(desc[r, pos // page, 1] * page + pos % page)
    M = sum(new)
    pad = 5 if c["ragged"] else 0  # rows behind the last request, as a padded batch has
    slot_map = np.concatenate(slot_map + [np.full(pad, -1)]).astype(np.int32)
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    return {"q4": _cache_rows(g, Q4, (n4 + 1) * page, cv), "q2": _cache_rows(g, Q2, (n2 + 1) * page, cv),
            "descriptors": torch.from_numpy(desc).to(DEV), "slots": torch.from_numpy(slot_map).to(DEV),
            "row_starts": torch.from_numpy(starts).to(DEV), "max_new": max(max(new), 1),
            "tokens": torch.tensor([a + n for a, n in zip(cached, new)], dtype=torch.int32, device=DEV),
            "max_tokens": max(a + n for a, n in zip(cached, new)), "rows": M, "q4_slots": n4 + 1,
            "query": _randn(g, M + pad, H, HD), "keys": _randn(g, M + pad, cv),
            "values": _randn(g, M + pad, cv, std=0.6), "out": torch.zeros(M + pad, H, HD, device=DEV)}


def prepare(case, seed):
    c = dict(case)
    s = {"case": c, **_inputs(c, seed)}
    op = c["op"]
    if op == "project":
        t = torch.float16 if c["half"] else torch.float32
        s["y"] = torch.empty(c["batch"], c["rows"], dtype=t, device=DEV)
    elif op == "rope":
        s["q_out"] = torch.empty(c["rows"], c["heads"], HD, device=DEV)
        s["k_out"] = torch.empty(c["rows"], c["kv_heads"], HD, device=DEV)
    if own:  # the resident matrix, descriptors and workspaces that a serving program keeps
        _keep(s)
    return s


# ---------------------------------------------------------------- the library's calls
def _keep(s):
    c, ctox = s["case"], _ctox()
    op = c["op"]
    if op == "project":
        def half(v):
            return None if v is None else ctox.ScaleSlice.F16Le(v.cpu().numpy())
        s["matrix"] = hip().prepare(ctox.FusedMatVec(
            ctox.TensorDType(c["dtype"]), s["w"].cpu().numpy(), c["rows"], c["columns"], s_in=half(s["s_in"]),
            s_out=half(s["s_out"]), bias=None if s["bias"] is None else s["bias"].cpu().numpy(),
            activation=ctox.Activation.Silu if c["silu"] else ctox.Activation.Identity))
        s["type"] = ctox.TensorDType.F16 if c["half"] else ctox.TensorDType.F32
        s["workspace"] = torch.empty(s["matrix"].rows_workspace(c["batch"], s["type"]), dtype=torch.uint8, device=DEV)
    elif op == "rope":
        H, KV, row = c["heads"], c["kv_heads"], s["proj"].shape[1]
        s["call"] = ctox.RopeAxes(
            d_q=s["proj"].data_ptr(), d_k=s["proj"].data_ptr() + 4 * 2 * H * HD, d_q_out=s["q_out"].data_ptr(),
            d_k_out=s["k_out"].data_ptr(), d_q_norm=s["q_norm"].data_ptr(), d_k_norm=s["k_norm"].data_ptr(),
            d_positions=s["positions"].data_ptr(), axis_of_pair=s["axis"], q_strides=(row, 2 * HD),
            k_strides=(row, HD), rows=c["rows"], q_heads=H, k_heads=KV, head_dim=HD, rotary_dim=c["rotary"],
            axes=c["axes"], theta=1e7, eps=EPS)
    elif op == "plan":
        s["call"] = ctox.PagedPlan(
            d_cached=s["cached"].data_ptr(), d_added=s["added"].data_ptr(), d_descriptors=s["descriptors"].data_ptr(),
            d_free_slots=s["free"].data_ptr(), d_row_starts=s["row_starts"].data_ptr(),
            d_tokens=s["tokens"].data_ptr(), d_page_counts=s["page_counts"].data_ptr(),
            d_positions=s["positions"].data_ptr(), d_slots=s["slots"].data_ptr(), d_status=s["status"].data_ptr(),
            requests=c["requests"], page_tokens=c["page"], max_pages=s["descriptors"].shape[1],
            free_count=s["free"].numel(), q4_slots=s["q4_slots"], max_rows=s["max_rows"])
    else:
        H, KV, page, cv = c["heads"], c["kv_heads"], c["page"], c["kv_heads"] * HD
        b4, b2 = s["q4"].shape[1], s["q2"].shape[1]
        params = ctox.PagedGqaParams(H, KV, HD, s["max_tokens"], page, s["descriptors"].shape[1], 2 * cv, b2, b4,
                                     page * b2, page * b4, 1.0 / math.sqrt(HD))
        s["call"] = ctox.PagedGqaRows(
            d_query=s["query"].data_ptr(), d_out=s["out"].data_ptr(), d_q2_pages=s["q2"].data_ptr(),
            d_q4_pages=s["q4"].data_ptr(), d_descriptors=s["descriptors"].data_ptr(),
            d_row_starts=s["row_starts"].data_ptr(), d_tokens=s["tokens"].data_ptr(), rows=s["query"].shape[0],
            requests=c["requests"], max_rows=s["max_new"], params=params)
        s["workspace"] = torch.empty(hip().paged_gqa_rows_workspace(s["call"]), dtype=torch.uint8, device=DEV)
        s["call"].bind_workspace(s["workspace"].data_ptr(), s["workspace"].numel())


def _run_own(s):
    c = s["case"]
    op = c["op"]
    if op == "project":
        s["matrix"].dispatch_rows(
            s["x"].data_ptr(), c["batch"], s["y"].data_ptr(),
            d_residual=None if s["residual"] is None else s["residual"].data_ptr(), x_dtype=s["type"],
            y_dtype=s["type"], d_workspace=s["workspace"].data_ptr(), workspace_bytes=s["workspace"].numel(),
            stream=_stream())
        return s["y"]
    if op == "rope":
        hip().rope_axes_device(s["call"], _stream())
        return {"q": s["q_out"], "k": s["k_out"]}
    if op == "plan":
        hip().paged_plan_device(s["call"], _stream())
        return {k: s[k] for k in PLANNED}
    cv = c["kv_heads"] * HD
    hip().kv_append_q4_device(s["q4"].data_ptr(), s["keys"].data_ptr(), s["values"].data_ptr(), s["slots"].data_ptr(),
                              s["query"].shape[0], cv, c["page"], s["q4_slots"], c["page"] * s["q4"].shape[1],
                              stream=_stream())
    hip().paged_gqa_rows_device(s["call"], _stream())
    return {"out": s["out"], "cache": s["q4"]}


PLANNED = ("row_starts", "tokens", "page_counts", "positions", "slots", "descriptors", "status")


# ---------------------------------------------------------------- plain forms, 32 bits
def _unpack(w, dtype):
    """Packed blocks [..., block bytes] to float32 values [..., 64]."""
    bits = BITS[dtype]
    scale = w[..., :2].contiguous().view(torch.float16).float()
    shifts = torch.arange(0, 8, bits, dtype=torch.uint8, device=w.device)
    codes = ((w[..., 2:, None] >> shifts) & (2 ** bits - 1)).flatten(-2)
    return scale * ((2.0 * codes.float() - LEVELS[dtype]) / LEVELS[dtype])


def _pack_q4(v):
    """Float32 blocks [..., 64] to Q4 bytes: scale max |v|, codes round(v / max * 7.5 + 7.5), halves up."""
    m = v.abs().amax(-1, keepdim=True)
    n = torch.where(m > 0, v / m, torch.zeros_like(v)).clamp(-1.0, 1.0)
    sel = n * 7.5 + 7.5
    low = torch.floor(sel)
    codes = (low + ((sel - low) >= 0.5)).clamp(0, 15) * (m > 0)
    codes = codes.to(torch.uint8).unflatten(-1, (32, 2))
    return torch.cat([m.half().view(torch.uint8), codes[..., 0] | (codes[..., 1] << 4)], -1)


def _plain_project(s):
    c = s["case"]
    x = s["x"].float()
    if s["s_in"] is not None:
        x = x * s["s_in"].float()
    y = x @ _unpack(s["w"], c["dtype"]).flatten(1).T
    if s["bias"] is not None:
        y = y + s["bias"]
    y = y * s["s_out"].float()
    if c["silu"]:
        y = y * torch.sigmoid(y)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["x"].dtype)


def _plain_rope(s):
    c = s["case"]
    T, H, KV, rd = c["rows"], c["heads"], c["kv_heads"], c["rotary"]
    half = rd // 2
    inv = 1e7 ** (-2.0 * torch.arange(half, dtype=torch.float64, device=DEV) / rd)
    axis = torch.tensor(s["axis"], device=DEV)
    angle = s["positions"][:, axis].double() * inv
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def turn(x, w):
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * (1.0 + w)
        a, b = x[..., :half], x[..., half:rd]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., rd:]], -1)

    q = s["proj"][:, :2 * H * HD].unflatten(1, (H, 2 * HD))[..., :HD]
    k = s["proj"][:, 2 * H * HD:(2 * H + KV) * HD].unflatten(1, (KV, HD))
    return {"q": turn(q, s["q_norm"]), "k": turn(k, s["k_norm"])}


def _plain_plan(s):
    c = s["case"]
    page, R, desc = c["page"], c["requests"], s["descriptors"]
    cached, added = s["cached"].long(), s["added"].long()
    tokens = cached + added
    held, pages = (cached + page - 1) // page, (tokens + page - 1) // page
    zero = torch.zeros(1, dtype=torch.long, device=DEV)
    starts = torch.cat([zero, torch.cumsum(added, 0)])
    taken = torch.cat([zero, torch.cumsum(pages - held, 0)])
    # descriptors: pages that were there get their new token count, new pages the next free slots
    p = torch.arange(desc.shape[1], device=DEV)[None]
    fresh = (p >= held[:, None]) & (p < pages[:, None])
    slot = s["free"].long()[(taken[:-1, None] + p - held[:, None]).clamp(0, s["free"].numel() - 1)]
    count = (tokens[:, None] - p * page).clamp(0, page)
    new = torch.stack([torch.ones_like(slot), slot, count, (p * page).expand_as(slot)], -1).to(torch.int32)
    touched = torch.where((p < held[:, None])[..., None], torch.stack(
        [desc[..., 0], desc[..., 1], count.to(torch.int32), desc[..., 3]], -1), desc)
    out = torch.where(fresh[..., None], new, touched)
    # every row's request, position and slot
    i = torch.arange(s["max_rows"], device=DEV)
    r = torch.searchsorted(starts[1:].contiguous(), i, right=True).clamp(max=R - 1)
    pos = cached[r] + i - starts[r]
    inside = i < starts[R]
    where = out[r, (pos // page).clamp(max=desc.shape[1] - 1), 1].long() * page + pos % page
    return {"row_starts": starts.to(torch.int32), "tokens": tokens.to(torch.int32),
            "page_counts": pages.to(torch.int32),
            "positions": torch.where(inside, pos, torch.zeros_like(pos)).to(torch.int32),
            "slots": torch.where(inside, where, torch.full_like(where, -1)).to(torch.int32), "descriptors": out,
            "status": torch.stack([zero[0], taken[R], starts[R], pages.sum()]).to(torch.int32)}


def _plain_attention(s):
    c = s["case"]
    H, KV, page, R, M = c["heads"], c["kv_heads"], c["page"], c["requests"], s["rows"]
    rows = torch.cat([s["keys"][:M], s["values"][:M]], 1).unflatten(1, (-1, 64))
    s["q4"][s["slots"][:M].long()] = _pack_q4(rows).flatten(1)
    # every request's tokens, padded to the longest
    j = torch.arange(s["max_tokens"], device=DEV)
    desc = s["descriptors"].long()[:, j // page]
    at = desc[..., 1] * page + j % page
    present = j < s["tokens"][:, None]
    is4 = desc[..., 0] == Q4
    kv4 = _unpack(s["q4"][torch.where(is4 & present, at, 0)].unflatten(-1, (-1, 34)), Q4)
    kv2 = _unpack(s["q2"][torch.where(is4 | ~present, 0, at)].unflatten(-1, (-1, 18)), Q2)
    kv = torch.where(is4[..., None, None], kv4, kv2).view(R, -1, 2, KV, HD)
    k, v = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)             # [R][KV][tokens][HD]
    # every request's rows, padded to the most
    n, i = s["max_new"], torch.arange(s["max_new"], device=DEV)
    starts = s["row_starts"].long()
    count = starts[1:] - starts[:-1]
    src = (starts[:-1, None] + i).clamp(max=max(M - 1, 0))
    q = s["query"][src].view(R, n, KV, H // KV, HD).permute(0, 2, 1, 3, 4).reshape(R, KV, -1, HD)
    last = (s["tokens"].long() - count)[:, None] + i                            # the last token a row sees
    seen = (j <= last[..., None]) & present[:, None]                            # [R][n][tokens]
    x = (q @ k.transpose(2, 3)).view(R, KV, n, H // KV, -1) * (1.0 / math.sqrt(HD))
    x = x.masked_fill(~seen[:, None, :, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    o = (p.view(R, KV, -1, p.shape[-1]) @ v).view(R, KV, n, H // KV, HD) / torch.where(total > 0, total, 1.0)
    out = torch.zeros_like(s["out"])
    mine = i < count[:, None]
    out[src[mine]] = o.permute(0, 2, 1, 3, 4).reshape(R, n, H, HD)[mine]
    return {"out": out, "cache": s["q4"]}


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    if op == "project":
        return _plain_project(state)
    if op == "rope":
        return _plain_rope(state)
    if op == "plan":
        return _plain_plan(state)
    return _plain_attention(state)


# ---------------------------------------------------------------- 64 bits
def _values64(w, dtype):
    bits, per = BITS[dtype], 8 // BITS[dtype]
    scale = w[..., :2].contiguous().view(torch.float16).double()
    codes = torch.stack([(w[..., 2:] >> (bits * i)) & (2 ** bits - 1) for i in range(per)], -1)
    return scale * (codes.flatten(-2).double() * (2.0 / LEVELS[dtype]) - 1.0)


def _stored64(v):
    """What the cache holds of float32 blocks [..., 64]; the format's codes are defined in 32-bit steps."""
    m = v.abs().max(-1, keepdim=True).values
    sel = (v / m) * 7.5 + 7.5
    codes = torch.floor(sel.double() + 0.5).clamp(0, 15)
    return torch.where(m > 0, m.half().double() * (codes - 7.5) / 7.5, 0.0)


def _exact_project(c, i):
    x = i["x"].double()
    if c["s_in"]:
        x = x * i["s_in"].double()
    parts = [x @ _values64(i["w"][r:r + 4096], c["dtype"]).flatten(1).T for r in range(0, c["rows"], 4096)]
    y = torch.cat(parts, 1)
    if c["bias"]:
        y += i["bias"].double()
    y *= i["s_out"].double()
    if c["silu"]:
        y = y / (1.0 + torch.exp(-y))
    return y + i["residual"].double() if c["residual"] else y


def _exact_rope(c, i):
    H, KV, half = c["heads"], c["kv_heads"], c["rotary"] // 2
    inv = torch.tensor([math.exp(-2.0 * p / c["rotary"] * math.log(1e7)) for p in range(half)], dtype=torch.float64,
                       device=DEV)
    out = {}
    for name, at, heads, step, w in (("q", 0, H, 2 * HD, i["q_norm"]), ("k", 2 * H * HD, KV, HD, i["k_norm"])):
        x = i["proj"][:, at:at + heads * step].double().view(-1, heads, step)[..., :HD]
        x = x * torch.rsqrt(x.square().sum(-1, keepdim=True) / HD + EPS) * (1.0 + w.double())
        y = x.clone()
        for p in range(half):
            a = (i["positions"][:, i["axis"][p]].double() * inv[p])[:, None]
            y[..., p] = x[..., p] * torch.cos(a) - x[..., p + half] * torch.sin(a)
            y[..., p + half] = x[..., p + half] * torch.cos(a) + x[..., p] * torch.sin(a)
        out[name] = y
    return out


def _exact_attention(c, i):
    H, KV, page, cv = c["heads"], c["kv_heads"], c["page"], c["kv_heads"] * HD
    G, (cached, new) = H // KV, _lengths(c)
    out = torch.zeros(i["out"].shape, dtype=torch.float64, device=DEV)
    at = 0
    for r in range(c["requests"]):
        n, old = new[r], cached[r]
        if n == 0:
            continue
        j = torch.arange(old, device=DEV)
        d = i["descriptors"][r].long()[j // page]
        where = d[:, 1] * page + j % page
        kv = torch.zeros(old + n, 2 * cv, dtype=torch.float64, device=DEV)
        is4 = (d[:, 0] == Q4).nonzero()[:, 0]
        is2 = (d[:, 0] == Q2).nonzero()[:, 0]
        kv[is4] = _values64(i["q4"][where[is4]].unflatten(-1, (-1, 34)), Q4).flatten(1)
        kv[is2] = _values64(i["q2"][where[is2]].unflatten(-1, (-1, 18)), Q2).flatten(1)
        fresh = torch.cat([i["keys"][at:at + n], i["values"][at:at + n]], 1)
        kv[old:] = _stored64(fresh.view(n, -1, 64)).flatten(1)
        hidden = torch.arange(old + n, device=DEV) > old + torch.arange(n, device=DEV)[:, None]
        for h in range(KV):
            k, v = kv[:, h * HD:(h + 1) * HD], kv[:, cv + h * HD:cv + (h + 1) * HD]
            for g in range(G):
                x = i["query"][at:at + n, h * G + g].double() @ k.T / 16.0
                out[at:at + n, h * G + g] = torch.softmax(x.masked_fill_(hidden, -math.inf), -1) @ v
        at += n
    return {"out": out, "cache": None}


def exact(case, seed):
    c = dict(case)
    if c["op"] == "plan":
        return None  # whole numbers
    i = _inputs(c, seed)
    return {"project": _exact_project, "rope": _exact_rope, "attention": _exact_attention}[c["op"]](c, i)


# ---------------------------------------------------------------- work
def work(case):
    c = dict(case)
    op = c["op"]
    if op == "project":
        M, N, K = c["batch"], c["rows"], c["columns"]
        size = 2 if c["half"] else 4
        moved = N * (K // 64) * BLOCK_BYTES[c["dtype"]] + M * K * size + M * N * size * (2 if c["residual"] else 1)
        return {"bytes": moved + 2 * N + (2 * K if c["s_in"] else 0) + (4 * N if c["bias"] else 0),
                "flops": 2 * M * N * K}
    if op == "rope":
        n = c["rows"] * (c["heads"] + c["kv_heads"]) * HD
        return {"bytes": 8 * n + 4 * c["rows"] * c["axes"], "flops": 6 * n}
    cached, new = _lengths(c)
    page = c["page"]
    if op == "plan":
        pages = sum(-(-(a + n) // page) + (-a // page) for a, n in zip(cached, new))
        return {"bytes": 20 * c["requests"] + 20 * pages + 8 * sum(new), "flops": 0}
    H, cv = c["heads"], c["kv_heads"] * HD
    moved = pairs = 0
    for a, n in zip(cached, new):
        if n:
            moved += sum(min(page, a - p * page) * 2 * cv // 64 * (18 if q2 else 34)
                         for p, q2 in enumerate(_q2_pages(a, page)))
            pairs += n * a + n * (n + 1) // 2
    M = sum(new)
    # new rows: K / V read and stored, the query read, the output written
    moved += M * (8 * cv + 2 * cv // 64 * 34 + 8 * H * HD)
    return {"bytes": moved, "flops": 4 * HD * H * pairs}
