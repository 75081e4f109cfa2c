"""Operators of a decode step in which every request of a batch has a tree of drafted tokens.

A case is a dict of plain values whose "op" names the operator:

  tree       ancestor masks and positions of the drafted nodes, from their parents
  attention  append of the nodes' K / V rows to the paged mixed Q2 / Q4 cache, then attention in
             which a node sees the cached tokens and its own ancestors
  verify     which path of each tree the target's probabilities accept, and the next token, from
             given random numbers
  pages      what the accepted path leaves of the cache: kept tokens closed up in all layers'
             pages, the lists of free slots, survivors forked into the places of ended requests
  delta      the gated-delta (GatedDeltaNet) token mixer over a tree, then the state after its
             accepted path

A request's nodes are numbered so that a parent comes before its children; node 0 is the root,
the token that was chosen last. `run` computes the plain forms with elementary torch operations
in 32 bits (verification in 64: the borders of 150 thousand tokens lie closer than 32 bits tell
apart); where `own` is set it calls the library. `exact` evaluates the same inputs in float64.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda"
Q2, Q4 = 0, 1
BLOCK_BYTES = {Q2: 18, Q4: 34}
BITS = {Q2: 2, Q4: 4}
LEVELS = {Q2: 3, Q4: 15}  # value = scale * (2 code - LEVELS) / LEVELS
HD = 256
SINK, RECENT = 128, 256   # tokens that the cache keeps in Q4 pages at either end
NODES = 64                # of one tree
POINT, WITH, WITHOUT = 0, 1, 2  # how siblings were drawn: chosen outright, with / without replacement
LEAST_MASS = 2.0 ** -40   # siblings are offered while the draft has this much undrawn mass left
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
        # The trees of one decode step of eight requests.
        {"name": "tree_8x16", "op": "tree", "requests": 8, "nodes": 16, "width": 4},
        # The same for a full batch of large trees.
        {"name": "tree_512x64", "op": "tree", "requests": 512, "nodes": 64, "width": 4},
        # One request's small tree behind a conversation's context: a lone user's decode step.
        {"name": "attention_1x12_8k", "op": "attention", "requests": 1, "nodes": 12, "width": 3, "cached": 8192,
         "page": 16, "heads": 24, "kv_heads": 4, "ragged": False},
        # A serving batch of trees of up to 32 nodes, contexts of up to 8192 tokens.
        {"name": "attention_16x32_8k", "op": "attention", "requests": 16, "nodes": 32, "width": 4, "cached": 8192,
         "page": 16, "heads": 24, "kv_heads": 4, "ragged": True},
        # The largest tree behind a long document, pages that end inside any tile.
        {"name": "attention_4x64_32k", "op": "attention", "requests": 4, "nodes": 64, "width": 4, "cached": 32768,
         "page": 24, "heads": 24, "kv_heads": 4, "ragged": False},
        # A chain of four drafts of one request, as the draft layer makes it.
        {"name": "verify_chain_1x5", "op": "verify", "requests": 1, "nodes": 5, "width": 1, "vocab": 151936,
         "draft_vocab": 0, "drawn": WITHOUT, "temperature": 0.7, "ragged": False},
        # A serving batch's trees, siblings drawn without replacement.
        {"name": "verify_16x32", "op": "verify", "requests": 16, "nodes": 32, "width": 4, "vocab": 151936,
         "draft_vocab": 0, "drawn": WITHOUT, "temperature": 1.0, "ragged": True},
        # Greedy decoding with the best tokens of a restricted draft head as children.
        {"name": "verify_greedy_8x16", "op": "verify", "requests": 8, "nodes": 16, "width": 4, "vocab": 151936,
         "draft_vocab": 32768, "drawn": POINT, "temperature": 0.0, "ragged": True},
        # Four requests end a step over the model's sixteen attention layers; one ended, one goes on twice.
        {"name": "pages_4x16", "op": "pages", "requests": 4, "nodes": 16, "cached": 300, "page": 16, "layers": 16,
         "kv_heads": 4, "forks": 1},
        # A full batch, a quarter of it ended and filled up from the others.
        {"name": "pages_128x64", "op": "pages", "requests": 128, "nodes": 64, "cached": 700, "page": 16, "layers": 8,
         "kv_heads": 4, "forks": 32},
        # One recurrent layer of a lone request's small tree.
        {"name": "delta_1x12", "op": "delta", "requests": 1, "nodes": 12, "width": 3, "heads": 48, "key_heads": 16,
         "key_dim": 128, "value_dim": 128, "kernel": 4, "blocked": True, "ragged": False},
        # The same layer of a serving batch with the largest trees.
        {"name": "delta_16x64", "op": "delta", "requests": 16, "nodes": 64, "width": 4, "heads": 48, "key_heads": 16,
         "key_dim": 128, "value_dim": 128, "kernel": 4, "blocked": True, "ragged": True},
    ]


def _log_int(rng, lo, hi, multiple=1):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / multiple)) * multiple))


def draw(rng):
    op = rng.choice(["tree", "attention", "attention", "attention", "verify", "verify", "verify", "pages", "pages",
                     "delta", "delta", "delta"])
    width = rng.choice([1, 2, 3, 4, 4, 8])
    if op == "tree":
        return {"op": op, "requests": _log_int(rng, 1, 512), "nodes": _log_int(rng, 1, NODES), "width": width}
    if op == "attention":
        heads, kv_heads = rng.choice([(24, 4), (24, 4), (16, 4), (8, 2), (8, 8)])
        requests, nodes = _log_int(rng, 1, 16), _log_int(rng, 1, NODES)
        # The plain form's scores stay within 2^28 values, its keys and values within 2^28.
        most = min(32768, 2 ** 28 // (requests * nodes * heads), 2 ** 28 // (requests * kv_heads * HD * 2))
        return {"op": op, "requests": requests, "nodes": nodes, "width": width,
                "cached": _log_int(rng, 1, max(1, most - nodes)), "page": rng.choice([16, 16, 128, 24, 7]),
                "heads": heads, "kv_heads": kv_heads, "ragged": rng.random() < 0.7}
    if op == "verify":
        requests, nodes, vocab = _log_int(rng, 1, 32), _log_int(rng, 1, NODES), _log_int(rng, 1000, 151936)
        requests = min(requests, max(1, 16 * 32 * 151936 // (nodes * vocab)))
        return {"op": op, "requests": requests, "nodes": nodes, "width": width, "vocab": vocab,
                "draft_vocab": rng.choice([0, 0, vocab // 4]), "drawn": rng.choice([POINT, WITH, WITHOUT, WITHOUT]),
                "temperature": rng.choice([0.0, 0.3, 0.7, 1.0, 1.0, 1.4]), "ragged": rng.random() < 0.7}
    if op == "pages":
        requests = _log_int(rng, 1, 128)
        return {"op": op, "requests": requests, "nodes": _log_int(rng, 1, NODES), "cached": _log_int(rng, 1, 700),
                "page": rng.choice([16, 16, 8, 24, 128]), "layers": rng.choice([1, 2, 5, 8]),
                "kv_heads": rng.choice([4, 2, 1]), "forks": rng.randint(0, requests // 2)}
    heads, key_heads = rng.choice([(48, 16), (48, 16), (32, 16), (8, 8)])
    return {"op": op, "requests": _log_int(rng, 1, 16), "nodes": _log_int(rng, 1, NODES), "width": width,
            "heads": heads, "key_heads": key_heads, "key_dim": rng.choice([128, 128, 128, 64, 96]),
            "value_dim": rng.choice([128, 128, 128, 64, 80]), "kernel": rng.choice([4, 4, 4, 3]),
            "blocked": rng.random() < 0.5, "ragged": rng.random() < 0.7}


# ---------------------------------------------------------------- lengths and trees
def _lengths(c):
    """(cached, nodes) of every request. Ragged batches spread both along a fixed sequence; every seventh
    request or so has no nodes."""
    R, most, cached = c["requests"], c["nodes"], c.get("cached", 0)
    if not c.get("ragged", True):
        return [cached] * R, [most] * R
    old, nodes = [], []
    for r in range(R):
        f, g = (0.618034 * r) % 1.0, (0.754878 * r) % 1.0
        old.append(int(round(cached * (1.0 - f))))
        nodes.append(0 if r % 7 == 6 else max(1, int(round(most * (1.0 - 0.8 * g)))))
    return old, nodes


def _parents(rng, n, width):
    """A tree of n nodes, none with more than `width` children; the first nodes have the most."""
    parent, count = [-1], [0]
    for i in range(1, n):
        p = min(i - 1, int(i * rng.random() ** 1.5))
        while count[p] >= width:
            p += 1
        parent.append(p)
        count.append(0)
        count[p] += 1
    return parent[:n]


def _forest(c, seed, nodes):
    rng = random.Random(int(seed) * 31 + 7)
    return [_parents(rng, n, c["width"]) for n in nodes]


def _q2_pages(cached, page):
    """Whether each of a request's pages was demoted: past the sink, wholly older than the recent window."""
    sink = -(-SINK // page) * page
    return [p * page >= sink and (p + 1) * page <= cached - RECENT for p in range(-(-cached // page))]


# ---------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 7919 + 41)
    return g


def _randn(g, *shape, std=1.0):
    return torch.randn(*shape, device=DEV, generator=g) * std


def _int32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


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


def _table(c, g, cached, total, max_pages, spare):
    """Page descriptors over a random order of slots, and the pools' slot counts."""
    page = c["page"]
    kinds = [[Q2 if p < len(old) and old[p] else Q4 for p in range(-(-t // page))]
             for old, t in zip([_q2_pages(a, page) for a in cached], total)]
    n2 = sum(k.count(Q2) for k in kinds)
    n4 = sum(len(k) for k in kinds) - n2
    slots4 = torch.randperm(n4 + spare, device=DEV, generator=g).cpu().numpy()
    slots2 = torch.randperm(n2 + 1, device=DEV, generator=g).cpu().numpy()
    desc, at = np.zeros((len(total), max_pages, 4), np.int32), {Q2: 0, Q4: 0}
    for r, ks in enumerate(kinds):
        for p, kind in enumerate(ks):
            desc[r, p] = (kind, (slots2 if kind == Q2 else slots4)[at[kind]], min(page, total[r] - p * page), p * page)
            at[kind] += 1
    return desc, n4 + spare, n2 + 1


def _starts(nodes):
    return np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32)


def _flat(forest):
    return _int32([p for parent in forest for p in parent])


def _inputs_tree(c, seed):
    cached, nodes = _lengths({**c, "cached": 9000})
    rows = sum(nodes) + 5  # rows behind the last request, as a padded batch has
    parents = torch.full((rows,), -1, dtype=torch.int32, device=DEV)
    parents[:sum(nodes)] = _flat(_forest(c, seed, nodes))
    return {"parents": parents, "row_starts": torch.from_numpy(_starts(nodes)).to(DEV),
            "tokens": _int32([a + n for a, n in zip(cached, nodes)]), "rows": rows,
            "masks": torch.zeros(rows, dtype=torch.int64, device=DEV),
            "positions": torch.zeros(rows, dtype=torch.int32, device=DEV),
            "depths": torch.zeros(c["requests"], dtype=torch.int32, device=DEV)}


def _mask_words(forest):
    """Per node its ancestors and itself as the bits of one word."""
    words = []
    for parent in forest:
        mine = []
        for i, p in enumerate(parent):
            mine.append((mine[p] if p >= 0 else 0) | 1 << i)
        words += [w - (1 << 64) if w >> 63 else w for w in mine]
    return words


def _inputs_attention(c, seed):
    g = _gen(seed)
    H, KV, cv, page = c["heads"], c["kv_heads"], c["kv_heads"] * HD, c["page"]
    cached, nodes = _lengths(c)
    total = [a + n for a, n in zip(cached, nodes)]
    max_pages = max(1, max(-(-t // page) for t in total))
    desc, n4, n2 = _table(c, g, cached, total, max_pages, 1)
    M, pad = sum(nodes), 5 if c["ragged"] else 0
    slot_map = [desc[r, np.arange(a, t) // page, 1] * page + np.arange(a, t) % page
                for r, (a, t) in enumerate(zip(cached, total))]
    slot_map = np.concatenate(slot_map + [np.full(pad, -1)]).astype(np.int32)
    masks = torch.zeros(M + pad, dtype=torch.int64, device=DEV)
    masks[:M] = torch.tensor(_mask_words(_forest(c, seed, nodes)), dtype=torch.int64, device=DEV)
    return {"q4": _cache_rows(g, Q4, n4 * page, cv), "q2": _cache_rows(g, Q2, n2 * page, cv),
            "descriptors": torch.from_numpy(desc).to(DEV), "slots": torch.from_numpy(slot_map).to(DEV),
            "row_starts": torch.from_numpy(_starts(nodes)).to(DEV), "tokens": _int32(total), "masks": masks,
            "most": max(nodes), "max_tokens": max(total), "rows": M, "q4_slots": n4,
            "query": _randn(g, M + pad, H, HD), "keys": _randn(g, M + pad, cv),
            "values": _randn(g, M + pad, cv, std=0.6), "out": torch.zeros(M + pad, H, HD, device=DEV)}


def _inputs_verify(c, seed):
    g = _gen(seed)
    _, nodes = _lengths(c)
    V, DV, M, width = c["vocab"], c["draft_vocab"] or c["vocab"], sum(nodes), c["width"]
    target = _randn(g, M, V, std=3.2)
    ids = torch.arange(V, device=DEV) if DV == V else torch.randperm(V, device=DEV, generator=g)[:DV].sort().values
    draft = (target[:, ids] + 0.9 * _randn(g, M, DV)).contiguous()
    inverse = torch.full((V,), -1, dtype=torch.int32, device=DEV)
    inverse[ids] = torch.arange(DV, dtype=torch.int32, device=DEV)
    # Children's tokens: the draft's best ones, or drawn from it.
    forest = _forest(c, seed, nodes)
    T = c["temperature"] or 1.0
    if c["drawn"] == WITH:
        pick = torch.multinomial(torch.softmax(draft / T, 1), width, replacement=True, generator=g)
    else:
        score = draft / T
        if c["drawn"] == WITHOUT:
            score = score - torch.log(-torch.log(torch.rand(M, DV, device=DEV, generator=g).clamp(1e-20, 1 - 1e-7)))
        pick = torch.topk(score, width, 1).indices
    row, rank, is_child, base = [], [], [], 0
    for parent in forest:
        seen = [0] * len(parent)
        for p in parent:
            row.append(base + max(p, 0))
            rank.append(seen[p] if p >= 0 else 0)
            is_child.append(p >= 0)
            if p >= 0:
                seen[p] += 1
        base += len(parent)
    tokens = ids[pick[torch.tensor(row, device=DEV), torch.tensor(rank, device=DEV)]]
    tokens = torch.where(torch.tensor(is_child, device=DEV), tokens,
                         torch.randint(0, V, (M,), device=DEV, generator=g)).to(torch.int32)
    R = c["requests"]
    return {"target": target, "draft": None if c["drawn"] == POINT else draft, "tokens": tokens,
            "inverse": None if DV == V else inverse, "parents": _flat(forest),
            "row_starts": torch.from_numpy(_starts(nodes)).to(DEV),
            "accept": torch.rand(M, device=DEV, generator=g), "sample": torch.rand(R, device=DEV, generator=g),
            "counts": torch.zeros(R, dtype=torch.int32, device=DEV), "next": torch.zeros(R, dtype=torch.int32, device=DEV),
            "path": torch.zeros(M, dtype=torch.int32, device=DEV), "most": max(nodes), "draft_vocab": DV}


def _kept(rng, n):
    """A path's nodes: the first m of the tree, then ones further on."""
    keep = rng.randint(1, min(n, 9))
    m = rng.randint(1, keep)
    if keep > m and n - keep < keep - m:
        m = keep
    return list(range(m)) + sorted(rng.sample(range(keep, n), keep - m))


def _inputs_pages(c, seed):
    g, rng = _gen(seed), random.Random(int(seed) * 17 + 3)
    page, R, cv, F = c["page"], c["requests"], c["kv_heads"] * HD, c["forks"]
    cached, nodes = _lengths(c)
    total = [a + n for a, n in zip(cached, nodes)]
    max_pages = max(-(-t // page) for t in total) + 2
    desc, n4, n2 = _table(c, g, cached, total, max_pages, F + 3)
    token_bytes = 2 * cv // 64 * 34
    pool = torch.randint(0, 256, (c["layers"], n4 * page, token_bytes), dtype=torch.uint8, device=DEV, generator=g)
    # Some requests have ended; those that go on are forked into their places.
    ended = sorted(rng.sample(range(R), F))
    going = [r for r in range(R) if r not in set(ended)]
    kept = [[] if r in set(ended) or not n else _kept(rng, n) for r, n in enumerate(nodes)]
    path = [kept[r] + [-1] * (nodes[r] - len(kept[r])) for r in range(R)]
    return {"pool": pool, "descriptors": torch.from_numpy(desc).to(DEV), "row_starts": torch.from_numpy(_starts(nodes)).to(DEV),
            "tokens": _int32(total), "counts": _int32([-1 if r in set(ended) else len(kept[r]) for r in range(R)]),
            "path": _int32([i for p in path for i in p]), "live": torch.zeros(R, dtype=torch.int32, device=DEV),
            "free4": torch.zeros(n4, dtype=torch.int32, device=DEV), "free2": torch.zeros(n2, dtype=torch.int32, device=DEV),
            "free_counts": torch.zeros(2, dtype=torch.int32, device=DEV), "most": max(nodes),
            "source": _int32([rng.choice(going) for _ in ended]), "target": _int32(ended),
            "commit_status": torch.zeros(R, dtype=torch.int32, device=DEV),
            "fork_status": torch.zeros(2, dtype=torch.int32, device=DEV), "token_bytes": token_bytes}


def _inputs_delta(c, seed):
    g, rng = _gen(seed), random.Random(int(seed) * 13 + 5)
    H, KH, dk, dv, K, R = c["heads"], c["key_heads"], c["key_dim"], c["value_dim"], c["kernel"], c["requests"]
    _, nodes = _lengths(c)
    forest, M = _forest(c, seed, nodes), sum(nodes)
    C = 2 * KH * dk + H * dv
    stride = C + H * dv + 2 * H  # q | k | v, the gate z, a, b
    proj = _randn(g, M, stride)
    # The accepted path: from the root down as far as it goes.
    path, counts = [], []
    for parent in forest:
        deep = [0] if parent else []
        while deep and rng.random() < 0.8:
            below = [i for i, p in enumerate(parent) if p == deep[-1]]
            if not below:
                break
            deep.append(rng.choice(below))
        counts.append(len(deep))
        path += deep + [-1] * (len(parent) - len(deep))
    S = -(-dv // 16)
    state = _randn(g, R, H, dk, dv, std=0.1)
    return {"proj": proj, "conv_w": _randn(g, C, K, std=0.4), "windows": _randn(g, R, C, K),
            "a_log": torch.log(0.05 + 0.95 * torch.rand(H, device=DEV, generator=g)),
            "dt_bias": -2.0 + _randn(g, H, std=0.5), "parents": _flat(forest), "path": _int32(path),
            "counts": _int32(counts), "row_starts": torch.from_numpy(_starts(nodes)).to(DEV),
            "state": _blocked(state) if c["blocked"] else state, "out": torch.zeros(M, H, dv, device=DEV),
            "state_out": torch.zeros((R, H, S, 256, 8) if c["blocked"] else (R, H, dk, dv), device=DEV),
            "windows_out": torch.zeros(R, C, K, device=DEV), "most": max(nodes), "channels": C}


def _blocked(s):
    """[..][key][value] states in the engine's order: runs of the eight rows i, i + 16, .. of a column."""
    R, H, dk, dv = s.shape
    S = -(-dv // 16)
    full = torch.zeros(R, H, 128, 16 * S, dtype=s.dtype, device=s.device)
    full[:, :, :dk, :dv] = s
    return full.view(R, H, 8, 16, S, 16).permute(0, 1, 4, 3, 5, 2).reshape(R, H, S, 256, 8).contiguous()


def _unblocked(s, dk, dv):
    R, H, S = s.shape[:3]
    return s.view(R, H, S, 16, 16, 8).permute(0, 1, 5, 3, 2, 4).reshape(R, H, 128, 16 * S)[:, :, :dk, :dv]


INPUTS = {"tree": _inputs_tree, "attention": _inputs_attention, "verify": _inputs_verify, "pages": _inputs_pages,
          "delta": _inputs_delta}


def prepare(case, seed):
    c = dict(case)
    s = {"case": c, **INPUTS[c["op"]](c, seed)}
    if own:  # the descriptions of the calls and the workspaces that a serving program keeps
        _keep(s)
    return s


# ---------------------------------------------------------------- the library's calls
def _bytes(n):
    return torch.empty(max(n, 16), dtype=torch.uint8, device=DEV)


def _keep(s):
    c, ctox = s["case"], _ctox()
    op, R = c["op"], c["requests"]

    def ptr(name):
        return None if s[name] is None else s[name].data_ptr()

    if op == "tree":
        s["call"] = ctox.TreePlan(
            d_row_starts=ptr("row_starts"), d_tokens=ptr("tokens"), d_parents=ptr("parents"), d_masks=ptr("masks"),
            d_positions=ptr("positions"), d_depths=ptr("depths"), requests=R, rows=s["rows"])
    elif op == "attention":
        KV, page, cv = c["kv_heads"], c["page"], c["kv_heads"] * HD
        b4, b2 = s["q4"].shape[1], s["q2"].shape[1]
        params = ctox.PagedGqaParams(c["heads"], KV, HD, s["max_tokens"], page, s["descriptors"].shape[1], 2 * cv, b2,
                                     b4, page * b2, page * b4, 1.0 / math.sqrt(HD))
        s["call"] = ctox.PagedGqaTree(
            d_query=ptr("query"), d_out=ptr("out"), d_q2_pages=ptr("q2"), d_q4_pages=ptr("q4"),
            d_descriptors=ptr("descriptors"), d_row_starts=ptr("row_starts"), d_tokens=ptr("tokens"),
            d_masks=ptr("masks"), rows=s["query"].shape[0], requests=R, max_rows=s["most"], params=params)
        s["workspace"] = _bytes(hip().paged_gqa_tree_workspace(s["call"]))
        s["call"].bind_workspace(s["workspace"].data_ptr(), s["workspace"].numel())
    elif op == "verify":
        s["call"] = ctox.VerifyTree(
            d_target=ptr("target"), d_draft=ptr("draft"), d_draft_inverse=ptr("inverse"), d_tokens=ptr("tokens"),
            d_parents=ptr("parents"), d_row_starts=ptr("row_starts"), d_accept_draws=ptr("accept"),
            d_sample_draws=ptr("sample"), d_counts=ptr("counts"), d_path=ptr("path"), d_next=ptr("next"),
            requests=R, rows=s["target"].shape[0], vocab=c["vocab"], draft_vocab=s["draft_vocab"],
            max_children=c["width"], without_replacement=c["drawn"] == WITHOUT, temperature=c["temperature"])
        s["workspace"] = _bytes(hip().verify_tree_workspace(s["call"]))
        s["call"].bind_workspace(s["workspace"].data_ptr(), s["workspace"].numel())
    elif op == "pages":
        pools = [s["pool"][i].data_ptr() for i in range(c["layers"])]
        page_bytes, max_pages = c["page"] * s["token_bytes"], s["descriptors"].shape[1]
        geometry = {"requests": R, "page_tokens": c["page"], "max_pages": max_pages, "q4_slots": s["free4"].numel()}
        s["commit"] = ctox.PagedCommit(
            q4_pools=pools, d_descriptors=ptr("descriptors"), d_row_starts=ptr("row_starts"), d_tokens=ptr("tokens"),
            d_counts=ptr("counts"), d_path=ptr("path"), d_new_tokens=ptr("live"), d_status=ptr("commit_status"),
            rows=s["path"].numel(), token_bytes=s["token_bytes"], q4_page_bytes=page_bytes, **geometry)
        s["free"] = ctox.PagedFreeSlots(
            d_descriptors=ptr("descriptors"), d_tokens=ptr("live"), d_q4_free=ptr("free4"), d_q2_free=ptr("free2"),
            d_counts=ptr("free_counts"), q2_slots=s["free2"].numel(), **geometry)
        s["workspace"] = _bytes(hip().paged_free_slots_workspace(s["free"]))
        s["free"].bind_workspace(s["workspace"].data_ptr(), s["workspace"].numel())
        s["fork"] = ctox.PagedFork(
            q4_pools=pools, d_descriptors=ptr("descriptors"), d_tokens=ptr("live"), d_sources=ptr("source"),
            d_targets=ptr("target"), d_free_slots=ptr("free4"), d_free_count=ptr("free_counts"),
            d_status=ptr("fork_status"), forks=c["forks"], token_bytes=s["token_bytes"], q4_page_bytes=page_bytes,
            **geometry)
    else:
        H, KH, dk, dv = c["heads"], c["key_heads"], c["key_dim"], c["value_dim"]
        C = s["channels"]
        s["call"] = ctox.GdnTree(
            d_proj=ptr("proj"), d_conv_w=ptr("conv_w"), d_conv_in=ptr("windows"), d_a_log=ptr("a_log"),
            d_dt_bias=ptr("dt_bias"), d_state_in=ptr("state"), d_row_starts=ptr("row_starts"),
            d_parents=ptr("parents"), d_out=ptr("out"), d_counts=ptr("counts"), d_path=ptr("path"),
            d_conv_out=ptr("windows_out"), d_state_out=ptr("state_out"), proj_stride=s["proj"].shape[1],
            a_off=C + H * dv, b_off=C + H * dv + H, requests=R, rows=s["proj"].shape[0], max_rows=s["most"], heads=H,
            key_heads=KH, key_dim=dk, value_dim=dv, kernel=c["kernel"], blocked=c["blocked"])
        s["workspace"] = _bytes(hip().gdn_tree_workspace(s["call"]))
        s["call"].bind_workspace(s["workspace"].data_ptr(), s["workspace"].numel())


def _run_own(s):
    c, st = s["case"], _stream()
    op = c["op"]
    if op == "tree":
        hip().tree_plan_device(s["call"], st)
        return {k: s[k] for k in ("masks", "positions", "depths")}
    if op == "attention":
        cv = c["kv_heads"] * HD
        hip().kv_append_q4_device(s["q4"].data_ptr(), s["keys"].data_ptr(), s["values"].data_ptr(),
                                  s["slots"].data_ptr(), s["query"].shape[0], cv, c["page"], s["q4_slots"],
                                  c["page"] * s["q4"].shape[1], stream=st)
        hip().paged_gqa_tree_device(s["call"], st)
        return {"out": s["out"], "cache": s["q4"]}
    if op == "verify":
        hip().verify_tree_device(s["call"], st)
        return {k: s[k] for k in ("counts", "path", "next")}
    if op == "pages":
        hip().paged_commit_device(s["commit"], st)
        hip().paged_free_slots_device(s["free"], st)
        hip().paged_fork_device(s["fork"], st)
        return {k: s[k] for k in PAGED}
    hip().gdn_tree_device(s["call"], st)
    hip().gdn_tree_commit_device(s["call"], st)
    return {"out": s["out"], "state": s["state_out"], "windows": s["windows_out"]}


PAGED = ("pool", "descriptors", "live", "free4", "free2", "free_counts", "commit_status", "fork_status")


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


def _rows_of(starts, rows):
    """Every row's request (of rows behind the last: the last), and its number in it."""
    i = torch.arange(rows, device=DEV)
    R = starts.numel() - 1
    r = torch.searchsorted(starts[1:].contiguous(), i, right=True).clamp(max=R - 1)
    return r, i - starts[r]


def _lineage(parents, starts, rows):
    """A row's ancestors and itself, [rows][NODES] by their numbers in its request, and its parent's row or -1."""
    r, local = _rows_of(starts, rows)
    up = torch.where((parents >= 0) & (parents < local), starts[r] + parents, -1)
    seen = torch.nn.functional.one_hot(local.clamp(max=NODES - 1), NODES).bool()
    jump = up
    for _ in range(6):  # 1, 2, 4 .. generations
        seen = seen | (seen[jump] & (jump >= 0)[:, None])
        jump = torch.where(jump >= 0, jump[jump], -1)
    return seen, up


def _plain_tree(s):
    starts, rows = s["row_starts"].long(), s["rows"]
    seen, _ = _lineage(s["parents"].long(), starts, rows)
    r, local = _rows_of(starts, rows)
    inside = torch.arange(rows, device=DEV) < starts[-1]
    depth = seen.sum(1) - 1
    bits = torch.where(seen, torch.ones(1, dtype=torch.int64, device=DEV) << torch.arange(NODES, device=DEV), 0)
    past = s["tokens"].long() - (starts[1:] - starts[:-1])
    zero = torch.zeros_like(depth)
    depths = torch.zeros_like(past).scatter_reduce(0, r, torch.where(inside, depth + 1, zero), "amax")
    return {"masks": torch.where(inside, bits.sum(1), zero),
            "positions": torch.where(inside, past[r] + depth, zero).to(torch.int32),
            "depths": depths.to(torch.int32)}


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
    # every request's nodes, padded to the most
    n, i = s["most"], torch.arange(s["most"], device=DEV)
    starts = s["row_starts"].long()
    count = starts[1:] - starts[:-1]
    src = (starts[:-1, None] + i).clamp(max=max(M - 1, 0))
    q = s["query"][src].view(R, n, KV, H // KV, HD).permute(0, 2, 1, 3, 4).reshape(R, KV, -1, HD)
    node = j - (s["tokens"].long() - count)[:, None]                            # [R][tokens]: a token's node
    bit = (s["masks"][src][..., None] >> node.clamp(0, 63)[:, None]) & 1 == 1    # [R][n][tokens]
    visible = ((node < 0)[:, None] | bit) & present[:, None]
    x = (q @ k.transpose(2, 3)).view(R, KV, n, H // KV, -1) * (1.0 / math.sqrt(HD))
    x = x.masked_fill(~visible[:, None, :, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    o = (p.view(R, KV, -1, p.shape[-1]) @ v).view(R, KV, n, H // KV, HD) / torch.where(total > 0, total, 1.0)
    out = torch.zeros_like(s["out"])
    mine = i < count[:, None]
    out[src[mine]] = o.permute(0, 2, 1, 3, 4).reshape(R, n, H, HD)[mine]
    return {"out": out, "cache": s["q4"]}


def _plain_verify(s):
    c = s["case"]
    M, V, W, R = s["target"].shape[0], c["vocab"], c["width"], c["requests"]
    starts, tokens, u = s["row_starts"].long(), s["tokens"].long(), s["accept"].double()
    seen, up = _lineage(s["parents"].long(), starts, M)
    r, local = _rows_of(starts, M)
    row = torch.arange(M, device=DEV)
    # child[w]: every row's child number w, or -1
    same = (up[:, None] == up[None]) & (up >= 0)[:, None] & (row[None] < row[:, None])
    rank = same.sum(1)
    child = torch.full((W, M + 1), -1, device=DEV)
    child[rank.clamp(max=W - 1), torch.where((up >= 0) & (rank < W), up, M)] = row
    child = child[:, :M]
    chosen = torch.full((M,), -1, device=DEV)
    if c["temperature"] == 0.0:
        best = s["target"].argmax(1)
        for k in range(W - 1, -1, -1):
            chosen = torch.where((child[k] >= 0) & (tokens[child[k]] == best), child[k], chosen)
    else:
        p = torch.softmax(s["target"].double() / c["temperature"], 1)
        lam, undrawn, left = (torch.full((M,), x, dtype=torch.float64, device=DEV) for x in (0.0, 1.0, 1.0))
        point = s["draft"] is None
        rest = p.clone()
        if not point:
            q = torch.softmax(s["draft"].double() / c["temperature"], 1)
            if s["inverse"] is not None:
                q = torch.where(s["inverse"] >= 0, q[:, s["inverse"].clamp(min=0).long()], 0.0)
        offered = torch.ones(M, dtype=torch.bool, device=DEV)
        for k in range(W):
            offered &= (child[k] >= 0) & (chosen < 0) & (undrawn > LEAST_MASS)
            t = tokens[child[k]]
            qt = torch.ones_like(left) if point else q[row, t]
            yes = offered & (u[child[k]] * (qt / undrawn) * left < rest[row, t])
            chosen = torch.where(yes, child[k], chosen)
            no = offered & ~yes
            if point:
                rest[row, t] = torch.where(no, 0.0, rest[row, t])
            else:
                lam = torch.where(no, lam + left / undrawn, lam)
                undrawn = torch.where(no & (c["drawn"] == WITHOUT), undrawn - qt, undrawn)
                rest = torch.where(no[:, None], (p - lam[:, None] * q).clamp(min=0.0), rest)
            left = rest.sum(1)
    # a node is accepted where every step on its path was
    step = (local == 0) | ((up >= 0) & (chosen[up] == row))
    wrong = torch.zeros(R * NODES, dtype=torch.bool, device=DEV)
    wrong[(r * NODES + local)[~step]] = True
    on = ~(seen & wrong.view(R, NODES)[r]).any(1)
    counts = torch.zeros(R, dtype=torch.long, device=DEV).index_add(0, r, on.long())
    path = torch.full((M + 1,), -1, device=DEV)
    path[torch.where(on, starts[r] + seen.sum(1) - 1, M)] = local
    last = torch.full((R,), -1, device=DEV).scatter_reduce(0, r, torch.where(on, row, -1), "amax")
    there, last = last >= 0, last.clamp(min=0)
    if c["temperature"] == 0.0:
        token = best[last]
    else:
        w = torch.where((left[last] > 0.0)[:, None], rest[last], p[last])
        running = torch.cumsum(w, 1)
        token = (running <= s["sample"].double()[:, None] * running[:, -1:]).sum(1)
    token = torch.where(there, token, -1)
    return {"counts": counts.to(torch.int32), "path": path[:M].to(torch.int32), "next": token.to(torch.int32)}


def _plain_pages(s):
    c = s["case"]
    page, R, desc, starts = c["page"], c["requests"], s["descriptors"], s["row_starts"].long()
    tokens, counts = s["tokens"].long(), s["counts"].long()
    nodes = starts[1:] - starts[:-1]
    past = tokens - nodes
    # kept tokens to their places
    i = torch.arange(s["path"].numel(), device=DEV)
    r, j = _rows_of(starts, i.numel())
    live = j < counts[r]
    slot = desc[..., 1].long()

    def place(position):
        return slot[r, position // page] * page + position % page

    src, dst = place(past[r] + s["path"].long().clamp(min=0)), place(past[r] + j)
    src = torch.where(live, src, dst)
    s["pool"][:, dst] = s["pool"][:, src]
    length = torch.where(counts < 0, 0, past + counts)
    first = torch.arange(desc.shape[1], device=DEV) * page
    cut = (length[:, None] - first).clamp(0, page).to(torch.int32)
    desc[..., 2] = torch.where(first < tokens[:, None], cut, desc[..., 2])
    # slots that no live page holds
    held = first < length[:, None]
    lists, found = [], []
    for kind, name in ((Q4, "free4"), (Q2, "free2")):
        n = s[name].numel()
        used = torch.zeros(n + 1, dtype=torch.bool, device=DEV)
        used[torch.where(held & ((desc[..., 0] != 0) == (kind == Q4)), slot, n)] = True
        free = ~used[:n]
        at = torch.cumsum(free, 0) - 1
        out = torch.full((n + 1,), -1, dtype=torch.int32, device=DEV)
        out[torch.where(free, at, n)] = torch.arange(n, dtype=torch.int32, device=DEV)
        lists.append(out[:n])
        found.append(free.sum())
    # forks: full pages shared, a part-filled one copied
    a, b = s["source"].long(), s["target"].long()
    part = length[a] % page
    order = torch.cumsum(part > 0, 0) - (part > 0).long()
    fresh = lists[0].long()[order.clamp(max=lists[0].numel() - 1)]
    end = length[a] // page
    rows = torch.where(held[a][..., None], desc[a], desc[b])
    tail = (torch.arange(desc.shape[1], device=DEV) == end[:, None]) & (part > 0)[:, None]
    rows[..., 1] = torch.where(tail, fresh[:, None].to(torch.int32), rows[..., 1])
    t = torch.arange(page, device=DEV)
    some = (t < part[:, None])
    came = (slot[a, end.clamp(max=desc.shape[1] - 1)][:, None] * page + t)[some]
    goes = (fresh[:, None] * page + t)[some]
    s["pool"][:, goes] = s["pool"][:, came]
    desc[b] = rows
    length = length.index_copy(0, b, length[a])
    zero = torch.zeros_like(found[0])
    return {"pool": s["pool"], "descriptors": desc, "live": length.to(torch.int32), "free4": lists[0],
            "free2": lists[1], "free_counts": torch.stack(found).to(torch.int32),
            "commit_status": torch.zeros(R, dtype=torch.int32, device=DEV),
            "fork_status": torch.stack([zero, (part > 0).sum()]).to(torch.int32)}


def _taps(up, depth, windows, r, x, K):
    """A node's inputs of the last K positions, [K][rows][channels]: ancestors', then the window's."""
    at, inputs = torch.arange(up.numel(), device=DEV), []
    for t in range(K):
        old = windows[r, :, (K - t + depth).clamp(max=K - 1)]
        inputs.append(torch.where((at >= 0)[:, None], x[at], old))
        at = torch.where(at >= 0, up[at], -1)
    return torch.stack(inputs)


def _plain_delta(s):
    c = s["case"]
    H, KH, dk, dv, K, R, C, M = (c["heads"], c["key_heads"], c["key_dim"], c["value_dim"], c["kernel"], c["requests"],
                                 s["channels"], s["proj"].shape[0])
    starts, n = s["row_starts"].long(), s["most"]
    seen, up = _lineage(s["parents"].long(), starts, M)
    r, local = _rows_of(starts, M)
    depth = seen.sum(1) - 1
    x = s["proj"][:, :C]
    taps = _taps(up, depth, s["windows"], r, x, K)
    y = (taps * s["conv_w"].T.flip(0)[:, None]).sum(0)
    y = y * torch.sigmoid(y)
    unit = [y[:, i * KH * dk:(i + 1) * KH * dk].view(M, KH, dk) for i in range(2)]
    q, k = ((z / torch.sqrt((z * z).sum(-1, keepdim=True) + 1e-6)).repeat_interleave(H // KH, 1) for z in unit)
    v = y[:, 2 * KH * dk:].view(M, H, dv)
    g = s["proj"][:, C + H * dv:C + H * dv + H] + s["dt_bias"]
    decay = -torch.exp(s["a_log"]) * torch.where(g > 20.0, g, torch.log1p(torch.exp(g.clamp(max=20.0))))
    beta = torch.sigmoid(s["proj"][:, C + H * dv + H:])
    # requests padded to the most nodes
    here = torch.zeros(R, n, dtype=torch.bool, device=DEV)
    here[r, local] = True

    def pad(z):
        return torch.zeros(R, n, *z.shape[1:], device=DEV, dtype=z.dtype).index_put((r, local), z)

    q, k, v, decay, beta = (pad(z).transpose(1, 2) for z in (q * dk ** -0.5, k, v, decay, beta))  # [R][H][n][..]
    line = pad(seen[:, :n])                                                     # [R][n][n]
    L = line.float()[:, None] @ decay[..., None]                                # [R][H][n][1]
    away = torch.exp((L - L.transpose(2, 3)).masked_fill(~line[:, None], -math.inf))
    state = _unblocked(s["state"], dk, dv) if c["blocked"] else s["state"]
    delta = beta[..., None] * (v - torch.exp(L) * (k @ state))
    kk = beta[..., None] * away * (k @ k.transpose(2, 3))
    for i in range(1, n):
        delta[:, :, i] -= (kk[:, :, i, None, :i] @ delta[:, :, :i])[:, :, 0]
    o = torch.exp(L) * (q @ state) + (away * (q @ k.transpose(2, 3))) @ delta
    # the state behind the accepted path
    counts = s["counts"].long()
    last = (starts[:-1] + s["path"].long()[(starts[:-1] + counts - 1).clamp(0, M - 1)]).clamp(0, M - 1)
    some, end = counts > 0, local[last]
    on = line[torch.arange(R, device=DEV), end] & some[:, None]
    g = L[torch.arange(R, device=DEV), :, end]                                  # [R][H][1]
    w = torch.exp((g - L[..., 0]).masked_fill(~on[:, None], -math.inf))
    after = torch.exp(g)[..., None] * state + (k * w[..., None]).transpose(2, 3) @ delta
    after = torch.where(some[:, None, None, None], after, state)
    windows = torch.where(some[:, None, None], taps[:, last].flip(0).permute(1, 2, 0), s["windows"])
    return {"out": o.transpose(1, 2)[r, local], "state": _blocked(after) if c["blocked"] else after,
            "windows": windows.contiguous()}


PLAIN = {"tree": _plain_tree, "attention": _plain_attention, "verify": _plain_verify, "pages": _plain_pages,
         "delta": _plain_delta}


def run(state):
    if own:
        return _run_own(state)
    return PLAIN[state["case"]["op"]](state)


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


def _exact_attention(c, seed, i):
    H, KV, page, cv = c["heads"], c["kv_heads"], c["page"], c["kv_heads"] * HD
    G, (cached, nodes) = H // KV, _lengths(c)
    forest = _forest(c, seed, nodes)
    out = torch.zeros(i["out"].shape, dtype=torch.float64, device=DEV)
    at = 0
    for r in range(c["requests"]):
        n, old = nodes[r], cached[r]
        if n == 0:
            continue
        j = torch.arange(old, device=DEV)
        d = i["descriptors"][r].long()[j // page]
        where = d[:, 1] * page + j % page
        kv = torch.zeros(old + n, 2 * cv, dtype=torch.float64, device=DEV)
        is4, is2 = (d[:, 0] == Q4).nonzero()[:, 0], (d[:, 0] == Q2).nonzero()[:, 0]
        kv[is4] = _values64(i["q4"][where[is4]].unflatten(-1, (-1, 34)), Q4).flatten(1)
        kv[is2] = _values64(i["q2"][where[is2]].unflatten(-1, (-1, 18)), Q2).flatten(1)
        fresh = torch.cat([i["keys"][at:at + n], i["values"][at:at + n]], 1)
        kv[old:] = _stored64(fresh.view(n, -1, 64)).flatten(1)
        hidden = torch.ones(n, old + n, dtype=torch.bool)
        hidden[:, :old] = False
        for t in range(n):
            a = t
            while a >= 0:
                hidden[t, old + a] = False
                a = forest[r][a]
        hidden = hidden.to(DEV)
        for h in range(KV):
            k, v = kv[:, h * HD:(h + 1) * HD], kv[:, cv + h * HD:cv + (h + 1) * HD]
            for g in range(G):
                x = i["query"][at:at + n, h * G + g].double() @ k.T / 16.0
                out[at:at + n, h * G + g] = torch.softmax(x.masked_fill_(hidden, -math.inf), -1) @ v
        at += n
    return {"out": out, "cache": None}


def _exact_delta(c, seed, i):
    H, KH, dk, dv, K, C = c["heads"], c["key_heads"], c["key_dim"], c["value_dim"], c["kernel"], i["channels"]
    _, nodes = _lengths(c)
    forest = _forest(c, seed, nodes)
    S0 = (_unblocked(i["state"], dk, dv) if c["blocked"] else i["state"]).double()
    proj, weight, windows = i["proj"].double(), i["conv_w"].double(), i["windows"].double()
    scale = -torch.exp(i["a_log"].double())
    path, counts = i["path"].tolist(), i["counts"].tolist()
    out = torch.zeros(i["out"].shape, dtype=torch.float64, device=DEV)
    after, slid, at = S0.clone(), windows.clone(), 0
    for r, parent in enumerate(forest):
        end = path[at + counts[r] - 1] if counts[r] else -1
        states, slides = [], []
        for t, p in enumerate(parent):
            S, win = (states[p], slides[p]) if p >= 0 else (S0[r], windows[r])
            row = proj[at + t]
            win = torch.cat([win[:, 1:], row[:C, None]], 1)
            y = (win * weight).sum(1)
            y = y / (1.0 + torch.exp(-y))
            q, k = y[:KH * dk].view(KH, dk), y[KH * dk:2 * KH * dk].view(KH, dk)
            q = (q / torch.sqrt(q.square().sum(1, keepdim=True) + 1e-6)).repeat_interleave(H // KH, 0)
            k = (k / torch.sqrt(k.square().sum(1, keepdim=True) + 1e-6)).repeat_interleave(H // KH, 0)
            v = y[2 * KH * dk:].view(H, dv)
            g = torch.nn.functional.softplus(row[C + H * dv:C + H * dv + H] + i["dt_bias"].double(), threshold=40.0)
            beta = torch.sigmoid(row[C + H * dv + H:])
            S = S * torch.exp(scale * g)[:, None, None]
            error = (v - (S * k[:, :, None]).sum(1)) * beta[:, None]
            S = S + k[:, :, None] * error[:, None, :]
            out[at + t] = (S * q[:, :, None]).sum(1) / math.sqrt(dk)
            states.append(S)
            slides.append(win)
        if end >= 0:
            after[r], slid[r] = states[end], slides[end]
        at += len(parent)
    return {"out": out, "state": _blocked(after) if c["blocked"] else after, "windows": slid}


def exact(case, seed):
    c = dict(case)
    if c["op"] not in ("attention", "delta"):
        return None  # whole numbers, and bytes that are moved
    i = INPUTS[c["op"]](c, seed)
    return {"attention": _exact_attention, "delta": _exact_delta}[c["op"]](c, seed, i)


# ---------------------------------------------------------------- work
def work(case):
    c = dict(case)
    op = c["op"]
    cached, nodes = _lengths(c)
    M, R = sum(nodes), c["requests"]
    if op == "tree":
        return {"bytes": 16 * M + 8 * R, "flops": 0}
    if op == "attention":
        H, cv, page = c["heads"], c["kv_heads"] * HD, c["page"]
        moved = pairs = 0
        for a, n in zip(cached, nodes):
            if n:
                moved += sum(min(page, a - p * page) * 2 * cv // 64 * (18 if q2 else 34)
                             for p, q2 in enumerate(_q2_pages(a, page)))
                pairs += n * (a + 1)  # (and the ancestors, a few each)
        # new rows: K / V read and stored, the query read, the output written
        moved += M * (8 * cv + 2 * cv // 64 * 34 + 8 * H * HD)
        return {"bytes": moved, "flops": 4 * HD * H * pairs}
    if op == "verify":
        drafts = 0 if c["drawn"] == POINT or c["temperature"] == 0.0 else c["draft_vocab"] or c["vocab"]
        return {"bytes": 4 * M * (c["vocab"] + drafts), "flops": 4 * M * (c["vocab"] + drafts)}
    if op == "pages":
        page, token = c["page"], 2 * c["kv_heads"] * HD // 64 * 34
        pages = sum(-(-(a + n) // page) for a, n in zip(cached, nodes))
        # a few tokens of every request move in every layer, half a page of every fork
        moved = c["layers"] * token * (2 * (R - c["forks"]) + c["forks"] * page // 2)
        return {"bytes": 2 * moved + 36 * pages + 8 * M, "flops": 0}
    H, KH, dk, dv, K = c["heads"], c["key_heads"], c["key_dim"], c["value_dim"], c["kernel"]
    C = 2 * KH * dk + H * dv
    # states and windows read twice (by the rows and by the path) and written once; rows read, written
    moved = R * 4 * (3 * H * dk * dv + 3 * C * K) + 4 * M * (C + 2 * H + H * dv)
    return {"bytes": moved, "flops": M * H * 4 * dk * dv + sum(n * n for n in nodes) * H * 2 * (dk + dv) // 2}
