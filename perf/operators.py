"""The serving operators around a paged key / value cache, as cases that can be timed and compared: attention
inside a sliding window with sinks (a whole prompt, or one token per user), attention of a tree of drafted tokens,
committing the accepted drafts, copying cache blocks, and sampling from a row of logits.

`run` computes a case in plain torch (32 bits, 64 where a sum has to be told from a border) while `own` is false,
and through the kernel library (include/ttb_kernels.h) while it is true; `exact` is the definition in 64 bits.
"""

import ctypes
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_TAGS = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}     # TTB_DTYPE_*


# ---------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # One user verifies a short draft: the latency of a single speculative step.
        dict(name="tree_one_user", op="tree", users=1, nodes=8, heads=32, kv_heads=8, dim=128, ctx=1000, block=32, dtype="bf16",
             window=0, sinks=0),
        # A loaded server: sixteen users of different lengths, trees of up to 31 nodes.
        dict(name="tree_server", op="tree", users=16, nodes=31, heads=32, kv_heads=8, dim=128, ctx=8192, block=64, dtype="bf16",
             window=0, sinks=0),
        # One token of one chat on a model with one key head per query head and an odd window.
        dict(name="window_decode_one_user", op="window_decode", users=1, heads=8, kv_heads=8, dim=64, ctx=1501, block=16,
             dtype="f16", window=1000, sinks=4),
        # A full decode batch deep in long conversations: the window bounds what is read.
        dict(name="window_decode_batch", op="window_decode", users=64, heads=32, kv_heads=8, dim=128, ctx=16384, block=64,
             dtype="bf16", window=4096, sinks=16),
        # Two short prompts of odd length, the second padded, continued behind 700 cached tokens.
        dict(name="window_prompt_chunk", op="window", users=2, heads=12, kv_heads=4, dim=64, queries=837, keys=1537, offset=700,
             dtype="f16", window=300, sinks=4, ragged=True),
        # A long document with the decoder block's heads.
        dict(name="window_prompt_long", op="window", users=1, heads=32, kv_heads=8, dim=128, queries=16384, keys=16384, offset=0,
             dtype="bf16", window=2048, sinks=64, ragged=False),
        # One sequence forks: its last, half-filled block is duplicated in the two caches of one layer.
        dict(name="copy_fork_one_layer", op="copy", caches=2, blocks=64, kv_heads=8, block=32, dim=128, pairs=1, dtype="bf16"),
        # Beams of a whole model are reordered: 96 blocks in the caches of sixteen layers.
        dict(name="copy_fork_model", op="copy", caches=32, blocks=256, kv_heads=8, block=32, dim=128, pairs=96, dtype="bf16"),
        # The accepted path of one user's draft, one layer, odd blocks.
        dict(name="commit_one_user", op="commit", caches=2, users=1, nodes=8, kv_heads=8, dim=64, ctx=1000, block=24, dtype="f16"),
        # The accepted paths of a full batch in all layers.
        dict(name="commit_model", op="commit", caches=32, users=48, nodes=31, kv_heads=8, dim=128, ctx=256, block=32, dtype="bf16"),
        # One chat samples its next token.
        dict(name="sample_one_row", op="sample", rows=1, vocab=32000, dtype="bf16", mode="mixed"),
        # A full batch with a large vocabulary and 32-bit logits, every row with its own settings.
        dict(name="sample_batch", op="sample", rows=256, vocab=128000, dtype="f32", mode="mixed"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tree", "tree", "window_decode", "window_decode", "window", "window", "copy", "commit", "sample", "sample"])
    kind = rng.choice(["bf16", "bf16", "f16"])
    kv_heads = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 4, 6, 8])
    dim = rng.choice([64, 128, 128, 256])
    block = rng.choice([8, 16, 24, 32, 64, 100, 128])
    if op == "tree":
        c = dict(op=op, users=_log_int(rng, 1, 16), nodes=rng.randint(1, 64), heads=kv_heads * group, kv_heads=kv_heads, dim=dim,
                 ctx=_log_int(rng, 1, 8192), block=block, dtype=kind)
        c["window"] = rng.choice([0, 0, _log_int(rng, 1, 4096)])
        c["sinks"] = rng.randint(0, 64) if c["window"] else 0
        limit = 16 * 31 * 32 * 128 * 8192
        cost = c["users"] * c["nodes"] * c["heads"] * dim
        c["ctx"] = max(1, min(c["ctx"], limit // cost))
        return c
    if op == "window_decode":
        c = dict(op=op, users=_log_int(rng, 1, 64), heads=kv_heads * group, kv_heads=kv_heads, dim=dim, ctx=_log_int(rng, 1, 16384),
                 block=block, dtype=kind, window=_log_int(rng, 1, 8192), sinks=rng.choice([0, 1, 4, 16, 100]))
        limit = 64 * 8 * 128 * 16384
        c["ctx"] = max(1, min(c["ctx"], limit // (c["users"] * kv_heads * dim)))
        return c
    if op == "window":
        kind = rng.choice(["bf16", "bf16", "bf16", "f16", "f16", "f32"])
        c = dict(op=op, users=rng.randint(1, 4), heads=kv_heads * group, kv_heads=kv_heads, dim=dim, dtype=kind,
                 queries=_log_int(rng, 1, 8192 if kind != "f32" else 512), window=_log_int(rng, 1, 4096), sinks=rng.choice([0, 1, 4, 64, 200]),
                 ragged=rng.random() < 0.5)
        c["queries"] = max(1, min(c["queries"], int(math.sqrt(32 * 128 * 8192.0 ** 2 / (c["users"] * c["heads"] * dim)))))
        c["offset"] = rng.choice([0, 0, rng.randint(0, 1500)])
        c["keys"] = c["offset"] + c["queries"]
        return c
    if op == "copy":
        c = dict(op=op, caches=rng.randint(1, 32), blocks=rng.randint(4, 256), kv_heads=kv_heads, block=block, dim=dim, dtype=kind)
        c["blocks"] = max(4, min(c["blocks"], (1 << 28) // (c["caches"] * kv_heads * block * dim)))
        c["pairs"] = rng.randint(1, min(96, c["blocks"] // 2))
        return c
    if op == "commit":
        return dict(op=op, caches=rng.randint(1, 32), users=_log_int(rng, 1, 48), nodes=rng.randint(1, 64), kv_heads=kv_heads, dim=min(dim, 128),
                    ctx=rng.randint(0, 256), block=min(block, 32), dtype=kind)
    return dict(op="sample", rows=_log_int(rng, 1, 256), vocab=_log_int(rng, 2, 128000), dtype=rng.choice(["bf16", "f16", "f32"]),
                mode=rng.choice(["mixed", "mixed", "plain", "top_k", "top_p", "greedy"]))


# ---------------------------------------------------------------------------------------------- inputs
def _randn(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * scale).to(dtype)


def _page_table(gen, users, pages, used, spare):
    """A table of distinct blocks in random order; -1 where a user has no block yet."""
    order = torch.randperm(users * pages + spare, generator=gen, device="cuda")[:users * pages].to(torch.int32).view(users, pages)
    column = torch.arange(pages, device="cuda")
    return torch.where(column[None, :] < used[:, None], order, torch.full_like(order, -1)).contiguous()


def _lengths(gen, users, most):
    """Cached tokens per user, between half of `most` and all of it; the first user has all."""
    n = torch.randint((most + 1) // 2, most + 1, (users,), generator=gen, device="cuda", dtype=torch.int32)
    n[0] = most
    return n


def _trees(gen, users, nodes):
    """parents[b, t] < t: node 0 hangs on the cached text, later nodes on a recent earlier node (or on the text)."""
    t = torch.arange(nodes, device="cuda").expand(users, nodes)
    back = 1 + (torch.rand(users, nodes, generator=gen, device="cuda") ** 2 * torch.clamp(t, max=6)).floor().long()
    return torch.clamp(t - back, min=-1).to(torch.int32).contiguous()


def _inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed * 7919 + 17)
    c = dict(case)
    s = {"case": c}
    if c["op"] in ("tree", "window_decode"):
        dt = _DTYPES[c["dtype"]]
        users, heads, kvh, dim, block = c["users"], c["heads"], c["kv_heads"], c["dim"], c["block"]
        pages = (c["ctx"] + block - 1) // block
        lens = _lengths(gen, users, c["ctx"])
        s["table"] = _page_table(gen, users, pages, (lens + block - 1) // block, 3)
        blocks = users * pages + 3
        s["k"] = torch.empty(blocks, kvh, block, dim, device="cuda", dtype=dt).normal_(generator=gen)
        s["v"] = torch.empty(blocks, kvh, block, dim, device="cuda", dtype=dt).normal_(generator=gen)
        if c["op"] == "tree":
            nodes = c["nodes"]
            s["lens"] = lens
            s["q"] = _randn(gen, (users, nodes, heads, dim), dt)
            s["kd"] = _randn(gen, (users, nodes, kvh, dim), dt)
            s["vd"] = _randn(gen, (users, nodes, kvh, dim), dt)
            s["parents"] = _trees(gen, users, nodes)
        else:
            s["pos"] = lens - 1
            s["q"] = _randn(gen, (1, users, heads, dim), dt)
        s["out"] = torch.zeros_like(s["q"])
    elif c["op"] == "window":
        dt = _DTYPES[c["dtype"]]
        users, heads, kvh, dim = c["users"], c["heads"], c["kv_heads"], c["dim"]
        s["q"] = _randn(gen, (users, heads, c["queries"], dim), dt)
        s["k"] = _randn(gen, (users, kvh, c["keys"], dim), dt)
        s["v"] = _randn(gen, (users, kvh, c["keys"], dim), dt)
        s["lens"] = _lengths(gen, users, c["keys"]) if c["ragged"] else None
        s["out"] = torch.zeros_like(s["q"])
    elif c["op"] == "copy":
        dt = _DTYPES[c["dtype"]]
        s["caches"] = [torch.empty(c["blocks"], c["kv_heads"], c["block"], c["dim"], device="cuda", dtype=dt).normal_(generator=gen)
                       for _ in range(c["caches"])]
        order = torch.randperm(c["blocks"], generator=gen, device="cuda").to(torch.int32)
        dst = order[:c["pairs"]]
        rest = order[c["pairs"]:]
        src = rest[torch.randint(0, rest.numel(), (c["pairs"],), generator=gen, device="cuda")]  # a block may fork many times
        s["pairs"] = torch.stack([src, dst], dim=1).contiguous()
        s["ptrs"] = (ctypes.c_void_p * c["caches"])(*[t.data_ptr() for t in s["caches"]])
    elif c["op"] == "commit":
        dt = _DTYPES[c["dtype"]]
        users, nodes, kvh, dim, block = c["users"], c["nodes"], c["kv_heads"], c["dim"], c["block"]
        pages = (c["ctx"] + nodes + block - 1) // block
        lens = _lengths(gen, users, c["ctx"])
        s["lens"] = lens
        s["table"] = _page_table(gen, users, pages, torch.full_like(lens, pages), 3)
        s["caches"] = [torch.empty(users * pages + 3, kvh, block, dim, device="cuda", dtype=dt).normal_(generator=gen)
                       for _ in range(c["caches"])]
        s["drafts"] = [torch.empty(users, nodes, kvh, dim, device="cuda", dtype=dt).normal_(generator=gen) for _ in range(c["caches"])]
        # the accepted path: ascending nodes of the tree, from none to all of them
        s["path_len"] = torch.randint(0, nodes + 1, (users,), generator=gen, device="cuda", dtype=torch.int32)
        keys = torch.rand(users, nodes, generator=gen, device="cuda")
        chosen = keys.argsort(dim=1).argsort(dim=1) < s["path_len"][:, None]
        s["path"] = torch.where(chosen, 0, 1).argsort(dim=1, stable=True).to(torch.int32).contiguous()
        s["ptrs"] = (ctypes.c_void_p * c["caches"])(*[t.data_ptr() for t in s["caches"]])
        s["draft_ptrs"] = (ctypes.c_void_p * c["caches"])(*[t.data_ptr() for t in s["drafts"]])
    else:
        rows, vocab, mode = c["rows"], c["vocab"], c["mode"]
        logits = torch.randn(rows, vocab, generator=gen, device="cuda") * 2.5
        likely = torch.randint(0, vocab, (rows, 24), generator=gen, device="cuda")               # what a trained model puts on top
        logits.scatter_add_(1, likely, torch.rand(rows, 24, generator=gen, device="cuda") * 12.0)
        banned = torch.randint(1, vocab, (rows, max(1, vocab // 100)), generator=gen, device="cuda")
        logits.scatter_(1, banned, float("-inf"))
        s["logits"] = logits.to(_DTYPES[c["dtype"]])
        del logits

        def pick(values):
            v = torch.tensor(values, device="cuda")
            return v[torch.randint(0, len(values), (rows,), generator=gen, device="cuda")].contiguous()
        s["temperature"] = pick([0.0] if mode == "greedy" else ([0.7, 1.0, 1.3] if mode != "mixed" else [0.0, 0.5, 0.8, 1.0, 1.0, 1.5]))
        s["top_k"] = pick([0] if mode in ("plain", "top_p", "greedy") else [0, 1, 20, 50, 1000, 40000]).to(torch.int32)
        s["top_p"] = pick([1.0] if mode in ("plain", "top_k", "greedy") else [0.5, 0.9, 0.95, 0.99, 1.0])
        s["min_p"] = pick([0.0] if mode != "mixed" else [0.0, 0.0, 0.02, 0.1])
        s["uniform"] = torch.rand(rows, generator=gen, device="cuda")
        s["out"] = torch.zeros(rows, device="cuda", dtype=torch.int32)
        s["prob"] = torch.zeros(rows, device="cuda", dtype=torch.float32)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        _prepare_own(s)
    return s


# ---------------------------------------------------------------------------------------------- plain forms
def _softmax_rows(x):
    """softmax over the last dimension in x's type; a row of -inf only becomes zeros."""
    top = x.amax(dim=-1, keepdim=True)
    e = torch.exp(x - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = e.sum(dim=-1, keepdim=True)
    return e / torch.where(total > 0, total, torch.ones_like(total))


def _pages(cache, row):
    """One user's cached sequence [kv heads, positions, dim] in 32 bits."""
    blocks = cache[torch.clamp(row.long(), min=0)].float()          # [pages, kv heads, block, dim]
    return blocks.permute(1, 0, 2, 3).reshape(cache.shape[1], -1, cache.shape[3])


def _plain_window_decode(s):
    c, q = s["case"], s["q"][0].float()
    users, heads, dim = q.shape
    scale = 1.0 / math.sqrt(dim)
    outs = []
    for b in range(users):
        k, v = _pages(s["k"], s["table"][b]), _pages(s["v"], s["table"][b])
        j = torch.arange(k.shape[1], device="cuda")
        seen = (j <= s["pos"][b]) & ((j < c["sinks"]) | (j > s["pos"][b] - c["window"]))
        x = torch.matmul(q[b].view(k.shape[0], -1, dim), k.transpose(1, 2)) * scale
        x = x.masked_fill(~seen, float("-inf"))
        outs.append(torch.matmul(_softmax_rows(x), v).reshape(heads, dim))
    return torch.stack(outs)[None].to(s["q"].dtype)


def _ancestors(parents):
    """[users, nodes, nodes] truth values: column u is node t itself or one of its ancestors; and each node's depth."""
    users, nodes = parents.shape
    seen = torch.eye(nodes, device=parents.device, dtype=torch.bool).expand(users, nodes, nodes).clone()
    user = torch.arange(users, device=parents.device)
    at = torch.arange(nodes, device=parents.device).expand(users, nodes)
    for _ in range(nodes - 1):
        up = torch.gather(parents.long(), 1, torch.clamp(at, min=0))
        at = torch.where(at >= 0, up, at)
        hit = torch.zeros_like(seen)
        hit[user[:, None], torch.arange(nodes, device=parents.device)[None, :], torch.clamp(at, min=0)] = True
        seen |= hit & (at >= 0)[:, :, None]
    return seen, seen.sum(dim=2) - 1


def _plain_tree(s):
    c, q = s["case"], s["q"]
    users, nodes, heads, dim = q.shape
    scale = 1.0 / math.sqrt(dim)
    related, depth = _ancestors(s["parents"])
    outs = []
    for b in range(users):
        k = torch.cat([_pages(s["k"], s["table"][b]), s["kd"][b].float().transpose(0, 1)], dim=1)
        v = torch.cat([_pages(s["v"], s["table"][b]), s["vd"][b].float().transpose(0, 1)], dim=1)
        cached = k.shape[1] - nodes
        j = torch.arange(cached, device="cuda")
        seen = (j < s["lens"][b]).expand(nodes, cached)
        where = s["lens"][b] + depth[b]                               # position of each node
        fresh = related[b]
        if c["window"]:
            seen = seen & ((j[None, :] < c["sinks"]) | (j[None, :] > (where - c["window"])[:, None]))
            fresh = fresh & ((where[None, :] < c["sinks"]) | (where[None, :] > (where - c["window"])[:, None]))
        seen = torch.cat([seen, fresh], dim=1)                        # [nodes, keys]
        kvh = k.shape[0]
        qb = q[b].float().view(nodes, kvh, heads // kvh, dim).permute(1, 2, 0, 3)
        x = torch.matmul(qb, k.transpose(1, 2)[:, None]) * scale
        x = x.masked_fill(~seen, float("-inf"))
        o = torch.matmul(_softmax_rows(x), v[:, None])                # [kv heads, group, nodes, dim]
        outs.append(o.permute(2, 0, 1, 3).reshape(nodes, heads, dim))
    return torch.stack(outs).to(q.dtype)


def _plain_window(s):
    c, q = s["case"], s["q"]
    users, heads, queries, dim = q.shape
    kvh, keys = s["k"].shape[1], s["k"].shape[2]
    scale = 1.0 / math.sqrt(dim)
    out = torch.empty_like(q)
    j = torch.arange(keys, device="cuda")
    for b in range(users):
        live = j < (s["lens"][b] if s["lens"] is not None else keys)
        for h in range(kvh):
            k, v = s["k"][b, h].float(), s["v"][b, h].float()
            g = slice(h * (heads // kvh), (h + 1) * (heads // kvh))
            for i in range(0, queries, 4096):
                at = torch.arange(i, min(i + 4096, queries), device="cuda")[:, None] + c["offset"]
                seen = (j <= at) & ((j < c["sinks"]) | (j > at - c["window"])) & live
                x = torch.matmul(q[b, g, i:i + 4096].float(), k.t()) * scale
                x = x.masked_fill(~seen, float("-inf"))
                out[b, g, i:i + 4096] = torch.matmul(_softmax_rows(x), v).to(q.dtype)
    return out


def _plain_copy(s):
    src, dst = s["pairs"][:, 0].long(), s["pairs"][:, 1].long()
    for t in s["caches"]:
        t[dst] = t[src]
    return list(s["caches"])


def _plain_commit(s):
    c = s["case"]
    users, nodes = s["path"].shape
    i = torch.arange(nodes, device="cuda").expand(users, nodes)
    user = torch.arange(users, device="cuda")[:, None].expand(users, nodes)
    keep = i < s["path_len"][:, None]
    at = s["lens"][:, None] + i
    page = torch.clamp(at // c["block"], max=s["table"].shape[1] - 1).long()
    block = torch.gather(s["table"].long(), 1, page)[keep]
    slot = (at % c["block"])[keep].long()
    user, node = user[keep], s["path"].long()[keep]
    for t, d in zip(s["caches"], s["drafts"]):
        t[block, :, slot] = d[user, node]
    return list(s["caches"])


def _plain_sample(s):
    x = s["logits"].double()
    rows, vocab = x.shape
    value, index = torch.sort(x, dim=1, descending=True, stable=True)
    greedy = s["temperature"] <= 0
    heat = torch.where(greedy, torch.ones_like(s["temperature"]), s["temperature"]).double()
    w = torch.exp((value - value[:, :1]) / heat[:, None])
    rank = torch.arange(vocab, device="cuda")[None, :]
    k = torch.where((s["top_k"] > 0) & (s["top_k"] < vocab), s["top_k"], vocab)
    w = torch.where(rank < k[:, None], w, torch.zeros_like(w))
    p = s["top_p"].double()
    before = torch.cumsum(w, dim=1) - w
    cut = (p > 0) & (p < 1)
    w = torch.where(~cut[:, None] | (before < p[:, None] * w.sum(dim=1, keepdim=True)), w, torch.zeros_like(w))
    low = s["min_p"].double()
    w = torch.where((low <= 0)[:, None] | (w >= low[:, None]), w, torch.zeros_like(w))
    w = torch.where(greedy[:, None] & (rank > 0), torch.zeros_like(w), w)
    by_token = torch.zeros_like(w).scatter_(1, index, w)              # the draw runs over the tokens in order
    run = torch.cumsum(by_token, dim=1)
    total = run[:, -1:]
    token = (run <= s["uniform"].double()[:, None] * total).sum(dim=1, keepdim=True)
    token = torch.clamp(token, max=vocab - 1)
    return [token[:, 0].to(torch.int32), (torch.gather(by_token, 1, token) / total)[:, 0].float()]


# ---------------------------------------------------------------------------------------------- the framework's kernels
def _library():
    from __graft_entry__ import load_package
    load_package()
    from ttmlir_b200 import runtime_api
    return runtime_api.lib


_VP, _I, _L, _F, _Z = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float, ctypes.c_size_t
_SIGNATURES = {
    "ttb_sdpa_window": [_VP] * 5 + [_I] + [_L] * 6 + [_VP] * 4 + [_L] * 3 + [_F, _VP],
    "ttb_sdpa_window_decode": [_VP] * 6 + [_I] * 8 + [_L] * 2 + [_F, _VP, _Z, _VP],
    "ttb_sdpa_tree": [_VP] * 10 + [_I] * 10 + [_L] * 2 + [_F, _VP, _Z, _VP],
    "ttb_paged_copy_blocks": [_VP, _I, _VP, _I, _I, _L, _L, _L, _L, _VP],
    "ttb_paged_commit_draft": [_VP, _VP, _I, _VP, _VP, _VP, _VP, _I] + [_L] * 7 + [_VP],
    "ttb_sample_logits": [_VP] * 8 + [_I] + [_L] * 3 + [_VP, _Z, _VP],
}
_SIZES = {
    "ttb_sdpa_window_decode_workspace_bytes": [_I] * 4 + [_L] * 3,
    "ttb_sdpa_tree_workspace_bytes": [_I] * 5 + [_L],
    "ttb_sample_logits_workspace_bytes": [_L] * 2,
}


def _prepare_own(s):
    """What a serving loop sets up once: the library, its argument types and a workspace."""
    lib, c = _library(), s["case"]
    for table, result in ((_SIGNATURES, _I), (_SIZES, _Z)):
        for name, args in table.items():
            fn = getattr(lib, name)
            fn.argtypes, fn.restype = args, result
    s["lib"] = lib
    size = 0
    if c["op"] == "window_decode":
        pages = s["table"].shape[1]
        size = lib.ttb_sdpa_window_decode_workspace_bytes(c["users"], c["heads"], c["kv_heads"], c["dim"], pages * c["block"],
                                                          c["window"], c["sinks"])
    elif c["op"] == "tree":
        pages = s["table"].shape[1]
        size = lib.ttb_sdpa_tree_workspace_bytes(c["users"], c["nodes"], c["heads"], c["kv_heads"], c["dim"], pages * c["block"])
    elif c["op"] == "sample":
        size = lib.ttb_sample_logits_workspace_bytes(c["rows"], c["vocab"])
    s["work"] = torch.empty(max(int(size), 16), device="cuda", dtype=torch.uint8)


def _run_own(s):
    lib, c = s["lib"], s["case"]
    stream = torch.cuda.current_stream().cuda_stream
    work, size = s["work"].data_ptr(), s["work"].numel()
    scale = 1.0 / math.sqrt(c["dim"]) if "dim" in c else 1.0
    if c["op"] == "window_decode":
        rc = lib.ttb_sdpa_window_decode(s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), s["table"].data_ptr(), s["pos"].data_ptr(),
                                        s["out"].data_ptr(), _TAGS[s["q"].dtype], c["users"], c["heads"], c["kv_heads"], s["k"].shape[0],
                                        c["block"], s["table"].shape[1], c["dim"], c["window"], c["sinks"], scale, work, size, stream)
        res = s["out"]
    elif c["op"] == "tree":
        rc = lib.ttb_sdpa_tree(s["q"].data_ptr(), s["kd"].data_ptr(), s["vd"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(),
                               s["table"].data_ptr(), s["lens"].data_ptr(), s["parents"].data_ptr(), None, s["out"].data_ptr(),
                               _TAGS[s["q"].dtype], c["users"], c["nodes"], c["heads"], c["kv_heads"], s["k"].shape[0], c["block"],
                               s["table"].shape[1], c["dim"], c["users"], c["window"], c["sinks"], scale, work, size, stream)
        res = s["out"]
    elif c["op"] == "window":
        rc = lib.ttb_sdpa_window(s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), s["lens"].data_ptr() if s["lens"] is not None else None,
                                 s["out"].data_ptr(), _TAGS[s["q"].dtype], c["users"], c["heads"], c["kv_heads"], c["queries"], c["keys"],
                                 c["dim"], None, None, None, None, c["offset"], c["window"], c["sinks"], scale, stream)
        res = s["out"]
    elif c["op"] == "copy":
        rc = lib.ttb_paged_copy_blocks(s["ptrs"], c["caches"], s["pairs"].data_ptr(), c["pairs"], _TAGS[s["caches"][0].dtype], c["blocks"],
                                       c["kv_heads"], c["block"], c["dim"], stream)
        res = list(s["caches"])
    elif c["op"] == "commit":
        rc = lib.ttb_paged_commit_draft(s["ptrs"], s["draft_ptrs"], c["caches"], s["table"].data_ptr(), s["lens"].data_ptr(),
                                        s["path"].data_ptr(), s["path_len"].data_ptr(), _TAGS[s["caches"][0].dtype], c["users"], c["nodes"],
                                        c["kv_heads"], s["caches"][0].shape[0], c["block"], s["table"].shape[1], c["dim"], stream)
        res = list(s["caches"])
    else:
        rc = lib.ttb_sample_logits(s["logits"].data_ptr(), s["uniform"].data_ptr(), s["temperature"].data_ptr(), s["top_k"].data_ptr(),
                                   s["top_p"].data_ptr(), s["min_p"].data_ptr(), s["out"].data_ptr(), s["prob"].data_ptr(),
                                   _TAGS[s["logits"].dtype], c["rows"], c["vocab"], c["vocab"], work, size, stream)
        res = [s["out"], s["prob"]]
    if rc:
        raise RuntimeError(lib.ttb_last_error().decode())
    return res


_PLAIN = {"tree": _plain_tree, "window_decode": _plain_window_decode, "window": _plain_window, "copy": _plain_copy,
          "commit": _plain_commit, "sample": _plain_sample}


def run(state):
    return _run_own(state) if own else _PLAIN[state["case"]["op"]](state)


# ---------------------------------------------------------------------------------------------- work and definition
def _visible(length, window, sinks):
    """Keys that the token at position length - 1 sees."""
    return min(length, window) + min(sinks, max(0, length - window))


def work(case):
    c = case
    size = 4 if c["dtype"] == "f32" else 2
    if c["op"] == "window_decode":
        seen = 0.75 * c["users"] * _visible(c["ctx"], c["window"], c["sinks"]) if c["ctx"] <= c["window"] else \
            c["users"] * _visible(c["ctx"], c["window"], c["sinks"])
        return {"bytes": seen * c["kv_heads"] * c["dim"] * 2 * size + 2 * c["users"] * c["heads"] * c["dim"] * size,
                "flops": 4.0 * seen * c["heads"] * c["dim"]}
    if c["op"] == "tree":
        length = (0.75 * (c["users"] - 1) + 1) * c["ctx"]            # cached tokens of all users, on average
        if c["window"]:
            length = min(length, c["users"] * (c["window"] + c["sinks"]))
        rows = c["users"] * c["nodes"]
        return {"bytes": (length + rows) * c["kv_heads"] * c["dim"] * 2 * size + 2 * rows * c["heads"] * c["dim"] * size,
                "flops": 4.0 * c["nodes"] * length * c["heads"] * c["dim"]}
    if c["op"] == "window":
        seen = sum(_visible(i + 1, c["window"], c["sinks"]) for i in range(c["offset"], c["offset"] + c["queries"])) * c["users"]
        return {"bytes": 2.0 * c["users"] * c["dim"] * size * (c["heads"] * c["queries"] + c["kv_heads"] * c["keys"]),
                "flops": 4.0 * seen * c["heads"] * c["dim"]}
    if c["op"] == "copy":
        return {"bytes": 2.0 * c["caches"] * c["pairs"] * c["kv_heads"] * c["block"] * c["dim"] * size, "flops": 0.0}
    if c["op"] == "commit":
        return {"bytes": 2.0 * c["caches"] * c["users"] * 0.5 * c["nodes"] * c["kv_heads"] * c["dim"] * size, "flops": 0.0}
    return {"bytes": float(c["rows"]) * c["vocab"] * size, "flops": 4.0 * c["rows"] * c["vocab"]}


def exact(case, seed):
    """`run`'s outputs from the definitions: one query row at a time as far as that is affordable, 64 bits throughout."""
    c = case
    s = _inputs(case, seed)
    if c["op"] == "copy":
        before = [t.clone() for t in s["caches"]]
        for src, dst in s["pairs"].tolist():
            for old, t in zip(before, s["caches"]):
                t[dst].copy_(old[src])
        return list(s["caches"])
    if c["op"] == "commit":
        lens, path, count, table = s["lens"].tolist(), s["path"].tolist(), s["path_len"].tolist(), s["table"].tolist()
        if c["caches"] * sum(count) > 60000:
            return None
        for b in range(c["users"]):
            for i in range(count[b]):
                page, slot = divmod(lens[b] + i, c["block"])
                for t, d in zip(s["caches"], s["drafts"]):
                    t[table[b][page], :, slot].copy_(d[b, path[b][i]])
        return list(s["caches"])
    if c["op"] == "sample":
        tokens, probs = [], []
        for r in range(c["rows"]):
            x = s["logits"][r].double()
            vocab = x.numel()
            order = sorted_desc(x)
            heat, k = float(s["temperature"][r]), int(s["top_k"][r])
            p, low, u = float(s["top_p"][r]), float(s["min_p"][r]), float(s["uniform"][r])
            if heat <= 0:
                tokens.append(int(order[0]))
                probs.append(1.0)
                continue
            kept = order[:k] if 0 < k < vocab else order
            mass = torch.exp((x[kept] - x[order[0]]) / heat)
            if 0 < p < 1:
                ends = torch.cumsum(mass, 0)
                count = int((ends < p * ends[-1]).sum()) + 1
                kept, mass = kept[:count], mass[:count]
            if low > 0:
                kept, mass = kept[mass >= low], mass[mass >= low]
            kept, back = torch.sort(kept)
            ends = torch.cumsum(mass[back], 0)
            at = min(int((ends <= u * ends[-1]).sum()), kept.numel() - 1)
            tokens.append(int(kept[at]))
            probs.append(float(mass[back][at] / ends[-1]))
        return [torch.tensor(tokens, dtype=torch.int32, device="cuda"), torch.tensor(probs, dtype=torch.float64, device="cuda")]
    group, scale = c["heads"] // c["kv_heads"], 1.0 / math.sqrt(c["dim"])

    def attend(q, k, v, seen):
        """q [heads, dim] against k, v [kv heads, keys, dim]; `seen` are the indices of the visible keys."""
        if seen.numel() == 0:
            return torch.zeros_like(q)
        ks, vs = k[:, seen], v[:, seen]
        x = torch.einsum("hgd,hkd->hgk", q.view(c["kv_heads"], group, -1), ks) * scale
        e = torch.exp(x - x.max(dim=2, keepdim=True).values)
        return (torch.einsum("hgk,hkd->hgd", e, vs) / e.sum(dim=2, keepdim=True)).reshape(q.shape)

    def inside(j, at):
        return (j < c["sinks"]) | (j > at - c["window"])
    if c["op"] == "window":
        if c["users"] * c["queries"] > 20000 or c["heads"] * c["queries"] * min(c["keys"], c["window"] + c["sinks"]) * c["dim"] > 2 ** 38:
            return None
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        for b in range(c["users"]):
            n = int(s["lens"][b]) if s["lens"] is not None else c["keys"]
            k, v, q = s["k"][b].double(), s["v"][b].double(), s["q"][b].double()
            j = torch.arange(n, device="cuda")
            for i in range(c["queries"]):
                at = i + c["offset"]
                first = max(0, at - c["window"] + 1)
                keys = torch.cat([j[:min(c["sinks"], first, at + 1)], j[first:at + 1]])
                out[b, :, i] = attend(q[:, i], k, v, keys)
        return out
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    parents = s["parents"].tolist() if c["op"] == "tree" else None
    for b in range(c["users"]):
        n = int(s["lens"][b]) if c["op"] == "tree" else int(s["pos"][b]) + 1
        rows = torch.arange(n, device="cuda")
        block = s["table"][b].long()[rows // c["block"]]
        k = s["k"][block, :, rows % c["block"]].double().transpose(0, 1)
        v = s["v"][block, :, rows % c["block"]].double().transpose(0, 1)
        if c["op"] == "window_decode":
            out[0, b] = attend(s["q"][0, b].double(), k, v, rows[inside(rows, n - 1)])
            continue
        k = torch.cat([k, s["kd"][b].double().transpose(0, 1)], dim=1)
        v = torch.cat([v, s["vd"][b].double().transpose(0, 1)], dim=1)
        depth = []
        for t in range(c["nodes"]):
            depth.append(0 if parents[b][t] < 0 else depth[parents[b][t]] + 1)
        for t in range(c["nodes"]):
            line, up = [], t
            while up >= 0:
                line.append(up)
                up = parents[b][up]
            at = n + depth[t]
            old = rows
            if c["window"]:
                old = rows[inside(rows, at)]
                line = [u for u in line if inside(n + depth[u], at)]
            out[b, t] = attend(s["q"][b, t].double(), k, v, torch.cat([old, torch.tensor(line, device="cuda", dtype=torch.long) + n]))
    return out


def sorted_desc(x):
    """Indices of x from the largest value down; of equal values the lower index first."""
    return torch.sort(x, descending=True, stable=True).indices
