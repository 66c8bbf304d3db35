"""Plain 64-bit forms of the serving operators, and calls of the kernel library on CPU tensors, for the tests."""

import ctypes
import math

import torch

from helpers import KernelHarness

TAG = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2, torch.int32: 12, torch.int8: 17, torch.uint8: 11}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def attend(q, k, v, seen, scale, dtype):
    """q [H, R, D] against k, v [Hkv, N, D] with seen [R, N]: the result in 64 bits and how far a kernel may be off.

    The kernel accumulates scores in f32: a score is off by at most (D + 4) 2^-24 times the sum of |q k| scale, and a
    weight by twice that (once in the numerator, once in the sum), plus N 2^-24 of the sums and 2^-21 for exp2.  With
    16-bit operands the weights are rounded once more (half a step), and the result is rounded once."""
    H, R, D = q.shape
    g = H // k.shape[0]
    q, k, v = q.double(), k.double(), v.double()
    out = torch.zeros(H, R, D, dtype=torch.float64)
    tol = torch.zeros(H, R, D, dtype=torch.float64)
    used = seen.any(dim=0)
    k = torch.where(used[None, :, None], k, 0.0)                     # what no row sees may hold anything
    v = torch.where(used[None, :, None], v, 0.0)
    for h in range(H):
        s = q[h] @ k[h // g].T * scale
        size = (q[h].abs() @ k[h // g].abs().T * abs(scale)).max() if s.numel() else torch.tensor(0.0)
        s = s.masked_fill(~seen, float("-inf"))
        top = s.amax(dim=1, keepdim=True) if s.shape[1] else torch.full((R, 1), float("-inf"), dtype=torch.float64)
        e = torch.exp(s - torch.where(torch.isinf(top), 0.0, top))
        total = e.sum(dim=1, keepdim=True)
        w = e / torch.where(total > 0, total, 1.0)
        out[h] = w @ v[h // g]
        spread = w @ v[h // g].abs()
        weight = 2 * (D + 4) * 2.0 ** -24 * size + (seen.shape[1] + 8) * 2.0 ** -24 + 2.0 ** -21
        if dtype != torch.float32:
            weight = weight + half_step(dtype)
        tol[h] = half_step(dtype) * out[h].abs() * (1 + 2 ** -6) + weight * spread * (1 + 2 ** -6) + 1e-7
    return out, tol


def check(got, want, tol, what=""):
    if want.numel() == 0:
        return
    assert torch.isfinite(got.double()).all(), f"{what}: not finite"
    over = ((got.double() - want).abs() - tol).max().item()
    assert over <= 0, f"{what}: beyond the tolerance by {over}, worst error {(got.double() - want).abs().max().item()}"


def window_seen(positions, n, window, sinks):
    """[rows, n]: which of n keys the tokens at `positions` see (window 0: all up to themselves)."""
    j = torch.arange(n)[None, :]
    p = positions[:, None]
    near = j > p - window if window else torch.ones_like(j <= p)
    return (j <= p) & (near | (j < sinks))


def tree_lines(parents):
    """related[t, u]: u is t or an ancestor of t."""
    n = len(parents)
    related = torch.zeros(n, n, dtype=torch.bool)
    for t in range(n):
        u = t
        while u >= 0:
            related[t, u] = True
            u = parents[u]
    return related


class Kernels(KernelHarness):
    """The entry points on CPU tensors: uploads, calls, downloads.  `raw` entry points return the status."""

    def __init__(self, rt):
        super().__init__(rt)
        for n in ("ttb_sdpa_window_decode_workspace_bytes", "ttb_sdpa_tree_workspace_bytes", "ttb_sample_logits_workspace_bytes"):
            getattr(self.lib, n).restype = ctypes.c_size_t

    def args(self, *xs):
        res = []
        for x in xs:
            if isinstance(x, bool) or x is None:
                res.append(ctypes.c_void_p(None) if x is None else ctypes.c_int(int(x)))
            elif isinstance(x, int):
                res.append(ctypes.c_int64(x))
            elif isinstance(x, float):
                res.append(ctypes.c_float(x))
            else:
                res.append(x)
        return res

    def call(self, name, *xs):
        self._check(getattr(self.lib, name)(*self.args(*xs)))

    def bad(self):
        flag = ctypes.c_int()
        self._check(self.lib.ttb_index_status(ctypes.byref(flag)))
        return flag.value

    def up(self, t):
        return None if t is None else self.upload(t)

    def window(self, q, k, v, offset, window, sinks, lens=None, scale=None, out=None, permuted=False):
        B, H, S, D = q.shape
        scale = 1 / math.sqrt(D) if scale is None else scale
        strides = [None] * 4
        if permuted:   # [batch, seq, heads, dim] in memory
            q, k, v = (t.permute(0, 2, 1, 3).contiguous() for t in (q, k, v))
            I3 = ctypes.c_int64 * 3
            of = lambda t: I3(t.stride(0), t.stride(2), t.stride(1))
            strides = [of(q), of(k), of(v), of(q)]
            keys, kvh = k.shape[1], k.shape[2]
        else:
            keys, kvh = k.shape[2], k.shape[1]
        po = self.upload(torch.zeros_like(q) if out is None else out)
        self.call("ttb_sdpa_window", self.up(q), self.up(k), self.up(v), self.up(lens), po, TAG[q.dtype], B, H, kvh, S, keys, D,
                  *strides, offset, window, sinks, float(scale), self.stream)
        got = self.download(po, q.shape, q.dtype)
        return got.permute(0, 2, 1, 3) if permuted else got

    def decode(self, q, k, v, table, pos, window, sinks, scale=None):
        _, B, H, D = q.shape
        scale = 1 / math.sqrt(D) if scale is None else scale
        blocks, kvh, block = k.shape[:3]
        pages = table.shape[1] if table is not None else 1
        size = self.lib.ttb_sdpa_window_decode_workspace_bytes(*self.args(B, H, kvh, D, pages * block, window, sinks))
        po, work = self.empty(q.shape, q.dtype), self.empty((max(size, 16),), torch.uint8)
        self.call("ttb_sdpa_window_decode", self.up(q), self.up(k), self.up(v), self.up(table), self.up(pos), po, TAG[q.dtype], B, H, kvh,
                  blocks, block, pages, D, window, sinks, float(scale), work, ctypes.c_size_t(size), self.stream)
        return self.download(po, q.shape, q.dtype)

    def tree(self, q, kd, vd, k, v, table, lens, parents, window=0, sinks=0, draft_lens=None, scale=None, out=None):
        B, T, H, D = q.shape
        scale = 1 / math.sqrt(D) if scale is None else scale
        blocks, kvh, block = k.shape[:3]
        pages = table.shape[1] if table is not None else 1
        size = self.lib.ttb_sdpa_tree_workspace_bytes(*self.args(B, T, H, kvh, D, pages * block))
        po = self.upload(torch.zeros_like(q) if out is None else out)
        work = self.empty((max(size, 16),), torch.uint8)
        self.call("ttb_sdpa_tree", self.up(q), self.up(kd), self.up(vd), self.up(k), self.up(v), self.up(table), self.up(lens),
                  self.up(parents), self.up(draft_lens), po, TAG[q.dtype], B, T, H, kvh, blocks, block, pages, D, parents.shape[0],
                  window, sinks, float(scale), work, ctypes.c_size_t(size), self.stream)
        return self.download(po, q.shape, q.dtype)

    def sample(self, logits, uniform, temperature=None, top_k=None, top_p=None, min_p=None, stride=None):
        rows, vocab = logits.shape[0], logits.shape[1]
        pl = self.upload(logits)
        if stride is not None:
            vocab, stride = stride, vocab
        size = self.lib.ttb_sample_logits_workspace_bytes(*self.args(rows, vocab))
        work = self.empty((max(size, 16),), torch.uint8)
        out, prob = self.upload(torch.full((rows,), -7, dtype=torch.int32)), self.upload(torch.full((rows,), -7.0))
        self.call("ttb_sample_logits", pl, self.up(uniform), self.up(temperature), self.up(top_k), self.up(top_p), self.up(min_p), out, prob,
                  TAG[logits.dtype], rows, vocab, stride or vocab, work, ctypes.c_size_t(size), self.stream)
        return self.download(out, (rows,), torch.int32), self.download(prob, (rows,), torch.float32)

    def copy_blocks(self, caches, pairs):
        ps = [self.upload(c) for c in caches]
        arr = (ctypes.c_void_p * len(ps))(*[p.value for p in ps])
        b, h, s, d = caches[0].shape
        self.call("ttb_paged_copy_blocks", arr, len(ps), self.up(pairs), pairs.shape[0], TAG[caches[0].dtype], b, h, s, d, self.stream)
        return [self.download(p, c.shape, c.dtype) for p, c in zip(ps, caches)]

    def commit(self, caches, drafts, table, lens, path, path_lens):
        ps, ds = [self.upload(c) for c in caches], [self.upload(d) for d in drafts]
        arr, darr = ((ctypes.c_void_p * len(x))(*[p.value for p in x]) for x in (ps, ds))
        b, h, s, d = caches[0].shape
        users, nodes = path.shape
        self.call("ttb_paged_commit_draft", arr, darr, len(ps), self.up(table), self.up(lens), self.up(path), self.up(path_lens),
                  TAG[caches[0].dtype], users, nodes, h, b, s, table.shape[1], d, self.stream)
        return [self.download(p, c.shape, c.dtype) for p, c in zip(ps, caches)]


def sample_row(x, u, heat, k, p, low):
    """One row of ttb_sample_logits in 64 bits: (token, probability, distance of u to the nearest border of a token's share,
    distance of the cuts to the nearest border), or None where nothing can be taken."""
    x = x.double()
    x = torch.where(torch.isnan(x), float("-inf"), x)
    order = torch.sort(x, descending=True, stable=True).indices
    if x[order[0]] == float("-inf"):
        return -1, 0.0
    if not heat > 0:
        return int(order[0]), 1.0
    top = x[order[0]]
    w = torch.where(x == top, torch.ones_like(x), torch.exp((x - top) / heat))
    w = torch.where(x == float("-inf"), 0.0, torch.nan_to_num(w))
    kept = order[:k] if 0 < k < x.numel() else order
    if 0 < p < 1:
        mass = w[kept]
        before = torch.cumsum(mass, 0) - mass
        kept = kept[before < p * mass.sum()]
    if 0 < low <= 1:
        kept = kept[w[kept] >= low]
    kept = torch.sort(kept).values
    run = torch.cumsum(w[kept], 0)
    at = min(int((run <= u * run[-1]).sum()), kept.numel() - 1)
    return int(kept[at]), float(w[kept][at] / run[-1])
