"""A batch over a paged KV cache and rows of logits, in 64 bits with numpy: what
the paged append, attention and log probability tests check against."""
from __future__ import annotations

import ctypes

import numpy as np

import llmpager_amd as lp

GROUP = 32


def round7(x):
    """x > 0 to 7 significant bits, ties to even."""
    m, e = np.frexp(x)
    return np.ldexp(np.rint(m * 128.0) / 128.0, e)


def q4(x):
    """(codes 0 .. 15, scales) of rows x [..., D] as a q4 page takes them."""
    x = np.where(np.isnan(x), 0.0, x)
    g = x.reshape(*x.shape[:-1], -1, GROUP)
    with np.errstate(over="ignore"):
        s = np.clip(round7(np.abs(g).max(-1) / 7.0), 2.0 ** -17, 896.0)
    q = np.clip(np.rint(np.clip(g, -1e5, 1e5) / s[..., None]), -7, 7) + 8
    return q.reshape(x.shape).astype(np.uint8), s


class Batch:
    """Sequences of `new` tokens behind `past` ones in shuffled pages: host
    pools, table and lengths, and their device copies."""

    def __init__(self, cuda, new, past, heads, kv, dim, page, fmt, seed=0, pad=0, spare=3, cols=None):
        self.cuda, self.heads, self.kv, self.dim, self.page, self.fmt = cuda, heads, kv, dim, page, fmt
        self.new, self.past = list(new), list(past)
        self.lens = [n + p for n, p in zip(new, past)]
        self.batch, self.live = len(new), sum(new)
        self.tokens = self.live + pad
        rng = self.rng = np.random.default_rng(seed)
        need = [-(-n // page) for n in self.lens]
        self.pages = sum(need) + spare
        self.cols = cols or max(need + [1]) + 1
        order = rng.permutation(self.pages).astype(np.int32)
        self.table = np.full((self.batch, self.cols), -1, np.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + min(n, self.cols)]
            at += n
        self.starts = np.concatenate(([0], np.cumsum(new))).astype(np.int32)
        self.page_bytes = lp.kv_page_bytes(page, dim, fmt)
        self.pools = [self._pool(), self._pool()]
        self.freq = (1e6 ** (-np.arange(0, dim, 2) / dim)).astype(np.float32)
        self.ptrs = []

    def _pool(self):
        x = self.rng.standard_normal((self.pages, self.kv, self.page, self.dim))
        if self.fmt == lp.KV_F16:
            return np.ascontiguousarray(x.astype(np.float16).reshape(self.pages, self.kv, -1).view(np.uint8))
        codes, s = q4(x)
        nib = codes[..., 0::2] | codes[..., 1::2] << 4
        return np.concatenate((np.ascontiguousarray(s.astype(np.float16)).reshape(self.pages, self.kv, -1).view(np.uint8),
                               nib.reshape(self.pages, self.kv, -1)), 2)

    def values(self, pool):
        """The pool's values [pages, kv, page, D]."""
        if self.fmt == lp.KV_F16:
            return pool.view(np.float16).reshape(self.pages, self.kv, self.page, self.dim).astype(np.float64)
        n = self.page * (self.dim // GROUP) * 2
        s = np.ascontiguousarray(pool[..., :n]).view(np.float16).astype(np.float64)
        b = pool[..., n:].reshape(self.pages, self.kv, self.page, self.dim // 2)
        q = np.stack((b & 15, b >> 4), -1).reshape(self.pages, self.kv, self.page, -1, GROUP) - 8.0
        return (q * s.reshape(*q.shape[:-1], 1)).reshape(self.pages, self.kv, self.page, self.dim)

    def put(self, row, k=None, v=None, b=0):
        """Row `row` of sequence b as fp16 values [kv, D] (fp16 pools only)."""
        p, r = self.table[b, row // self.page], row % self.page
        for pool, x in zip(self.pools, (k, v)):
            if x is not None:
                pool.view(np.float16).reshape(self.pages, self.kv, self.page, self.dim)[p, :, r] = x

    def up(self, a):
        p = self.cuda.upload(np.ascontiguousarray(a))
        self.ptrs.append(p)
        return p

    def alloc(self, n):
        p = self.cuda.alloc_device(max(n, 256))
        self.ptrs.append(p)
        return p

    def device(self):
        self.dk, self.dv = self.up(self.pools[0]), self.up(self.pools[1])
        self.dtable = self.up(self.table)
        self.dstarts, self.dlens = self.up(self.starts), self.up(np.asarray(self.lens, np.int32))
        self.cache = lp.KvCache(k_pages=self.dk, v_pages=self.dv, table=self.dtable, pages=self.pages,
                                page_rows=self.page, max_pages=self.cols, kv_heads=self.kv, head_dim=self.dim,
                                format=self.fmt)
        return self

    def free(self):
        self.cuda.sync()
        for p in self.ptrs:
            self.cuda.free_device(p)
        self.ptrs = []

    # ---- what the entry points compute ----

    def places(self):
        """(token, sequence, position) of every live token."""
        return [(int(self.starts[b]) + i, b, self.past[b] + i) for b in range(self.batch) for i in range(self.new[b])]

    def turned(self, x, w, eps, pos, mscale=1.0):
        x = x.astype(np.float64)
        if w is not None:
            x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
        h = self.dim // 2
        a = pos * self.freq.astype(np.float64)
        c, s = np.cos(a) * mscale, np.sin(a) * mscale
        return np.concatenate((x[..., :h] * c - x[..., h:] * s, x[..., :h] * s + x[..., h:] * c), -1)

    def append(self, q, k, v, qw, kw, eps, mscale=1.0):
        """(q_out, values as held of k and v [tokens, kv, D], both pools after)."""
        qo = np.zeros((self.tokens, self.heads, self.dim))
        held = [np.zeros((self.tokens, self.kv, self.dim)) for _ in range(2)]
        pools = [p.copy() for p in self.pools]
        for t, b, pos in self.places():
            qo[t] = self.turned(q[t].reshape(self.heads, self.dim), qw, eps, pos, mscale)
            for n, x in enumerate((self.turned(k[t].reshape(self.kv, self.dim), kw, eps, pos, mscale),
                                   v[t].reshape(self.kv, self.dim).astype(np.float64))):
                col = pos // self.page
                page = self.table[b, col] if col < self.cols else -1
                r, ok = pos % self.page, 0 <= page < self.pages
                if self.fmt == lp.KV_F16:
                    with np.errstate(over="ignore"):
                        held[n][t] = x.astype(np.float16)
                    if ok:
                        pools[n].view(np.float16).reshape(self.pages, self.kv, self.page, self.dim)[page, :, r] = held[n][t]
                else:
                    codes, s = q4(x)
                    held[n][t] = ((codes - 8.0).reshape(self.kv, -1, GROUP) * s[..., None]).reshape(self.kv, -1)
                    if ok:
                        G = self.dim // GROUP
                        nb = self.page * G * 2
                        pools[n][page, :, 2 * G * r:2 * G * (r + 1)] = s.astype(np.float16).view(np.uint8).reshape(self.kv, -1)
                        pools[n][page, :, nb + r * self.dim // 2:nb + (r + 1) * self.dim // 2] = \
                            codes[:, 0::2] | codes[:, 1::2] << 4
        return qo, held[0], held[1], pools

    def attention(self, q, scale, max_seq=None):
        """out [tokens, heads, D] of q [tokens, heads, D]."""
        K, V = self.values(self.pools[0]), self.values(self.pools[1])
        out = np.zeros((self.tokens, self.heads, self.dim))
        G = self.heads // self.kv
        cap = min(max_seq or 1 << 30, self.cols * self.page)
        for b in range(self.batch):
            L = min(self.lens[b], cap)
            rows = np.arange(max(L, 0))
            page = self.table[b, rows // self.page]
            have = (page >= 0) & (page < self.pages)
            kk = K[np.where(have, page, 0), :, rows % self.page]
            vv = V[np.where(have, page, 0), :, rows % self.page]
            for i in range(self.new[b]):
                t, pos = int(self.starts[b]) + i, L - self.new[b] + i
                see = have & (rows <= pos)
                if not see.any():
                    continue
                x = q[t].astype(np.float64).reshape(self.kv, G, self.dim)
                with np.errstate(invalid="ignore", over="ignore"):
                    s = np.einsum("kgd,rkd->kgr", x, kk[see]) * scale
                    p = np.exp(s - s.max(-1, keepdims=True))
                    out[t] = (np.einsum("kgr,rkd->kgd", p, vv[see]) / p.sum(-1, keepdims=True)).reshape(self.heads, -1)
        return out


def logprobs(x, targets, top):
    """(logp, entropy, ids, their log probabilities) of rows x in 64 bits."""
    x = x.astype(np.float64)
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        d = x - np.where(np.isnan(x), -np.inf, x).max(1, keepdims=True)
        e = np.exp(d)
        lse = np.log(e.sum(1))
        ent = lse - np.where(e == 0, 0.0, e * np.where(e == 0, 0.0, d)).sum(1) / e.sum(1)
        p = d - lse[:, None]
    rows = np.arange(len(x))
    ok = (targets >= 0) & (targets < x.shape[1])
    logp = np.where(ok, p[rows, np.where(ok, targets, 0)], 0.0)
    ids = np.argsort(np.where(np.isnan(x), np.inf, -x), axis=1, kind="stable")[:, :top]
    tp = np.take_along_axis(p, ids, 1)
    gone = np.isnan(np.take_along_axis(x, ids, 1))
    return logp, ent, np.where(gone, -1, ids), np.where(gone, np.nan, tp)


class HipGraph:
    """What `launches(stream)` does, captured through the HIP runtime itself, as a
    program with graphs of its own does (not lp_graph_capture_*)."""

    _hip = None

    def __init__(self, stream, launches):
        if HipGraph._hip is None:  # the runtime that the library has loaded
            with open("/proc/self/maps") as f:
                HipGraph._hip = ctypes.CDLL(next(x.split()[-1] for x in f if "libamdhip64" in x))
        self.graph, self.exec = ctypes.c_void_p(), ctypes.c_void_p()
        self._call("hipStreamBeginCapture", ctypes.c_void_p(stream), 2)  # relaxed
        try:
            launches(stream)
        finally:
            self._call("hipStreamEndCapture", ctypes.c_void_p(stream), ctypes.byref(self.graph))
        self._call("hipGraphInstantiate", ctypes.byref(self.exec), self.graph, None, None, ctypes.c_size_t(0))

    def _call(self, name, *args):
        assert getattr(self._hip, name)(*args) == 0, name

    def launch(self, stream):
        self._call("hipGraphLaunch", self.exec, ctypes.c_void_p(stream))

    def close(self):
        self._call("hipGraphExecDestroy", self.exec)
        self._call("hipGraphDestroy", self.graph)
