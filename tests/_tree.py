"""Trees of drafted tokens over a paged KV cache and rows of logits, in 64 bits with
numpy: what the tests of the tree entry points check against."""
from __future__ import annotations

import numpy as np

import llmpager_amd as lp
from _paged import GROUP, Batch, q4


def ancestors(up):
    """(depths, masks as whole numbers) of the nodes with parents `up`."""
    deep, masks = [], []
    for i, p in enumerate(up):
        has = 0 <= p < i
        deep.append(deep[p] + 1 if has else 0)
        masks.append((1 << i) | (masks[p] if has else 0))
    return deep, masks


def random_tree(rng, n, limit=1 << 30):
    up, deep = [-1], [0]
    for i in range(1, n):
        p = int(i * rng.uniform(0.1, 1.0))
        while deep[p] >= limit:
            p = up[p]
        up.append(p)
        deep.append(deep[p] + 1)
    return up


def words_of(masks, words):
    """Whole numbers as rows of 64-bit words."""
    return np.array([[m >> (64 * w) & ((1 << 64) - 1) for w in range(words)] for m in masks], np.uint64).reshape(len(masks), words)


class Trees(Batch):
    """A batch whose sequences' new tokens are trees (lists of parents)."""

    def __init__(self, cuda, trees, past, heads, kv, dim, page, fmt, max_q=None, **kw):
        super().__init__(cuda, [len(t) for t in trees], past, heads, kv, dim, page, fmt, **kw)
        self.trees = trees
        self.max_q = max_q or max(self.new + [1])
        self.words = (self.max_q + 63) // 64
        pad = self.tokens - self.live
        self.parents = np.array([p for t in trees for p in t] + [0] * pad, np.int32)
        self.depths = np.array([d for t in trees for d in ancestors(t)[0]] + [9] * pad, np.int32)
        self.bits = [m for t in trees for m in ancestors(t)[1]] + [1] * pad

    def masks(self):
        return words_of(self.bits, self.words)

    def append_tree(self, q, k, v, qw, kw, eps, mscale=1.0):
        """(q_out, values as held of k and v [tokens, kv, D], both pools after)."""
        qo = np.zeros((self.tokens, self.heads, self.dim))
        held = [np.zeros((self.tokens, self.kv, self.dim)) for _ in range(2)]
        pools = [p.copy() for p in self.pools]
        for t, b, row in self.places():
            pos = self.past[b] + float(self.depths[t])
            qo[t] = self.turned(q[t].reshape(self.heads, self.dim), qw, eps, pos, mscale)
            for n, x in enumerate((self.turned(k[t].reshape(self.kv, self.dim), kw, eps, pos, mscale),
                                   v[t].reshape(self.kv, self.dim).astype(np.float64))):
                col = row // self.page
                page = self.table[b, col] if col < self.cols else -1
                r, ok = row % self.page, 0 <= page < self.pages
                if self.fmt == lp.KV_F16:
                    held[n][t] = x.astype(np.float16)
                    if ok:
                        pools[n].view(np.float16).reshape(self.pages, self.kv, self.page, self.dim)[page, :, r] = held[n][t]
                else:
                    codes, s = q4(x)
                    held[n][t] = ((codes - 8.0).reshape(self.kv, -1, GROUP) * s[..., None]).reshape(self.kv, -1)
                    if ok:
                        self.put_q4(pools[n], page, r, codes, s)
        return qo, held[0], held[1], pools

    def put_q4(self, pool, page, r, codes, s):
        G = self.dim // GROUP
        nb = self.page * G * 2
        pool[page, :, 2 * G * r:2 * G * (r + 1)] = s.astype(np.float16).view(np.uint8).reshape(self.kv, -1)
        pool[page, :, nb + r * self.dim // 2:nb + (r + 1) * self.dim // 2] = codes[:, 0::2] | codes[:, 1::2] << 4

    def attention_tree(self, q, scale, max_seq=None):
        """out [tokens, heads, D] of q [tokens, heads, D] by self.bits."""
        K, V = self.values(self.pools[0]), self.values(self.pools[1])
        out = np.zeros((self.tokens, self.heads, self.dim))
        G = self.heads // self.kv
        cap = min(max_seq or 1 << 30, self.cols * self.page)
        for b in range(self.batch):
            L = min(self.lens[b], cap)
            p0 = L - self.new[b]
            rows = np.arange(max(L, 0))
            page = self.table[b, rows // self.page]
            have = (page >= 0) & (page < self.pages)
            kk = K[np.where(have, page, 0), :, rows % self.page]
            vv = V[np.where(have, page, 0), :, rows % self.page]
            for i in range(min(self.new[b], self.max_q)):
                t = int(self.starts[b]) + i
                bit = np.array([bool(self.bits[t] >> int(j) & 1) if j < self.max_q else False for j in rows[rows >= p0] - p0], bool)
                see = have & np.concatenate((np.ones(min(max(p0, 0), len(rows)), bool), bit))
                if not see.any():
                    continue
                x = q[t].astype(np.float64).reshape(self.kv, G, self.dim)
                with np.errstate(invalid="ignore", over="ignore"):
                    s = np.einsum("kgd,rkd->kgr", x, kk[see]) * scale
                    p = np.exp(s - s.max(-1, keepdims=True))
                    out[t] = (np.einsum("kgr,rkd->kgd", p, vv[see]) / p.sum(-1, keepdims=True)).reshape(self.heads, -1)
        return out

    def keep(self, pools, paths):
        """The pools with the rows of each sequence's path one behind the other."""
        out = [p.copy() for p in pools]
        G, P = self.dim // GROUP, self.page
        parts = [(0, 2 * self.dim)] if self.fmt == lp.KV_F16 else [(0, 2 * G), (2 * G * P, self.dim // 2)]

        def page(b, row):
            if row < 0 or row // P >= self.cols:
                return -1
            p = int(self.table[b, row // P])
            return p if 0 <= p < self.pages else -1

        for b, path in enumerate(paths):
            for i, x in enumerate(path[:self.new[b]]):
                if not 0 <= x < self.new[b] or x == i:
                    continue
                a, z = self.past[b] + x, self.past[b] + i
                pa, pz = page(b, a), page(b, z)
                if pa < 0 or pz < 0:
                    continue
                for src, dst in zip(pools, out):
                    for at, n in parts:
                        dst[pz, :, at + z % P * n:at + (z % P + 1) * n] = src[pa, :, at + a % P * n:at + (a % P + 1) * n]
        return out


# ---- verification -----------------------------------------------------------------


def row_probs(x, temp):
    """p of a row of logits, None where nothing can be drawn."""
    x = x.astype(np.float64)
    if np.isnan(x).any() or (x == np.inf).any() or (x == -np.inf).all():
        return None
    if not temp > 0:
        p = np.zeros_like(x)
        p[int(np.argmax(x))] = 1.0
        return p
    e = np.exp((x - x.max()) / float(np.float32(temp)))
    return e / e.sum()


def pick(w, u):
    """The first id where the sums of w pass u of the whole."""
    n = np.cumsum(w)
    some = np.flatnonzero(w > 0)
    return int(some[min(np.searchsorted(n[some], u * n[-1], side="right"), len(some) - 1)])


def verify_one(x, drafts, up, temp, u, q, max_depth):
    """(path, next) of one sequence: x, q [n, vocab], drafts, up, u [n]."""
    path = [0]
    while True:
        here = path[-1]
        p = row_probs(x[here], temp)
        if p is None:
            return path, -1
        kids = [j for j in range(here + 1, len(up)) if up[j] == here] if len(path) <= max_depth else []
        kids = [j for j in kids if 0 <= drafts[j] < x.shape[1]]
        if q is None or not temp > 0:
            z = pick(p, float(u[here])) if temp > 0 else int(np.argmax(p))
            kids = [j for j in kids if drafts[j] == z]
            if not kids:
                return path, z
            path.append(kids[0])
            continue
        left, took = p, None
        for j in kids:
            d = drafts[j]
            if float(u[j]) * float(q[here][d]) < left[d]:
                took = j
                break
            rest = np.maximum(left - q[here].astype(np.float64), 0.0)
            left = rest / rest.sum() if rest.sum() > 0 else p
        if took is None:
            return path, pick(left, float(u[0]))
        path.append(took)


def verify(x, drafts, trees, starts, temps, u, q, max_depth):
    """(path [batch, max_depth + 1], kept, next)."""
    path = np.full((len(trees), max_depth + 1), -1, np.int32)
    kept, nxt = np.zeros(len(trees), np.int32), np.full(len(trees), -1, np.int32)
    for b, up in enumerate(trees):
        if not up:
            continue
        s = slice(int(starts[b]), int(starts[b]) + len(up))
        p, nxt[b] = verify_one(x[s], drafts[s], up, float(temps[b]), u[s], None if q is None else q[s], max_depth)
        kept[b] = len(p)
        path[b, :len(p)] = p
    return path, kept, nxt
