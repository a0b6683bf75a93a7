"""The operators of a step with drafted tokens over a batch's paged KV cache, as
calls to be timed.  Each sequence's new tokens are a tree: node 0 its last token,
the others drafted to follow a lower node.

  layout  Kernels.tree_layout: the nodes' depths and the masks of their ancestors
  append  Kernels.kv_append_tree: queries and keys normed per head and rotated by
          their nodes' depths, keys and values written into their pages
  attn    Kernels.attn_tree: queries over the pages of their context and, of the
          tree, over the rows that their masks name
  verify  Kernels.verify_tree: the drafted tokens that the target's logits keep, by
          given random numbers, and the token behind them
  keep    Kernels.kv_keep: the rows of the kept tokens moved one behind the other,
          in the caches of all layers

Pages hold `page` rows of one KV head, in fp16 or in the repository's q4 regions
(groups of 32 columns, f16 scales, then nibbles holding q + 8).  Attention shapes
are those of the repository's tests and bench (32 or 64 heads on 4 KV heads of 128)
and generic ones; the vocabulary and the 48 layers are the bench's."""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
EPS, THETA = 1e-6, 1e6
GROUP = 32                        # columns of a q4 scale
S_MIN, S_MAX = 2.0 ** -17, 896.0  # what a q4 page's scales may be


def listed():
    big = dict(heads=32, kv=4, dim=128)
    wide = dict(heads=64, kv=4, dim=128)
    return [
        # one conversation's tree of drafts: the latency of a launch
        dict(name="layout_b1", kind="layout", seqs=1, nodes=26, depth=5),
        # a serving batch's large trees
        dict(name="layout_b64", kind="layout", seqs=64, nodes=256, depth=12),
        # one conversation's drafts into a 4-bit cache
        dict(name="append_b1", kind="append", q4=True, seqs=1, nodes=26, depth=5, past=1500, page=64, **big),
        # a serving batch's drafts into an fp16 cache in small pages
        dict(name="append_b32", kind="append", q4=False, seqs=32, nodes=60, depth=8, past=4000, page=16, **wide),
        # one conversation's drafts over its context
        dict(name="attn_b1", kind="attn", q4=False, seqs=1, nodes=26, depth=5, past=1500, page=64, **big),
        # a serving batch's drafts over a 4-bit cache
        dict(name="attn_b16_q4", kind="attn", q4=True, seqs=16, nodes=32, depth=6, past=6000, page=64, **big),
        # few requests, each with as many drafts as spare compute allows
        dict(name="attn_wide", kind="attn", q4=False, seqs=4, nodes=256, depth=12, past=3001, page=16, **wide),
        # one conversation: which drafts stay
        dict(name="verify_b1", kind="verify", probs=False, greedy=0.0, seqs=1, nodes=26, depth=5, vocab=151936),
        # a serving batch of large trees, some requests at temperature 0
        dict(name="verify_b32", kind="verify", probs=False, greedy=0.3, seqs=32, nodes=60, depth=8, vocab=151936),
        # a serving batch of chains that a smaller model has drawn: its probabilities count
        dict(name="verify_chains", kind="verify", probs=True, greedy=0.0, seqs=32, nodes=6, depth=5, chain=True, vocab=151936),
        # one conversation's kept drafts, in the caches of 48 layers
        dict(name="keep_b1", kind="keep", q4=True, seqs=1, nodes=26, depth=5, past=300, page=64, layers=48, **big),
        # a serving batch's
        dict(name="keep_b64", kind="keep", q4=False, seqs=64, nodes=60, depth=8, past=90, page=16, layers=48, **big),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


SHAPES = [(32, 4, 128), (32, 4, 128), (64, 4, 128), (32, 8, 128), (16, 2, 128), (8, 8, 64), (24, 8, 64), (12, 4, 64),
          (5, 1, 128), (16, 1, 64)]


def draw(rng):
    kind = rng.choice(["layout", "append", "append", "attn", "attn", "attn", "attn", "verify", "verify", "verify", "keep"])
    nodes = _log(rng, 2, 256)
    c = dict(kind=kind, nodes=nodes, depth=rng.randint(1, 12), chain=rng.random() < 0.15)
    if kind == "layout":
        return dict(c, seqs=_log(rng, 1, 64), pad=rng.choice([0, 3]))
    if kind == "verify":
        vocab = _log(rng, 1000, 200000)
        probs = rng.random() < 0.4
        nodes = rng.randint(2, 8) if probs else min(nodes, 64)
        seqs = _log(rng, 1, max(2, min(32, int(2.4e8 / vocab / nodes))))
        return dict(c, probs=probs, greedy=rng.choice([0.0, 0.0, 0.4, 1.0]), seqs=seqs, nodes=nodes, vocab=vocab,
                    pad=rng.choice([0, 2]), chain=rng.random() < (0.6 if probs else 0.15))
    heads, kv, dim = rng.choice(SHAPES)
    c.update(q4=rng.random() < 0.5, heads=heads, kv=kv, dim=dim, page=rng.choice([16, 32, 64, 128, 256]), pad=rng.choice([0, 0, 3]))
    if kind == "append":
        return dict(c, seqs=_log(rng, 1, max(1, min(32, 1800 // nodes))), past=_log(rng, 1, 6000))
    if kind == "attn":
        return dict(c, seqs=_log(rng, 1, max(2, min(32, 700 // nodes))), past=rng.choice([0, _log(rng, 1, 3000), _log(rng, 16, 3000)]))
    return dict(c, nodes=rng.randint(16, 64), page=min(c["page"], 64), seqs=_log(rng, 1, 32), past=_log(rng, 1, 90),
                layers=rng.choice([1, 2, 24]))


def _trees(c, seed=None):
    """Each sequence's parents (-1: the root's) and context length with its new
    tokens: the first sequence is the largest.  Lengths go by the case alone, and the
    parents too where no seed is given."""
    r = random.Random("%d %d %d" % (c["seqs"], c["nodes"], c["depth"]))
    t = r if seed is None else random.Random("tree %d" % seed)
    trees, lens = [], []
    for b in range(c["seqs"]):
        n = c["nodes"] if b == 0 else max(1, int(c["nodes"] * r.uniform(0.4, 1.0)))
        up, deep = [-1], [0]
        for i in range(1, n):
            p = i - 1 if c.get("chain") and seed is None else int(i * t.uniform(0.1, 1.0))
            while deep[p] >= c["depth"] and (seed is not None or not c.get("chain")):
                p = up[p]
            up.append(p)
            deep.append(deep[p] + 1)
        trees.append(up)
        past = c.get("past", 0)
        lens.append(n + (past if b == 0 else int(past * r.uniform(0.2, 1.0))))
    return trees, lens


def _stays(c, node, at):
    return node == at or node > c["depth"]


def _paths(c):
    """The nodes of each sequence that are kept, the root first: down from it at
    random, all but the first stopping early now and then.  To be moved, those that are where they are to be or
    behind all that could be kept, so that a second pass finds and leaves the same rows."""
    r = random.Random("path %d %d %d" % (c["seqs"], c["nodes"], c["depth"]))
    out = []
    for up in _trees(c)[0]:
        path = [0]
        while len(path) <= c["depth"]:
            below = [i for i in range(len(up)) if up[i] == path[-1] and (not c["kind"] == "keep" or _stays(c, i, len(path)))]
            if not below or (out and r.random() < 0.2):
                break
            path.append(r.choice(below))
        out.append(path)
    return out


def _words(c):
    return (c["nodes"] + 63) // 64


def _row_bytes(c):
    return c["dim"] // 2 + c["dim"] // GROUP * 2 if c["q4"] else 2 * c["dim"]


def _ancestors(up):
    """Per node the whole number with a bit for itself and each node above it."""
    m = []
    for i, p in enumerate(up):
        m.append((1 << i) | (m[p] if p >= 0 else 0))
    return m


def work(c):
    trees, lens = _trees(c)
    T, W = sum(map(len, trees)), _words(c)
    kind = c["kind"]
    if kind == "layout":
        return {"bytes": T * (8 + 8 * W), "flops": 0}
    if kind == "verify":
        # chosen drafts: the rows of the nodes on the path; sampled ones: of every
        # node, and the draft's own of a node where one is turned down
        rows = T + len(trees) if c["probs"] else sum(map(len, _paths(c)))
        return {"bytes": rows * c["vocab"] * 4 + T * 16, "flops": 4 * rows * c["vocab"]}
    kv, D = c["kv"], c["dim"]
    if kind == "keep":
        rows = sum(i != x for p in _paths(c) for i, x in enumerate(p))
        return {"bytes": 2 * rows * 2 * kv * _row_bytes(c) * c["layers"] + 4 * sum(map(len, _paths(c))), "flops": 0}
    H = c["heads"]
    if kind == "append":
        return {"bytes": T * ((2 * H + 2 * kv) * D * 4 + 2 * kv * _row_bytes(c) + (2 * kv * D * 4 if c["q4"] else 0)),
                "flops": T * (H + kv) * D * 8 + T * kv * D * 4}
    pairs = sum(len(up) * (n - len(up)) + sum(bin(m).count("1") for m in _ancestors(up)) for up, n in zip(trees, lens))
    return {"bytes": 2 * T * H * D * 4 + 2 * sum(lens) * kv * _row_bytes(c) + 8 * T * W, "flops": 4 * D * H * pairs}


# ---- inputs ----------------------------------------------------------------


def _round7(x):
    """x > 0 to 7 significant bits, ties to even."""
    m, e = torch.frexp(x)
    return torch.ldexp(torch.round(m * 128.0) / 128.0, e)


def _quantise(x):
    """(codes 0 .. 15, scales) of x [..., D], in x's own precision."""
    g = x.unflatten(-1, (-1, GROUP))
    s = _round7(g.abs().amax(-1) / 7.0).clamp(S_MIN, S_MAX)
    return (torch.round(g / s[..., None]).clamp(-7, 7) + 8).flatten(-2).to(torch.uint8), s.to(torch.float16)


def _pool(g, c, pages):
    """Filled pages, bytes [pages, kv, page bytes]: rows of normal values with a
    part in common."""
    kv, P, D = c["kv"], c["page"], c["dim"]
    out = torch.empty(pages, kv, P * _row_bytes(c), dtype=torch.uint8, device=DEV)
    common = torch.randn(kv, 1, D, generator=g, device=DEV) * 0.4
    at = 0
    while at < pages:
        n = min(pages - at, max(1, (1 << 26) // (kv * P * D)))
        x = torch.randn(n, kv, P, D, generator=g, device=DEV) + common
        if c["q4"]:
            codes, s = _quantise(x)
            nib = codes[..., 0::2] | (codes[..., 1::2] << 4)
            out[at:at + n] = torch.cat((s.reshape(n, kv, -1).view(torch.uint8), nib.reshape(n, kv, -1)), 2)
        else:
            out[at:at + n] = x.to(torch.float16).reshape(n, kv, -1).view(torch.uint8)
        at += n
    return out


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _signed(x):
    """The 64-bit pattern x as int64 holds it."""
    return x - (1 << 64) if x >> 63 else x


def prepare(c, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 2654435761 % (1 << 62) + 1)
    trees, lens = _trees(c, seed if c["kind"] == "layout" else None)
    B, T, W = c["seqs"], sum(map(len, trees)) + c.get("pad", 0), _words(c)
    new = [len(up) for up in trees]
    s = dict(c=c, tokens=T, max_q=c["nodes"], max_seq=max(lens), lens=_i32(lens),
             starts=_i32([0] + new).cumsum(0).to(torch.int32))
    s["parents"] = _i32([p for up in trees for p in up] + [-1] * c.get("pad", 0))
    if own:
        cuda, s["K"] = _cuda()
    if c["kind"] == "layout":
        s["depths"] = torch.zeros(T, dtype=torch.int32, device=DEV)
        s["masks"] = torch.zeros(T, W, dtype=torch.int64, device=DEV)
        return s
    if c["kind"] == "verify":
        return _prepare_verify(s, g, trees)
    H, kv, D, P = c["heads"], c["kv"], c["dim"], c["page"]
    need = [-(-n // P) for n in lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    cols = max(need) + 1
    at = torch.tensor([0] + need[:-1]).cumsum(0)[:, None] + torch.arange(cols)
    table = order[at.clamp(max=pages - 1).to(DEV)]
    table[torch.arange(cols, device=DEV) >= _i32(need)[:, None]] = -1
    s["table"] = table.contiguous()
    s["all"] = torch.stack([_pool(g, c, pages) for _ in range(2 * c.get("layers", 1))])
    s["pools"] = [(s["all"][i], s["all"][i + 1]) for i in range(0, len(s["all"]), 2)]
    if own:
        import llmpager_amd as lp

        s["caches"] = (lp.KvCache * len(s["pools"]))(*(
            lp.KvCache(k_pages=k.data_ptr(), v_pages=v.data_ptr(), table=s["table"].data_ptr(), pages=pages, page_rows=P,
                       max_pages=cols, kv_heads=kv, head_dim=D, format=lp.KV_Q4 if c["q4"] else lp.KV_F16)
            for k, v in s["pools"]))
    if c["kind"] == "keep":
        paths = _paths(c)
        s["path"] = _i32([p + [-1] * (c["depth"] + 1 - len(p)) for p in paths])
        s["kept"] = _i32([len(p) for p in paths])
        s["lens_out"] = torch.zeros(B, dtype=torch.int32, device=DEV)
        return s
    if c["kind"] == "append":
        deep = []
        for up in trees:
            at = len(deep)
            for p in up:
                deep.append(deep[at + p] + 1 if p >= 0 else 0)
        s["depths"] = _i32(deep + [0] * c.get("pad", 0))
        # a projection's output: queries, keys and values of a token side by side
        s["qkv"] = torch.randn(T, (H + 2 * kv) * D, generator=g, device=DEV)
        s["qn"], s["kn"] = (0.8 + torch.rand(D, generator=g, device=DEV) for _ in range(2))
        s["freq"] = (THETA ** (-torch.arange(0, D, 2, device=DEV, dtype=torch.float64) / D)).float()
        s["q"] = torch.zeros(T, H * D, device=DEV)
        s["kout"], s["vout"] = (torch.zeros(T, kv * D, device=DEV) for _ in range(2))
        return s
    masks = [[_signed(m >> (64 * w) & ((1 << 64) - 1)) for w in range(W)] for up in trees for m in _ancestors(up)]
    s["masks"] = torch.tensor(masks + [[0] * W] * c.get("pad", 0), dtype=torch.int64, device=DEV)
    s["q"] = torch.randn(T, H * D, generator=g, device=DEV) * 1.5
    s["out"] = torch.zeros(T, H * D, device=DEV)
    if own:
        n = s["K"].attn_tree_ws_bytes(s["caches"][0], H, B, T, s["max_q"], s["max_seq"])
        s["ws"] = torch.empty(max(256, n), dtype=torch.uint8, device=DEV)
    return s


def _prepare_verify(s, g, trees):
    c, B, T, V = s["c"], s["c"]["seqs"], s["tokens"], s["c"]["vocab"]
    # most rows are undecided between a few tokens, some are sure of one
    x = torch.empty(T, V, device=DEV)
    for at in range(0, T, 256):
        y = x[at:at + 256]
        y.normal_(generator=g).mul_(2.0)
        y += 5.0 * (torch.rand(y.shape, generator=g, device=DEV) > 0.9995)
        y.copy_(y.to(torch.bfloat16))
    x[::3, V // 3] += 14.0
    s["logits"] = x
    r = random.Random("temperatures %d %d" % (B, V))
    temps = [0.0 if r.random() < c["greedy"] else r.choice([0.6, 0.8, 1.0]) for _ in range(B)]
    s["temps"] = torch.tensor(temps, device=DEV)
    s["uniforms"] = torch.rand(T, generator=g, device=DEV)
    starts = s["starts"].tolist()
    above = _i32([max(starts[b] + p, 0) if p >= 0 else starts[b] for b, up in enumerate(trees) for p in up]
                 + [0] * c.get("pad", 0)).long()
    s["probs"] = None
    if c["probs"]:
        # a smaller model's distributions, near the target's, and its draws
        s["probs"] = torch.empty(T, V, device=DEV)
        t = s["temps"].clamp(min=0.5).repeat_interleave(s["starts"].diff(), output_size=T - c.get("pad", 0))
        t = torch.cat((t, torch.ones(c.get("pad", 0), device=DEV)))
        for at in range(0, T, 256):
            y = x[at:at + 256] + torch.randn(x[at:at + 256].shape, generator=g, device=DEV) * 0.7
            s["probs"][at:at + 256] = torch.softmax(y / t[at:at + 256, None], 1)
        s["drafts"] = torch.cat([torch.multinomial(s["probs"][a], 1, generator=g) for a in above.split(256)])[:, 0].to(torch.int32)
    else:
        # the best tokens of the row above, but along each path the token that is drawn there
        pick = torch.randint(0, 8, (T,), generator=g, device=DEV)
        top = torch.cat([x[a].topk(8, 1).indices for a in above.split(256)])
        s["drafts"] = top.gather(1, pick[:, None])[:, 0].to(torch.int32)
        paths = _paths(c)
        for level in range(max(map(len, paths))):
            on = [b for b in range(B) if level < len(paths[b])]
            rows = _i32([starts[b] + paths[b][level] for b in on]).long()
            z = _plain_draw(x[rows], s["temps"][on], s["uniforms"][rows])
            below, want, use = [], [], []
            for i, b in enumerate(on):
                nxt = paths[b][level + 1] if level + 1 < len(paths[b]) else -1
                for j, p in enumerate(trees[b]):
                    if p == paths[b][level]:
                        below.append(starts[b] + j), use.append(i), want.append(j == nxt)
            if below:
                at, z = _i32(below).long(), z[torch.tensor(use, device=DEV)].to(torch.int32)
                d = s["drafts"][at]
                s["drafts"][at] = torch.where(torch.tensor(want, device=DEV), z, torch.where(d == z, (d + 1) % V, d))
    s["path"] = torch.zeros(B, c["depth"] + 1, dtype=torch.int32, device=DEV)
    s["kept"], s["next"] = (torch.zeros(B, dtype=torch.int32, device=DEV) for _ in range(2))
    if own:
        n = s["K"].verify_tree_ws_bytes(V, B, T, s["max_q"], c["depth"], c["probs"])
        s["ws"] = torch.empty(max(256, n), dtype=torch.uint8, device=DEV)
    return s


_handles = []


def _cuda():
    """This process's context and launchers."""
    if not _handles:
        import llmpager_amd as lp

        torch.cuda.init()
        cuda = lp.Cuda(0)
        _handles.extend((cuda, lp.Kernels(cuda)))
    return _handles


# ---- the framework's calls -----------------------------------------------------


def _own_layout(s):
    s["K"].tree_layout(s["parents"].data_ptr(), s["starts"].data_ptr(), s["c"]["seqs"], s["tokens"], s["max_q"],
                       s["depths"].data_ptr(), s["masks"].data_ptr())


def _own_append(s):
    c, D = s["c"], s["c"]["dim"]
    H, kv = c["heads"], c["kv"]
    W, at = (H + 2 * kv) * D, s["qkv"].data_ptr()
    s["K"].kv_append_tree(s["caches"][0], at, W, at + H * D * 4, W, at + (H + kv) * D * 4, W, s["qn"].data_ptr(),
                          s["kn"].data_ptr(), EPS, s["freq"].data_ptr(), 1.0, s["q"].data_ptr(), H * D,
                          s["kout"].data_ptr() if c["q4"] else 0, s["vout"].data_ptr() if c["q4"] else 0, H,
                          s["starts"].data_ptr(), s["lens"].data_ptr(), s["depths"].data_ptr(), c["seqs"], s["tokens"])


def _own_attn(s):
    c = s["c"]
    W = c["heads"] * c["dim"]
    s["K"].attn_tree(s["caches"][0], s["q"].data_ptr(), W, s["out"].data_ptr(), W, c["heads"], s["starts"].data_ptr(),
                     s["lens"].data_ptr(), s["masks"].data_ptr(), c["seqs"], s["tokens"], s["max_q"], s["max_seq"],
                     1.0 / math.sqrt(c["dim"]), s["ws"].data_ptr(), ws_bytes=s["ws"].numel())


def _own_verify(s):
    c = s["c"]
    s["K"].verify_tree(s["logits"].data_ptr(), c["vocab"], c["vocab"], s["drafts"].data_ptr(), s["parents"].data_ptr(),
                       s["starts"].data_ptr(), c["seqs"], s["tokens"], s["max_q"], c["depth"], s["temps"].data_ptr(),
                       s["probs"].data_ptr() if c["probs"] else 0, c["vocab"], s["uniforms"].data_ptr(),
                       s["path"].data_ptr(), s["kept"].data_ptr(), s["next"].data_ptr(), s["ws"].data_ptr(),
                       ws_bytes=s["ws"].numel())


def _own_keep(s):
    s["K"].kv_keep(s["caches"], s["path"].data_ptr(), s["c"]["depth"], s["kept"].data_ptr(), s["starts"].data_ptr(),
                   s["lens"].data_ptr(), s["lens_out"].data_ptr(), s["c"]["seqs"])


# ---- plain forms ------------------------------------------------------------------


def _places(s):
    """Each token's sequence, its number there and its row; which tokens belong to one."""
    t = torch.arange(s["tokens"], device=DEV)
    starts = s["starts"].long()
    b = (starts[None, 1:] <= t[:, None]).sum(1)
    live = b < len(s["lens"])
    b = b.clamp(max=len(s["lens"]) - 1)
    return live, b, t - starts[b], s["lens"].long()[b] - (starts[b + 1] - t)


def _plain_layout(s):
    live, b, i, _ = _places(s)
    first = s["starts"].long()[b]
    p = s["parents"].long()
    has = live & (p >= 0) & (p < i)
    at = torch.arange(s["tokens"], device=DEV)
    up = torch.where(has, first + p, at)
    see = i[:, None] == torch.arange(64 * _words(s["c"]), device=DEV)
    for _ in range(max(1, s["max_q"].bit_length())):  # twice as far up each time
        see = see | see[up]
        up = up[up]
    s["depths"][live] = (see.sum(1) - 1).to(torch.int32)[live]
    bit = torch.ones(64, dtype=torch.int64, device=DEV) << torch.arange(64, device=DEV)
    s["masks"][live] = (see.unflatten(1, (-1, 64)) * bit).sum(2)[live]


def _plain_append(s):
    c = s["c"]
    H, kv, D, P = c["heads"], c["kv"], c["dim"], c["page"]
    live, b, i, row = _places(s)
    # 64 bits: angles of far positions, and 4-bit values next to a border
    x = s["qkv"].double()
    q, k, v = (y.unflatten(1, (-1, D)) for y in x.split([H * D, kv * D, kv * D], 1))
    ang = (row - i + s["depths"]).double()[:, None, None] * s["freq"].double()
    cs, sn = ang.cos(), ang.sin()

    def turned(y, w):
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * w.double()
        a, z = y[..., :D // 2], y[..., D // 2:]
        return torch.cat((a * cs - z * sn, a * sn + z * cs), -1)

    s["q"][live] = turned(q, s["qn"]).flatten(1).float()[live]
    k = turned(k, s["kn"])[live]
    v = v[live]
    page, at = s["table"][b, row.clamp(min=0) // P].long()[live], (row % P)[live]
    for new, pool, out in zip((k, v), s["pools"][0], (s["kout"], s["vout"])):
        if c["q4"]:
            G = D // GROUP
            codes, scales = _quantise(new)
            pool.view(torch.float16)[..., :P * G].unflatten(2, (P, G))[page, :, at] = scales
            pool[..., 2 * P * G:].unflatten(2, (P, D // 2))[page, :, at] = codes[..., 0::2] | (codes[..., 1::2] << 4)
            out[live] = ((codes.float() - 8.0).unflatten(2, (G, GROUP)) * scales.float()[..., None]).flatten(1)
        else:
            pool.view(torch.float16).unflatten(2, (P, D))[page, :, at] = new.to(torch.float16)


def _rows(s, pool, n, dtype):
    """Rows 0 .. n - 1 of every sequence as [seqs, kv, n, D]; rows past a
    sequence's end are zero."""
    c = s["c"]
    D, P = c["dim"], c["page"]
    r = torch.arange(n, device=DEV)
    here = r < s["lens"][:, None]
    page, row = s["table"][:, r // P].long().clamp(min=0), (r % P).expand(len(s["lens"]), n)
    if c["q4"]:
        G = D // GROUP
        sc = pool.view(torch.float16)[..., :P * G].unflatten(2, (P, G))[page, :, row].to(dtype)
        b = pool[..., 2 * P * G:].unflatten(2, (P, D // 2))[page, :, row]
        x = torch.stack((b & 15, b >> 4), -1).flatten(-2).to(dtype) - 8.0
        x = (x.unflatten(-1, (G, GROUP)) * sc[..., None]).flatten(-2)
    else:
        x = pool.view(torch.float16).unflatten(2, (P, D))[page, :, row].to(dtype)
    return torch.where(here[:, :, None, None], x, 0).transpose(1, 2).contiguous()


def _plain_attn(s):
    c = s["c"]
    H, kv, D = c["heads"], c["kv"], c["dim"]
    B, Q, N, G = c["seqs"], s["max_q"], s["max_seq"], c["heads"] // c["kv"]
    starts, lens = s["starts"].long(), s["lens"].long()
    i = torch.arange(Q, device=DEV)
    new = starts[1:] - starts[:-1]
    live = i < new[:, None]
    t = (starts[:-1, None] + i).clamp(max=s["tokens"] - 1)
    q = s["q"][t].view(B, Q, kv, G, D).permute(0, 2, 1, 3, 4).reshape(B, kv, Q * G, D)
    k, v = (_rows(s, p, N, torch.float32) for p in s["pools"][0])
    x = q @ k.transpose(2, 3).contiguous() * (1.0 / math.sqrt(D))
    j = torch.arange(N, device=DEV) - (lens - new)[:, None]                         # [B, N]: the node of a row
    bits = s["masks"][t].gather(2, (j.clamp(0, Q - 1) // 64)[:, None].expand(B, Q, N))
    bits = bits >> (j.clamp(min=0) % 64)[:, None] & 1                               # [B, Q, N]
    seen = (j < 0)[:, None] | (bits.bool() & (j < new[:, None])[:, None])
    seen = seen.repeat_interleave(G, 1)[:, None]
    x = torch.where(seen, x, -math.inf)
    p = torch.where(seen, torch.exp(x - x.amax(-1, keepdim=True)), 0)
    norm = p.sum(-1, keepdim=True)
    y = torch.where(norm > 0, p @ v / norm, 0)
    y = y.view(B, kv, Q, G, D).permute(0, 2, 1, 3, 4).reshape(B, Q, H * D)
    s["out"][t[live]] = y[live]


def _plain_draw(x, temps, u):
    """The token of each row x [n, V]: the first whose probability with those before
    it passes u, at temperature 0 the first of the largest.  64 bits: the sums' borders."""
    y = x.double() - x.amax(1, keepdim=True)
    e = torch.exp(y / torch.where(temps > 0, temps, 1.0).double()[:, None])
    n = e.cumsum(1)
    hot = (n <= u.double()[:, None] * n[:, -1:]).sum(1).clamp(max=x.shape[1] - 1)
    return torch.where(temps > 0, hot, (y == 0).to(torch.uint8).argmax(1))


def _plain_verify(s):
    c, x, starts = s["c"], s["logits"], s["starts"].long()
    B, Q = c["seqs"], s["max_q"]
    b = torch.arange(B, device=DEV)
    i = torch.arange(Q, device=DEV)
    t = (starts[:-1, None] + i).clamp(max=s["tokens"] - 1)
    up = torch.where(i < (starts[1:] - starts[:-1])[:, None], s["parents"][t].long(), -2)
    drafts = s["drafts"].long()[t]
    cur, done = torch.zeros(B, dtype=torch.long, device=DEV), torch.zeros(B, dtype=torch.bool, device=DEV)
    length = torch.ones_like(cur)
    path, nxt = torch.full_like(s["path"], -1), torch.full_like(cur, -1)
    path[:, 0] = 0

    def go(to, where):
        path[b, length.clamp(max=c["depth"])] = torch.where(where, to, path[b, length.clamp(max=c["depth"])].long()).to(torch.int32)
        return length + where, torch.where(where, to, cur)

    if not c["probs"]:
        for _ in range(c["depth"] + 1):
            rows = starts[:-1] + cur
            z = _plain_draw(x[rows], s["temps"], s["uniforms"][rows])
            fits = (up == cur[:, None]) & (drafts == z[:, None])
            on = ~done & fits.any(1) & (length <= c["depth"])
            nxt = torch.where(done, nxt, z)
            done = ~on
            length, cur = go(fits.to(torch.uint8).argmax(1), on)
    else:
        # 64 bits: what is left of a distribution after another's part is taken
        cold = s["temps"] <= 0
        last = torch.zeros_like(cur)  # children up to it have been tried
        a, Z = torch.zeros(B, 1, dtype=torch.float64, device=DEV), torch.ones(B, 1, dtype=torch.float64, device=DEV)
        u = s["uniforms"].double()
        for _ in range(Q):
            rows = starts[:-1] + cur
            y = x[rows].double() - x[rows].amax(1, keepdim=True)
            p = torch.exp(y / torch.where(cold, 1.0, s["temps"]).double()[:, None])
            p = torch.where(cold[:, None], torch.nn.functional.one_hot((y == 0).to(torch.uint8).argmax(1), c["vocab"]), p / p.sum(1, keepdim=True))
            q = s["probs"][rows].double()
            R = (p - a * q).clamp(min=0)
            n = R.cumsum(1)
            z = (n <= u[starts[:-1]][:, None] * n[:, -1:]).sum(1).clamp(max=c["vocab"] - 1)
            below = (up == cur[:, None]) & (i > last[:, None])
            has = below.any(1) & (length <= c["depth"]) & ~done
            nxt = torch.where(done, nxt, z)
            done = ~has
            child = below.to(torch.uint8).argmax(1)
            d = drafts[b, child][:, None]
            rc, qc = R.gather(1, d), q.gather(1, d)
            keeps = torch.where(cold[:, None], rc > 0, u[t[b, child]][:, None] * qc * Z < rc)[:, 0] & has
            length, cur = go(child, keeps)
            last = torch.where(has, child, last)
            turned = (has & ~keeps & ~cold)[:, None]
            a1 = torch.where(turned, a + Z, torch.where(keeps[:, None], 0.0, a))
            Z = torch.where(turned, (p - a1 * q).clamp(min=0).sum(1, keepdim=True), torch.where(keeps[:, None], 1.0, Z))
            a = a1
            last = torch.where(keeps, torch.zeros_like(last), last)
        # the node that the last round came to
        rows = starts[:-1] + cur
        y = x[rows].double() - x[rows].amax(1, keepdim=True)
        p = torch.exp(y / torch.where(cold, 1.0, s["temps"]).double()[:, None])
        n = (p / p.sum(1, keepdim=True) - a * s["probs"][rows].double()).clamp(min=0).cumsum(1)
        z = (n <= u[starts[:-1]][:, None] * n[:, -1:]).sum(1).clamp(max=c["vocab"] - 1)
        nxt = torch.where(done, nxt, torch.where(cold, (y == 0).to(torch.uint8).argmax(1), z))
    s["path"].copy_(path)
    s["kept"].copy_(length)
    s["next"].copy_(nxt)


def _plain_keep(s):
    c, starts, lens = s["c"], s["starts"].long(), s["lens"].long()
    D, P = c["dim"], c["page"]
    first = lens - (starts[1:] - starts[:-1])
    i = torch.arange(c["depth"] + 1, device=DEV)
    on = i < s["kept"][:, None]
    b = torch.arange(c["seqs"], device=DEV)[:, None].expand_as(on)[on]
    src, dst = (first[:, None] + s["path"])[on], (first[:, None] + i)[on]
    ps, pd = s["table"][b, src // P].long(), s["table"][b, dst // P].long()
    for pool in s["all"]:
        if c["q4"]:
            G = D // GROUP
            for v in (pool.view(torch.float16)[..., :P * G].unflatten(2, (P, G)), pool[..., 2 * P * G:].unflatten(2, (P, D // 2))):
                v[pd, :, dst % P] = v[ps, :, src % P]
        else:
            v = pool.view(torch.float16).unflatten(2, (P, D))
            v[pd, :, dst % P] = v[ps, :, src % P]
    s["lens_out"].copy_(first + s["kept"])


PLAIN = dict(layout=_plain_layout, append=_plain_append, attn=_plain_attn, verify=_plain_verify, keep=_plain_keep)
OWN = dict(layout=_own_layout, append=_own_append, attn=_own_attn, verify=_own_verify, keep=_own_keep)


def run(s):
    c = s["c"]
    (OWN if own else PLAIN)[c["kind"]](s)
    if c["kind"] == "layout":
        return {"depths": s["depths"], "masks": s["masks"]}
    if c["kind"] == "append":
        if c["q4"]:  # the values that the 4-bit rows stand for
            return {"q": s["q"], "k": s["kout"], "v": s["vout"]}
        return {"q": s["q"], "kpages": s["pools"][0][0].view(torch.float16), "vpages": s["pools"][0][1].view(torch.float16)}
    if c["kind"] == "attn":
        return {"out": s["out"]}
    if c["kind"] == "verify":
        return {"path": s["path"], "kept": s["kept"], "next": s["next"]}
    # moved, not computed: the pages' bytes
    return {"lens": s["lens_out"], "pools": s["all"] if c["q4"] else s["all"].view(torch.float16)}


# ---- from the definition, in 64 bits --------------------------------------------------


def _exact_q4(x):
    """[n, D] as a q4 row stands for it."""
    g = x.reshape(-1, GROUP)
    s = g.abs().max(1).values / 7.0
    step = 2.0 ** (torch.floor(torch.log2(torch.where(s > 0, s, 1.0))) - 6.0)
    s = torch.round(s / step) * step
    s = torch.minimum(torch.maximum(s, torch.full_like(s, S_MIN)), torch.full_like(s, S_MAX))[:, None]
    return (torch.minimum(torch.maximum(torch.round(g / s), torch.full_like(g, -7)), torch.full_like(g, 7)) * s).reshape(x.shape)


def _exact_turn(x, w, pos, freq):
    """RMS norm of [n, D] by w, then pairs (i, i + D/2) turned by pos * freq[i]."""
    x = x / torch.sqrt((x * x).sum(1, keepdim=True) / x.shape[1] + EPS) * w
    z = torch.complex(x[:, :x.shape[1] // 2], x[:, x.shape[1] // 2:])
    z = z * torch.polar(torch.ones_like(freq), pos * freq)
    return torch.cat((z.real, z.imag), 1)


def _exact_page(c, raw):
    """One page's rows [kv, page, D] from its bytes [kv, page bytes]."""
    kv, P, D = c["kv"], c["page"], c["dim"]
    if not c["q4"]:
        return raw.contiguous().view(torch.float16).double().view(kv, P, D)
    n = P * (D // GROUP) * 2
    sc = raw[:, :n].contiguous().view(torch.float16).double().view(kv, P, D // GROUP, 1)
    lo, hi = (raw[:, n:] % 16).double() - 8, torch.div(raw[:, n:], 16, rounding_mode="floor").double() - 8
    return (torch.stack((lo, hi), 2).view(kv, P, D // GROUP, GROUP) * sc).view(kv, P, D)


def _exact_append(c, s, trees, lens):
    H, kv, D, P, T = c["heads"], c["kv"], c["dim"], c["page"], s["tokens"]
    Q = torch.zeros(T, H * D, dtype=torch.float64, device=DEV)
    K, V = (torch.zeros(T, kv * D, dtype=torch.float64, device=DEV) for _ in range(2))
    held = [] if c["q4"] else [p.view(torch.float16).double().unflatten(2, (P, D)) for p in s["pools"][0]]
    freq, t = s["freq"].double(), 0
    for b, (up, L) in enumerate(zip(trees, lens)):
        n = len(up)
        pos = torch.tensor([L - n + bin(m).count("1") - 1 for m in _ancestors(up)], dtype=torch.float64, device=DEV)[:, None]
        at = torch.arange(L - n, L, device=DEV)
        page = s["table"][b][at // P].long()
        for i in range(H + 2 * kv):
            x = s["qkv"][t:t + n, i * D:(i + 1) * D].double()
            if i < H:
                Q[t:t + n, i * D:(i + 1) * D] = _exact_turn(x, s["qn"].double(), pos, freq)
                continue
            k, h = i < H + kv, (i - H) % kv
            if k:
                x = _exact_turn(x, s["kn"].double(), pos, freq)
            if c["q4"]:
                (K if k else V)[t:t + n, h * D:(h + 1) * D] = _exact_q4(x)
            else:
                held[not k][page, h, at % P] = x
        t += n
    if c["q4"]:
        return {"q": Q, "k": K, "v": V}
    return {"q": Q, "kpages": held[0].flatten(2), "vpages": held[1].flatten(2)}


def _exact_attn(c, s, trees, lens):
    H, D, P, G = c["heads"], c["dim"], c["page"], c["heads"] // c["kv"]
    O, t = torch.zeros(s["tokens"], H * D, dtype=torch.float64, device=DEV), 0
    for b, (up, L) in enumerate(zip(trees, lens)):
        n = len(up)
        ids = s["table"][b, :-(-L // P)].tolist()
        k, v = (torch.cat([_exact_page(c, p[i]) for i in ids], 1)[:, :L] for p in s["pools"][0])
        seen = torch.ones(n, L, dtype=torch.bool)
        seen[:, L - n:] = torch.tensor([[m >> j & 1 for j in range(n)] for m in _ancestors(up)]).bool()
        seen = seen.to(DEV)
        q = s["q"][t:t + n].double().view(n, H, D)
        for h in range(H):
            a = torch.softmax((q[:, h] @ k[h // G].T / math.sqrt(D)).masked_fill(~seen, -math.inf), 1)
            O[t:t + n, h * D:(h + 1) * D] = a @ v[h // G]
        t += n
    return {"out": O}


def _exact_pick(w, u):
    """The first place where the sums of w pass u of the whole."""
    n = torch.cumsum(w, 0)
    return min(int(torch.searchsorted(n, u * float(n[-1]), right=True)), len(w) - 1)


def _exact_verify(c, s, trees):
    u, temps, drafts = s["uniforms"].double().tolist(), s["temps"].double().tolist(), s["drafts"].tolist()
    paths, nexts, t0 = [], [], 0
    for up, T in zip(trees, temps):
        def p_of(i):
            x = s["logits"][t0 + i].double()
            if T <= 0:
                p = torch.zeros_like(x)
                p[int(torch.nonzero(x == x.max())[0])] = 1.0
                return p
            return torch.softmax(x / T, 0)

        path = [0]
        while True:
            here = path[-1]
            p = p_of(here)
            below = [j for j in range(len(up)) if up[j] == here] if len(path) <= c["depth"] else []
            if not c["probs"]:
                z = _exact_pick(p, u[t0 + here])
                below = [j for j in below if drafts[t0 + j] == z]
                if not below:
                    break
                path.append(below[0])
                continue
            q, took = s["probs"][t0 + here].double(), None
            for j in below:
                d = drafts[t0 + j]
                if (float(p[d]) > 0.5) if T <= 0 else (u[t0 + j] * float(q[d]) < float(p[d])):
                    took = j
                    break
                if T > 0:  # what is left of the target's, as a distribution again
                    p = torch.relu(p - q)
                    p = p / p.sum()
            if took is None:
                z = _exact_pick(p, u[t0])
                break
            path.append(took)
        paths.append(path)
        nexts.append(z)
        t0 += len(up)
    return {"path": _i32([p + [-1] * (c["depth"] + 1 - len(p)) for p in paths]), "kept": _i32([len(p) for p in paths]),
            "next": _i32(nexts)}


def _exact_keep(c, s, trees, lens):
    G = c["dim"] // GROUP
    out, rows, P = [], [], c["page"]
    for b, (path, up, L) in enumerate(zip(_paths(c), trees, lens)):
        ids, first = s["table"][b].tolist(), L - len(up)
        rows += [(ids[(first + x) // P], (first + x) % P, ids[(first + i) // P], (first + i) % P) for i, x in enumerate(path)]
    a, ra, z, rz = torch.tensor(rows, device=DEV).T
    for pool in s["all"]:
        new = pool.clone()
        parts = [(0, c["dim"] * 2)] if not c["q4"] else [(0, 2 * G), (2 * G * P, c["dim"] // 2)]
        for at, n in parts:
            x = pool[..., at:at + P * n].unflatten(2, (P, n))[a, :, ra]
            new[..., at:at + P * n].unflatten(2, (P, n))[z, :, rz] = x
        out.append(new)
    out = torch.stack(out)
    return {"lens": _i32([L - len(up) + len(p) for L, up, p in zip(lens, trees, _paths(c))]),
            "pools": out if c["q4"] else out.view(torch.float16)}


def exact(c, seed):
    global own
    before, own = own, False
    try:
        s = prepare(c, seed)
    finally:
        own = before
    trees, lens = _trees(c, seed if c["kind"] == "layout" else None)
    if c["kind"] == "append":
        return _exact_append(c, s, trees, lens)
    if c["kind"] == "attn":
        return _exact_attn(c, s, trees, lens)
    if c["kind"] == "verify":
        return _exact_verify(c, s, trees)
    if c["kind"] == "keep":
        return _exact_keep(c, s, trees, lens)
    deep, masks = [], []
    for up in trees:
        for m in _ancestors(up):
            deep.append(bin(m).count("1") - 1)
            masks.append([_signed(m >> (64 * w) & ((1 << 64) - 1)) for w in range(_words(c))])
    pad = c.get("pad", 0)
    return {"depths": _i32(deep + [0] * pad),
            "masks": torch.tensor(masks + [[0] * _words(c)] * pad, dtype=torch.int64, device=DEV)}
