"""The operators around a batch's paged KV cache and its logits, as calls to be
timed: appending to the cache, attention over it, log probabilities.

Four kinds of pass, each through the public entry points:

  append    Kernels.kv_append_paged: the new tokens' queries and keys normed
            per head and rotated, keys and values written into their pages
  attn      Kernels.attn_paged: queries of one or many tokens a sequence over
            the pages of its context, causal
  step      both, one behind the other, as a model's layer calls them
  logprobs  Kernels.logprobs: log probability of a given token, entropy and
            the top alternatives of each row of logits

Pages hold `page` rows of one KV head, in fp16 or in the repository's q4
regions (groups of 32 columns, f16 scales, then nibbles holding q + 8).
Attention shapes are those of the repository's tests and bench (32 or 64 heads
on 4 KV heads of 128) and generic ones; the vocabulary is the bench's."""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
EPS, THETA = 1e-6, 1e6
GROUP = 32                      # columns of a q4 scale
S_MIN, S_MAX = 2.0 ** -17, 896.0  # what a q4 page's scales may be


def listed():
    big = dict(heads=32, kv=4, dim=128)
    wide = dict(heads=64, kv=4, dim=128)
    return [
        # one conversation's next token: the latency of a launch
        dict(name="append_b1", kind="append", q4=True, seqs=1, new=1, past=1500, page=64, **big),
        # a serving batch's next tokens, long and short contexts
        dict(name="append_b64", kind="append", q4=False, seqs=64, new=1, past=4000, page=16, **wide),
        # prompts arriving together, 2048 tokens or so in chunks of odd sizes
        dict(name="append_prompts", kind="append", q4=True, seqs=5, new=640, past=900, page=32, **big),
        # one conversation's next token over its context
        dict(name="attn_b1", kind="attn", q4=False, seqs=1, new=1, past=1500, page=64, **big),
        # a serving batch over a 4-bit cache, contexts up to 8192
        dict(name="attn_b32_q4", kind="attn", q4=True, seqs=32, new=1, past=8191, page=64, **big),
        # a larger batch over an fp16 cache in small pages
        dict(name="attn_b64", kind="attn", q4=False, seqs=64, new=1, past=4000, page=16, **big),
        # several guessed tokens a sequence, checked in one pass
        dict(name="attn_guess", kind="attn", q4=True, seqs=12, new=5, past=6000, page=128, **wide),
        # a prompt's chunk of 2048 tokens behind 6000 others
        dict(name="attn_chunk", kind="attn", q4=False, seqs=1, new=2048, past=6001, page=64, **big),
        # short prompts of ragged lengths, nothing before them, then a layer's append too
        dict(name="step_prompts", kind="step", q4=True, seqs=6, new=700, past=0, page=32, **big),
        # the next token's logits of one conversation
        dict(name="logprobs_b1", kind="logprobs", rows=1, vocab=151936, top=5),
        # a serving batch with the most alternatives an API offers
        dict(name="logprobs_b32", kind="logprobs", rows=32, vocab=151936, top=20),
        # scoring a text: no alternatives
        dict(name="logprobs_score", kind="logprobs", rows=777, vocab=151936, top=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


SHAPES = [(32, 4, 128), (32, 4, 128), (64, 4, 128), (32, 8, 128), (16, 2, 128), (8, 8, 64), (24, 8, 64), (12, 4, 64),
          (5, 1, 128), (16, 1, 64)]


def draw(rng):
    kind = rng.choice(["append"] * 3 + ["attn"] * 6 + ["step"] * 3 + ["logprobs"] * 3)
    if kind == "logprobs":
        vocab = _log(rng, 1000, 200000)
        return dict(kind=kind, rows=_log(rng, 1, max(2, min(1500, int(1.1e8 / vocab)))), vocab=vocab,
                    top=rng.choice([0, 1, 5, 10, 20, 64]))
    heads, kv, dim = rng.choice(SHAPES)
    c = dict(kind=kind, q4=rng.random() < 0.6, heads=heads, kv=kv, dim=dim, page=rng.choice([16, 32, 64, 128, 256]))
    form = rng.choice(["token", "token", "guess", "prompt", "chunk"])
    if form == "token":
        return dict(c, seqs=_log(rng, 1, 64), new=1, past=_log(rng, 1, 4000), pad=rng.choice([0, 0, 3]))
    if form == "guess":
        return dict(c, seqs=_log(rng, 1, 16), new=rng.randint(2, 8), past=_log(rng, 16, 6000), pad=rng.choice([0, 5]))
    if form == "prompt":
        return dict(c, seqs=rng.randint(1, 6), new=_log(rng, 17, 700), past=rng.choice([0, 0, _log(rng, 1, 1000)]), pad=0)
    return dict(c, seqs=rng.randint(1, 2), new=_log(rng, 64, 1000), past=_log(rng, 400, 2900), pad=rng.choice([0, 0, 7]))


def _lens(c):
    """(new tokens, context length with them) of each sequence, from the case
    alone: the first sequence is the longest, the others ragged."""
    r = random.Random("%d %d %d" % (c["seqs"], c["new"], c["past"]))
    new, lens = [], []
    for b in range(c["seqs"]):
        n = c["new"] if b == 0 or c["new"] == 1 else max(1, int(c["new"] * r.uniform(0.3, 1.0)))
        p = c["past"] if b == 0 else int(c["past"] * r.uniform(0.2, 1.0))
        new.append(n)
        lens.append(p + n)
    return new, lens


def _row_bytes(c):
    return c["dim"] // 2 + c["dim"] // GROUP * 2 if c["q4"] else 2 * c["dim"]


def work(c):
    if c["kind"] == "logprobs":
        n = c["rows"] * c["vocab"]
        return {"bytes": 4 * n + c["rows"] * (12 + 8 * c["top"]), "flops": 6 * n}
    new, lens = _lens(c)
    T, H, kv, D = sum(new), c["heads"], c["kv"], c["dim"]
    nbytes = flops = 0
    if c["kind"] in ("append", "step"):
        nbytes += T * (2 * H + 2 * kv) * D * 4 + 2 * T * kv * _row_bytes(c)
        nbytes += 2 * T * kv * D * 4 if c["q4"] else 0  # the values as held
        flops += T * (H + kv) * D * 8 + T * kv * D * 4
    if c["kind"] in ("attn", "step"):
        nbytes += 2 * T * H * D * 4 + 2 * sum(lens) * kv * _row_bytes(c)
        pairs = sum(n * (s - n) + n * (n + 1) // 2 for n, s in zip(new, lens))
        flops += 4 * D * H * pairs
    return {"bytes": nbytes, "flops": flops}


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
    """Filled pages, bytes [pages, kv, page bytes]: rows of normal values with
    a part in common."""
    kv, P, D = c["kv"], c["page"], c["dim"]
    out = torch.empty(pages, kv, P * _row_bytes(c), dtype=torch.uint8, device=DEV)
    common = torch.randn(kv, 1, D, generator=g, device=DEV) * 0.4
    at = 0
    while at < pages:
        n = min(pages - at, max(1, (1 << 24) // (kv * P * D)))
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


def prepare(c, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 2654435761 % (1 << 62) + 1)
    s = dict(c=c)
    if c["kind"] == "logprobs":
        R, V = c["rows"], c["vocab"]
        # most rows are undecided between a few tokens, some are sure of one;
        # values on a coarse grid, as a bf16 head gives them, so some are equal
        x = torch.randn(R, V, generator=g, device=DEV) * 2.0
        x += 4.0 * (torch.rand(R, V, generator=g, device=DEV) > 0.9995)
        x[::3, V // 3] += 18.0
        s["logits"] = x.to(torch.bfloat16).float()
        s["targets"] = torch.randint(0, V, (R,), generator=g, device=DEV, dtype=torch.int32)
        s["targets"][::2] = s["logits"][::2].argmax(1).to(torch.int32)
        s["logp"], s["entropy"] = (torch.zeros(R, device=DEV) for _ in range(2))
        s["ids"] = torch.zeros(R, c["top"], dtype=torch.int32, device=DEV)
        s["top"] = torch.zeros(R, c["top"], device=DEV)
        if own:
            _, K = _cuda()
            s["K"] = K
            s["ws"] = torch.empty(max(256, K.logprobs_ws_bytes(R, V, c["top"])), dtype=torch.uint8, device=DEV)
        return s
    H, kv, D, P = c["heads"], c["kv"], c["dim"], c["page"]
    new, lens = _lens(c)
    T = sum(new) + c.get("pad", 0)
    need = [-(-n // P) for n in lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    cols = max(need) + 1
    at = torch.tensor([0] + need[:-1]).cumsum(0)[:, None] + torch.arange(cols)
    table = order[at.clamp(max=pages - 1).to(DEV)]
    table[torch.arange(cols, device=DEV) >= _i32(need)[:, None]] = -1
    s.update(lens=_i32(lens), starts=_i32([0] + new).cumsum(0).to(torch.int32), table=table.contiguous(),
             tokens=T, max_q=max(new), max_seq=max(lens), kpool=_pool(g, c, pages), vpool=_pool(g, c, pages))
    # a projection's output: queries, keys and values of a token side by side
    s["qkv"] = torch.randn(T, (H + 2 * kv) * D, generator=g, device=DEV)
    s["qn"], s["kn"] = (0.8 + torch.rand(D, generator=g, device=DEV) for _ in range(2))
    s["freq"] = (THETA ** (-torch.arange(0, D, 2, device=DEV, dtype=torch.float64) / D)).float()
    s["q"] = torch.randn(T, H * D, generator=g, device=DEV) * 1.5 if c["kind"] == "attn" else torch.zeros(T, H * D, device=DEV)
    s["kout"], s["vout"] = (torch.zeros(T, kv * D, device=DEV) for _ in range(2))
    s["out"] = torch.zeros(T, H * D, device=DEV)
    if own:
        import llmpager_amd as lp

        cuda, K = _cuda()
        s["K"] = K
        s["cache"] = lp.KvCache(k_pages=s["kpool"].data_ptr(), v_pages=s["vpool"].data_ptr(), table=s["table"].data_ptr(),
                                pages=pages, page_rows=P, max_pages=cols, kv_heads=kv, head_dim=D,
                                format=lp.KV_Q4 if c["q4"] else lp.KV_F16)
        n = K.attn_paged_ws_bytes(s["cache"], H, c["seqs"], T, s["max_q"], s["max_seq"])
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


def _own_append(s):
    c, D = s["c"], s["c"]["dim"]
    H, kv = c["heads"], c["kv"]
    W, at = (H + 2 * kv) * D, s["qkv"].data_ptr()
    s["K"].kv_append_paged(s["cache"], at, W, at + H * D * 4, W, at + (H + kv) * D * 4, W, s["qn"].data_ptr(),
                           s["kn"].data_ptr(), EPS, s["freq"].data_ptr(), 1.0, s["q"].data_ptr(), H * D,
                           s["kout"].data_ptr() if c["q4"] else 0, s["vout"].data_ptr() if c["q4"] else 0, H,
                           s["starts"].data_ptr(), s["lens"].data_ptr(), c["seqs"], s["tokens"])


def _own_attn(s):
    c = s["c"]
    W = c["heads"] * c["dim"]
    s["K"].attn_paged(s["cache"], s["q"].data_ptr(), W, s["out"].data_ptr(), W, c["heads"], s["starts"].data_ptr(),
                      s["lens"].data_ptr(), c["seqs"], s["tokens"], s["max_q"], s["max_seq"], 1.0 / math.sqrt(c["dim"]),
                      s["ws"].data_ptr(), ws_bytes=s["ws"].numel())


def _own_logprobs(s):
    c = s["c"]
    s["K"].logprobs(s["logits"].data_ptr(), c["vocab"], c["rows"], c["vocab"], s["targets"].data_ptr(),
                    s["logp"].data_ptr(), s["entropy"].data_ptr(), c["top"], s["ids"].data_ptr(), s["top"].data_ptr(),
                    s["ws"].data_ptr(), ws_bytes=s["ws"].numel())


# ---- plain forms ------------------------------------------------------------------


def _places(s):
    """Each token's sequence and position; which rows belong to one."""
    t = torch.arange(s["tokens"], device=DEV)
    starts = s["starts"].long()
    b = (starts[None, 1:] <= t[:, None]).sum(1)
    live = b < len(s["lens"])
    b = b.clamp(max=len(s["lens"]) - 1)
    return live, b, s["lens"].long()[b] - (starts[b + 1] - t)


def _plain_append(s):
    c = s["c"]
    H, kv, D, P = c["heads"], c["kv"], c["dim"], c["page"]
    live, b, pos = _places(s)
    # 64 bits: angles of far positions, and 4-bit values next to a border
    x = s["qkv"].double()
    q, k, v = (y.unflatten(1, (-1, D)) for y in x.split([H * D, kv * D, kv * D], 1))
    ang = pos.double()[:, None, None] * s["freq"].double()
    cs, sn = ang.cos(), ang.sin()

    def turned(y, w):
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * w.double()
        a, z = y[..., :D // 2], y[..., D // 2:]
        return torch.cat((a * cs - z * sn, a * sn + z * cs), -1)

    s["q"][live] = turned(q, s["qn"]).flatten(1).float()[live]
    k = turned(k, s["kn"])[live]
    v = v[live]
    page, row = s["table"][b, pos.clamp(min=0) // P].long()[live], (pos % P)[live]
    for new, pool, out in ((k, s["kpool"], s["kout"]), (v, s["vpool"], s["vout"])):
        if c["q4"]:
            G = D // GROUP
            codes, scales = _quantise(new)
            pool.view(torch.float16)[..., :P * G].unflatten(2, (P, G))[page, :, row] = scales
            pool[..., 2 * P * G:].unflatten(2, (P, D // 2))[page, :, row] = codes[..., 0::2] | (codes[..., 1::2] << 4)
            out[live] = ((codes.float() - 8.0).unflatten(2, (G, GROUP)) * scales.float()[..., None]).flatten(1)
        else:
            pool.view(torch.float16).unflatten(2, (P, D))[page, :, row] = new.to(torch.float16)


def _rows(s, pool, n, dtype):
    """Rows 0 .. n - 1 of every sequence as [seqs, kv, n, D]; rows past a
    sequence's end are zero."""
    c = s["c"]
    kv, D, P = c["kv"], c["dim"], c["page"]
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
    live = i < (starts[1:] - starts[:-1])[:, None]
    t = (starts[:-1, None] + i).clamp(max=s["tokens"] - 1)
    q = s["q"][t].view(B, Q, kv, G, D).permute(0, 2, 1, 3, 4).reshape(B, kv, Q * G, D)
    k, v = _rows(s, s["kpool"], N, torch.float32), _rows(s, s["vpool"], N, torch.float32)
    x = q @ k.transpose(2, 3).contiguous() * (1.0 / math.sqrt(D))
    last = (lens - (starts[1:] - starts[:-1]))[:, None] + i                     # [B, Q]: the row of its own token
    seen = torch.arange(N, device=DEV) <= last.repeat_interleave(G, 1)[:, None, :, None]
    x = torch.where(seen, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.where(seen, torch.exp(x - top), 0)
    norm = p.sum(-1, keepdim=True)
    y = torch.where(norm > 0, p @ v / norm, 0)
    y = y.view(B, kv, Q, G, D).permute(0, 2, 1, 3, 4).reshape(B, Q, H * D)
    s["out"][t[live]] = y[live]


def _plain_logprobs(s):
    c, x = s["c"], s["logits"]
    # 64 bits for the sums: a sure row's entropy is all in the small terms
    y = x.double() - x.amax(1, keepdim=True)
    e = torch.exp(y)
    n = e.sum(1)
    lse = torch.log(n)
    s["logp"] = (y.gather(1, s["targets"].long()[:, None])[:, 0] - lse).float()
    s["entropy"] = (lse - (e * y).sum(1) / n).float()
    if c["top"]:
        # the order of (value, lowest index first) as one whole number
        bits = x.view(torch.int32).long()
        key = torch.where(bits < 0, -(bits & 0x7fffffff), bits) * (1 << 20) - torch.arange(c["vocab"], device=DEV)
        at = key.topk(c["top"], 1).indices
        s["ids"] = at.to(torch.int32)
        s["top"] = (y.gather(1, at) - lse[:, None]).float()


def run(s):
    kind = s["c"]["kind"]
    if kind == "logprobs":
        if own:
            _own_logprobs(s)
        else:
            _plain_logprobs(s)
        return {"logp": s["logp"], "entropy": s["entropy"], "ids": s["ids"], "top": s["top"]}
    out = {}
    if kind in ("append", "step"):
        if own:
            _own_append(s)
        else:
            _plain_append(s)
        out["q"] = s["q"]
        if s["c"]["q4"]:  # the values that the 4-bit rows stand for
            out.update(k=s["kout"], v=s["vout"])
        else:
            out.update(kpages=s["kpool"].view(torch.float16), vpages=s["vpool"].view(torch.float16))
    if kind in ("attn", "step"):
        if own:
            _own_attn(s)
        else:
            _plain_attn(s)
        out["out"] = s["out"]
    return out


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


def _exact_row(c, raw):
    """One page's rows [kv, page, D] from its bytes [kv, page bytes]."""
    kv, P, D = c["kv"], c["page"], c["dim"]
    if not c["q4"]:
        return raw.contiguous().view(torch.float16).double().view(kv, P, D)
    n = P * (D // GROUP) * 2
    sc = raw[:, :n].contiguous().view(torch.float16).double().view(kv, P, D // GROUP, 1)
    lo, hi = (raw[:, n:] % 16).double() - 8, torch.div(raw[:, n:], 16, rounding_mode="floor").double() - 8
    return (torch.stack((lo, hi), 2).view(kv, P, D // GROUP, GROUP) * sc).view(kv, P, D)


def exact(c, seed):
    global own
    before, own = own, False
    try:
        s = prepare(c, seed)
    finally:
        own = before
    if c["kind"] == "logprobs":
        x = s["logits"].double()
        logp, ent, ids, top = [], [], [], []
        for r in range(c["rows"]):
            p = torch.log_softmax(x[r], 0)
            logp.append(p[int(s["targets"][r])])
            ent.append(-(p.exp() * p).sum())
            at = torch.sort(x[r], descending=True, stable=True).indices[:c["top"]]
            ids.append(at)
            top.append(p[at])
        return {"logp": torch.stack(logp), "entropy": torch.stack(ent), "ids": torch.stack(ids).to(torch.int32),
                "top": torch.stack(top)}
    new, lens = _lens(c)
    H, kv, D, P, G = c["heads"], c["kv"], c["dim"], c["page"], c["heads"] // c["kv"]
    T = s["tokens"]
    Q, O = s["q"].double(), torch.zeros(T, H * D, dtype=torch.float64, device=DEV)
    KO, VO = (torch.zeros(T, kv * D, dtype=torch.float64, device=DEV) for _ in range(2))
    freq, qn, kn = s["freq"].double(), s["qn"].double(), s["kn"].double()
    pages = {n: s[n].clone() for n in ("kpool", "vpool")}
    held = {n: s[n].view(torch.float16).double().unflatten(2, (P, D)) for n in pages} if not c["q4"] else {}
    t = 0
    for b, (n, L) in enumerate(zip(new, lens)):
        ids = s["table"][b, :-(-L // P)].tolist()
        ctx = {m: torch.cat([_exact_row(c, pages[m][i]) for i in ids], 1)[:, :L] for m in pages}
        if c["kind"] != "attn":
            for i in range(H + kv):
                x = s["qkv"][t:t + n, i * D:(i + 1) * D].double()
                pos = torch.arange(L - n, L, dtype=torch.float64, device=DEV)[:, None]
                y = _exact_turn(x, qn if i < H else kn, pos, freq)
                if i < H:
                    Q[t:t + n, i * D:(i + 1) * D] = y
                    continue
                v = s["qkv"][t:t + n, (i + kv) * D:(i + kv + 1) * D].double()
                at = torch.arange(L - n, L, device=DEV)
                page = torch.tensor(ids, device=DEV)[at // P]
                for m, z, store in (("kpool", y, KO), ("vpool", v, VO)):
                    if c["q4"]:
                        z = _exact_q4(z)
                        store[t:t + n, (i - H) * D:(i - H + 1) * D] = z
                        ctx[m][i - H, L - n:] = z
                    else:
                        held[m][page, i - H, at % P] = z
                        ctx[m][i - H, L - n:] = z.to(torch.float16).double()
        if c["kind"] != "append":
            q = (Q if c["kind"] == "attn" else Q.float().double())[t:t + n].view(n, kv, G, D)
            seen = torch.arange(L, device=DEV)[None, :] <= torch.arange(L - n, L, device=DEV)[:, None]
            for h in range(H):
                a = q[:, h // G, h % G] @ ctx["kpool"][h // G].T / math.sqrt(D)
                a = torch.softmax(a.masked_fill(~seen, -math.inf), 1)
                O[t:t + n, h * D:(h + 1) * D] = a @ ctx["vpool"][h // G]
        t += n
    out = {}
    if c["kind"] != "attn":
        out["q"] = Q
        out.update(dict(k=KO, v=VO) if c["q4"] else {n[0] + "pages": x.flatten(2) for n, x in held.items()})
    if c["kind"] != "append":
        out["out"] = O
    return out
