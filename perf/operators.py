"""The operators of a paged KV cache, as cases that can be timed and checked.

A pool holds the K (or V) rows of one attention layer for all sequences in pages
of `page` positions; `pages[b]` lists sequence b's pages in order. Five operators,
each through the framework's public entry points where `own` is true:

* "write": the rows of several sequences' new tokens into their pages, fp16 or
  quantised to the int8 format (32 dims share an fp16 scale), and their reading
  back, as a program does that hands a prompt's rows on (`paged_kv_store`,
  `paged_kv_load`).
* "read": whole cached contexts read back as dense fp16 rows (`paged_kv_load`).
* "prep": per-head RMSNorm of q and k, partial RoPE at each token's own
  position, and the store of k and v (`attn_prep_paged`).
* "chunk": causal attention of chunks of new tokens, several sequences packed
  behind each other, over the pages (`attention_prefill_paged`). `spans` lists
  the sequences as tokens@position.
* "decode": one to four tokens a sequence over the pages (`attn_decode_paged`).

A query at position p sees the rows r <= p with r > p - window or r < sinks, all
of them at window 0; its output passes the sigmoid output gate, the second half
of each head's q row. Where `own` is false the same is computed in elementary
torch operations in 32 bits.
"""
import math

import torch

own = False

HEADS, KV, DIM = 24, 4, 256
GROUP = HEADS // KV
ROPE, THETA, EPS = 64, 1e7, 1e-6
SCALE = DIM ** -0.5
F16, F32, F64, I32 = torch.float16, torch.float32, torch.float64, torch.int32


def listed():
    return [
        # a serving step's new rows, a token each of 48 sequences
        dict(name="write_48x1", kind="write", seqs=48, shortest=1, longest=1, pos=5000, page=64,
             kv8=False),
        # the chunks of a prefill batch, quantised as they are written
        dict(name="write_7_chunks_kv8", kind="write", seqs=7, shortest=33, longest=8192, pos=1001,
             page=16, kv8=True),
        # a short conversation's rows handed to another worker
        dict(name="read_1x777_kv8", kind="read", seqs=1, shortest=777, longest=777, pos=0, page=32,
             kv8=True),
        # the contexts of a batch moved off the card, fp16
        dict(name="read_5_contexts", kind="read", seqs=5, shortest=2500, longest=65536, pos=0,
             page=128, kv8=False),
        # a decode batch's q, k and v rows, far into their sequences
        dict(name="prep_32x1_far", kind="prep", seqs=32, shortest=1, longest=1, pos=98765, page=64,
             kv8=False),
        # a prefill batch's
        dict(name="prep_3_chunks", kind="prep", seqs=3, shortest=515, longest=4096, pos=777, page=16,
             kv8=False),
        # a fresh 8k prompt in one call
        dict(name="chunk_8k", kind="chunk", spans="8192@0", page=64, window=0, sinks=0, kv8=False),
        # the most products, a prefill batch as a scheduler mixes it over the int8 cache: sub-chunks of long
        # prompts, a follow-up message, short prompts and one sequence's single token
        dict(name="chunk_mixed_kv8", kind="chunk",
             spans="1024@30000 777@3001 130@0 515@12345 37@60000 1@9000", page=16, window=0, sinks=0,
             kv8=True),
        # sub-chunks of endless sessions: a window of 4096 rows and 4 first tokens kept
        dict(name="chunk_window_4x1k", kind="chunk", spans="1024@98000 1024@50001 1000@20000 1024@2000",
             page=128, window=4096, sinks=4, kv8=False),
        # the smallest call: one user's next token in a short chat
        dict(name="decode_1x500", kind="decode", seqs=1, shortest=500, longest=500, rows=1, page=16,
             window=0, sinks=0, kv8=False),
        # a full serving batch of unlike contexts over the int8 cache
        dict(name="decode_64_ragged_kv8", kind="decode", seqs=64, shortest=100, longest=32768, rows=1,
             page=64, window=0, sinks=0, kv8=True),
        # speculative rounds over long documents, fp16 cache: the most bytes
        dict(name="verify_6x100k", kind="decode", seqs=6, shortest=90000, longest=100000, rows=3,
             page=256, window=0, sinks=0, kv8=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["chunk", "chunk", "decode", "decode", "write", "read", "prep"])
    page = rng.choice([16, 32, 64, 128, 256])
    kv8 = rng.random() < 0.5
    if kind in ("write", "read", "prep"):
        top = {"write": 8192, "read": 65536, "prep": 4096}[kind]
        longest = _log(rng, 1, top)
        seqs = rng.randint(1, max(1, min(48, 2 * top // longest)))
        return dict(kind=kind, seqs=seqs, shortest=_log(rng, 1, longest), longest=longest,
                    pos=0 if kind == "read" else _log(rng, 1, 100000) - 1, page=page,
                    kv8=kv8 and kind != "prep")
    window, sinks = (_log(rng, 50, 16000), rng.choice([0, 1, 4, 100])) if rng.random() < 0.4 else (0, 0)
    if kind == "decode":
        seqs = _log(rng, 1, 96)
        longest = _log(rng, 1, min(100000, 600000 // seqs))
        return dict(kind=kind, seqs=seqs, shortest=_log(rng, 1, longest), longest=longest,
                    rows=rng.choice([1, 1, 1, 2, 3, 4]), page=page, window=window, sinks=sinks, kv8=kv8)
    # no more (query, row) pairs than a fresh 8k prompt's
    seqs, spans, pairs = rng.randint(1, 7), [], 3.3e7
    for i in range(seqs):
        share = pairs / (seqs - i)
        n = _log(rng, 1, max(1.0, min(8000.0, math.sqrt(2 * share) - 1)))
        deepest = int(min(60000, share / n - n / 2))
        p = _log(rng, 1, deepest + 1) - 1 if deepest > 0 else 0
        pairs -= n * (p + n / 2)
        spans.append(f"{n}@{p}")
    return dict(kind=kind, spans=" ".join(spans), page=page, window=window, sinks=sinks, kv8=kv8)


def _spans(case):
    """(tokens, position of the first) of every sequence: the chunk's as listed, else
    lengths spread geometrically from the shortest to the longest, not in order."""
    if case["kind"] == "chunk":
        return [tuple(int(x) for x in s.split("@")) for s in case["spans"].split()]
    n, lo, hi = case["seqs"], case["shortest"], case["longest"]
    lens = [int(round(lo * (hi / lo) ** (i / max(1, n - 1)))) for i in range(n)]
    if n == 1:
        lens = [hi]
    step = next(s for s in (5, 7, 11, 1) if math.gcd(s, n) == 1)
    lens = [lens[i * step % n] for i in range(n)]
    if case["kind"] == "decode":     # lens: the cached rows, the tokens' own among them
        return [(case["rows"], max(0, x - case["rows"])) for x in lens]
    return [(x, case["pos"] + (13 * i if case["pos"] else 0)) for i, x in enumerate(lens)]


# ---------------------------------------------------------------------------
# inputs, from the seed alone
# ---------------------------------------------------------------------------

def _randn(g, *shape, scale=1.0, dtype=F16):
    x = torch.empty(shape, dtype=F32, device="cuda").normal_(0.0, scale, generator=g)
    return x if dtype == F32 else x.to(dtype)


def _pool(g, rows, kv8, empty):
    """A pool of `rows` cached rows of KV heads: fp16 values or the int8 format
    (values [rows, KV, DIM] int8, then scales [rows, KV, DIM / 32] fp16, flat)."""
    if not kv8:
        return torch.zeros((rows, KV, DIM), dtype=F16, device="cuda") if empty else \
            _randn(g, rows, KV, DIM)
    vals, scales = rows * KV * DIM, rows * KV * (DIM // 32)
    pool = torch.zeros(vals + 2 * scales, dtype=torch.int8, device="cuda")
    if not empty:
        pool[:vals].random_(-127, 128, generator=g)
        pool[vals:] = (_randn(g, scales, dtype=F32).abs() * 0.005 + 0.012).half().view(torch.int8)
    return pool


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)
    kind, page, kv8 = case["kind"], case["page"], case["kv8"]
    spans = _spans(case)
    B, N = len(spans), sum(n for n, _ in spans)
    # the pages that a sequence has, in the order that a long-running pool hands them out
    count = [(p + n + page - 1) // page for n, p in spans]
    first = [p // page if kind in ("write", "prep") else 0 for _, p in spans]
    held = sum(c - f for c, f in zip(count, first))
    n_pages = held + 3
    order = torch.randperm(n_pages, generator=g, device="cuda").to(I32)
    pages = torch.full((B, max(count)), -1, dtype=I32, device="cuda")
    at = 0
    for b in range(B):
        # (what a write does not reach of a sequence's pages stays absent)
        pages[b, first[b]:count[b]] = order[at:at + count[b] - first[b]]
        at += count[b] - first[b]
    starts = [0]
    for n, _ in spans:
        starts.append(starts[-1] + n)
    s = dict(kind=kind, page=page, kv8=kv8, spans=spans, N=N, rows=n_pages * page, pages=pages,
             window=case.get("window", 0), sinks=case.get("sinks", 0),
             starts=torch.tensor(starts, dtype=I32, device="cuda"),
             pos0=torch.tensor([p for _, p in spans], dtype=I32, device="cuda"),
             Ts=[n for n, _ in spans], pos0s=[p for _, p in spans])
    empty = kind in ("write", "prep")
    for name in ("kpool", "vpool"):
        pool = _pool(g, s["rows"], kv8, empty)
        s[name] = pool if kv8 else pool.view(n_pages, page, KV, DIM)
    if kind in ("write", "prep"):
        s["k"], s["v"] = _randn(g, N, KV, DIM), _randn(g, N, KV, DIM)
    if kind == "prep":
        s["wq"], s["wk"] = (_randn(g, DIM, scale=0.1, dtype=F32) for _ in range(2))
        s["qg"] = _randn(g, N, HEADS, 2 * DIM)
        s["q_out"] = torch.empty((N, HEADS, DIM), dtype=F16, device="cuda")
    if kind == "chunk":
        s["qg"] = _randn(g, N, HEADS, 2 * DIM)
    if kind == "decode":
        s["qg"] = _randn(g, B, case["rows"], HEADS, 2 * DIM)
    return s


# ---------------------------------------------------------------------------
# the plain forms: elementary operations in 32 bits
# ---------------------------------------------------------------------------

def _at(s, b, lo, n):
    """The pool rows of sequence b's positions lo .. lo + n - 1."""
    p = torch.arange(lo, lo + n, device="cuda")
    return s["pages"][b].long()[p // s["page"]] * s["page"] + p % s["page"]


def _halves(s, pool):
    cut = s["rows"] * KV * DIM
    return pool[:cut].view(s["rows"], KV, DIM), pool[cut:].view(F16).view(s["rows"], KV, DIM // 32)


def _fetch(s, name, rows):
    """Cached rows in 32 bits."""
    if not s["kv8"]:
        return s[name].view(s["rows"], KV, DIM)[rows].float()
    values, scales = _halves(s, s[name])
    return values[rows].float() * scales[rows].float().repeat_interleave(32, -1)


def _put(s, name, rows, x):
    if not s["kv8"]:
        s[name].view(s["rows"], KV, DIM)[rows] = x
        return
    values, scales = _halves(s, s[name])
    blocks = x.float().view(-1, KV, DIM // 32, 32)
    scale = (blocks.abs().amax(-1) / 127.0).half()
    wide = scale.float()[..., None]
    q = torch.where(wide > 0, torch.round(blocks / wide).clamp(-127, 127), torch.zeros_like(blocks))
    values[rows] = q.to(torch.int8).view(-1, KV, DIM)
    scales[rows] = scale


def _all_rows(s):
    return torch.cat([_at(s, b, p, n) for b, (n, p) in enumerate(s["spans"])])


def _read(s):
    rows = _all_rows(s)
    return _fetch(s, "kpool", rows).half(), _fetch(s, "vpool", rows).half()


def _norm(x, w):
    x = x.float()
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * (1.0 + w)


def _rotate(x, pos):
    half = ROPE // 2
    freq = THETA ** (-2.0 * torch.arange(half, dtype=F64, device="cuda") / ROPE)
    angle = pos.double()[:, None] * freq
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    a, b = x[..., :half], x[..., half:ROPE]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., ROPE:]], -1)


def _prep(s):
    pos = torch.cat([torch.arange(p, p + n, device="cuda") for n, p in s["spans"]])
    rows = _all_rows(s)
    q = _rotate(_norm(s["qg"][..., :DIM], s["wq"]), pos).half()
    _put(s, "kpool", rows, _rotate(_norm(s["k"], s["wk"]), pos).half())
    _put(s, "vpool", rows, s["v"])
    return q, s["kpool"], s["vpool"]


def _attend(s, b, qg, pos):
    """One sequence's queries at positions pos .. over its pages: qg [n, HEADS, 2 DIM]."""
    n = qg.shape[0]
    out = torch.empty((n, HEADS, DIM), dtype=F16, device="cuda")
    for lo in range(0, n, 1024):
        hi = min(n, lo + 1024)
        last = pos + hi                                     # rows in sight: [0, last)
        kv_rows = torch.arange(last, device="cuda")
        if s["window"]:
            kv_rows = kv_rows[(kv_rows > pos + lo - s["window"]) | (kv_rows < s["sinks"])]
        at = s["pages"][b].long()[kv_rows // s["page"]] * s["page"] + kv_rows % s["page"]
        k, v = _fetch(s, "kpool", at), _fetch(s, "vpool", at)
        p = torch.arange(pos + lo, last, device="cuda")[:, None]
        hidden = kv_rows[None] > p
        if s["window"]:
            hidden |= (kv_rows[None] <= p - s["window"]) & (kv_rows[None] >= s["sinks"])
        for h in range(KV):
            q = qg[lo:hi, h * GROUP:(h + 1) * GROUP, :DIM].float()
            scores = (q.reshape(-1, DIM) @ k[:, h].t()).view(hi - lo, GROUP, -1) * SCALE
            scores.masked_fill_(hidden[:, None], float("-inf"))
            e = (scores - scores.amax(-1, keepdim=True)).exp()
            z = (e.view((hi - lo) * GROUP, -1) @ v[:, h]).view(hi - lo, GROUP, DIM)
            z = z / e.sum(-1, keepdim=True)
            gate = qg[lo:hi, h * GROUP:(h + 1) * GROUP, DIM:].float()
            out[lo:hi, h * GROUP:(h + 1) * GROUP] = (z / (1.0 + (-gate).exp())).half()
    return out


def _plain(s):
    if s["kind"] == "write":
        rows = _all_rows(s)
        _put(s, "kpool", rows, s["k"])
        _put(s, "vpool", rows, s["v"])
        return _read(s)
    if s["kind"] == "read":
        return _read(s)
    if s["kind"] == "prep":
        return _prep(s)
    if s["kind"] == "decode":
        return torch.stack([_attend(s, b, s["qg"][b], p) for b, (_, p) in enumerate(s["spans"])])
    out, at = [], 0
    for b, (n, p) in enumerate(s["spans"]):
        out.append(_attend(s, b, s["qg"][at:at + n], p))
        at += n
    return torch.cat(out)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    s = state
    if not own:
        return _plain(s)
    from __graft_entry__ import load_package
    ops = load_package().ops
    pools, table = (s["kpool"], s["vpool"]), (s["pages"], s["starts"], s["pos0"])
    if s["kind"] == "write":
        ops.paged_kv_store(s["k"], s["v"], *pools, *table, page_size=s["page"])
    if s["kind"] in ("write", "read"):
        return ops.paged_kv_load(*pools, *table, T=s["N"], page_size=s["page"])
    if s["kind"] == "prep":
        ops.attn_prep_paged(s["qg"], s["k"], s["v"], s["wq"], s["wk"], *pools, *table,
                            page_size=s["page"], q_out=s["q_out"])
        return s["q_out"], *pools
    if s["kind"] == "chunk":
        return ops.attention_prefill_paged(s["qg"], *pools, s["pages"], s["Ts"], s["pos0s"],
                                           page_size=s["page"], window=s["window"], sinks=s["sinks"],
                                           gated=True)
    return ops.attn_decode_paged(s["qg"], *pools, s["pages"], s["pos0"], page_size=s["page"],
                                 window=s["window"], sinks=s["sinks"])


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def _seen(p, window, sinks):
    """Rows that a query at position p sees."""
    if window == 0 or p < window:
        return p + 1
    return window + min(sinks, p - window + 1)


def work(case):
    spans, row = _spans(case), 272 if case["kv8"] else 512     # bytes of a cached head row
    n = sum(t for t, _ in spans)
    dense, cached = 2 * n * KV * DIM * 2, 2 * n * KV * row
    if case["kind"] == "write":
        return {"bytes": 2 * (dense + cached), "flops": 3 * 2 * n * KV * DIM}
    if case["kind"] == "read":
        return {"bytes": dense + cached, "flops": 2 * n * KV * DIM}
    if case["kind"] == "prep":
        return {"bytes": 2 * n * HEADS * DIM * 2 + dense + cached + 2 * DIM * 4,
                "flops": 6 * n * (HEADS + KV) * DIM}
    window, sinks = case["window"], case["sinks"]
    pairs = sum(_seen(q, window, sinks) for t, p in spans for q in range(p, p + t))
    rows = 0
    for t, p in spans:
        lo = max(0, p - window + 1) if window else 0
        rows += p + t - lo + min(sinks, lo)
    return {"bytes": 3 * n * HEADS * DIM * 2 + 2 * rows * KV * row, "flops": 4 * pairs * HEADS * DIM}


# ---------------------------------------------------------------------------
# from the definition, in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    R, page = s["rows"], s["page"]

    def values(pool):
        if not s["kv8"]:
            return pool.reshape(R, KV * DIM)
        cut = R * KV * DIM
        return pool[:cut].reshape(R, KV * DIM), pool[cut:].view(F16).reshape(R, KV * DIM // 32)

    def cached(pool, index):
        got = values(pool)
        if not s["kv8"]:
            return got[index].double().unflatten(-1, (KV, DIM))
        blocks = got[0][index].double().unflatten(-1, (-1, 32))
        return (blocks * got[1][index].double().unsqueeze(-1)).flatten(1).unflatten(-1, (KV, DIM))

    def where(b, positions):
        return s["pages"][b].long().gather(0, positions.div(page, rounding_mode="floor")) * page \
            + positions.remainder(page)

    own_rows = [where(b, torch.arange(p, p + t, device="cuda")) for b, (t, p) in enumerate(s["spans"])]
    if s["kind"] == "read":
        index = torch.cat(own_rows)
        return cached(s["kpool"], index), cached(s["vpool"], index)
    if s["kind"] == "write":
        out = []
        for x in (s["k"].double(), s["v"].double()):
            if s["kv8"]:
                blocks = x.unflatten(-1, (-1, 32))
                step = (blocks.abs().max(-1, keepdim=True).values / 127).half().double()
                level = (blocks / step.clamp_min(1e-300)).round().clamp(-127, 127) * (step > 0)
                x = (level * step).flatten(-2)
            out.append(x)
        return tuple(out)
    if s["kind"] == "prep":
        def heads(x, w):
            x = x.double()
            x = x / (x.square().sum(-1, keepdim=True) / DIM + EPS).sqrt() * (w.double() + 1)
            y, at = x.clone(), 0
            for t, p in s["spans"]:
                for j in range(ROPE // 2):
                    a = torch.arange(p, p + t, dtype=F64, device="cuda") * math.pow(THETA, -2 * j / ROPE)
                    c, d = torch.cos(a)[:, None], torch.sin(a)[:, None]
                    u, v = x[at:at + t, :, j], x[at:at + t, :, j + ROPE // 2]
                    y[at:at + t, :, j], y[at:at + t, :, j + ROPE // 2] = u * c - v * d, v * c + u * d
                at += t
            return y
        out = []
        for pool, x in ((s["kpool"], heads(s["k"], s["wk"])), (s["vpool"], s["v"].double())):
            y = pool.double().reshape(R, KV, DIM)
            y[torch.cat(own_rows)] = x
            out.append(y.reshape(pool.shape))
        return heads(s["qg"][..., :DIM], s["wq"]), *out
    # attention, a query head and a block of queries at a time
    outs, at = [], 0
    qg_rows = s["qg"].reshape(-1, HEADS, 2 * DIM)
    for b, (t, p) in enumerate(s["spans"]):
        z = torch.zeros((t, HEADS, DIM), dtype=F64, device="cuda")
        for t0 in range(0, t, 512):
            t1 = min(t, t0 + 512)
            pos = torch.arange(p + t0, p + t1, device="cuda").unsqueeze(1)
            first = max(0, p + t0 - s["window"] + 1) if s["window"] else 0
            keys = torch.cat([torch.arange(min(s["sinks"], first), device="cuda"),
                              torch.arange(first, p + t1, device="cuda")])
            index = where(b, keys)
            K, V = cached(s["kpool"], index), cached(s["vpool"], index)
            ok = keys <= pos
            if s["window"]:
                ok &= (keys > pos - s["window"]) | (keys < s["sinks"])
            for head in range(HEADS):
                q = qg_rows[at + t0:at + t1, head, :DIM].double()
                a = torch.where(ok, q @ K[:, head // GROUP].T / math.sqrt(DIM), -math.inf)
                z[t0:t1, head] = torch.softmax(a, -1) @ V[:, head // GROUP]
        outs.append(z * torch.sigmoid(qg_rows[at:at + t, :, DIM:].double()))
        at += t
    z = torch.cat(outs)
    return z.reshape(s["qg"].shape[:-1] + (DIM,)) if s["kind"] == "decode" else z
