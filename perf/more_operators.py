"""A round of tree-drafted tokens over the paged cache, as cases that can be timed and checked.

A drafter proposes several continuations of a sequence as a tree of up to 64 tokens;
one forward pass verifies all of them, and the path that is accepted becomes part of the
sequence. Token i of a sequence has the parent parents[b, i] < i, -1 for a child of the
context, -2 for a place in a padded batch that holds no token; it lies in cache row
pos0[b] + i, at position pos0[b] + its depth. Operators, each through the framework's
public entry points where `own` is true:

* "axes": per-head RMSNorm of q and k, partial RoPE whose pairs take their position from
  one of several axes (time, height, width of images and video; a single axis: a tree's
  depths), and the store of k and v into pages (`attn_prep_axes`).
* "tree": attention of the tree's tokens over the pages: the context's rows, a token's
  ancestors and itself; the output passes the sigmoid output gate (`attn_tree_paged`).
* "gdn": a gated DeltaNet layer over the tree, every token from the state that its path
  leaves, with its causal conv along the path and the gated output norm
  (`gdn_tree_normed`).
* "commit": the recurrent state and the conv frames after the accepted path
  (`gdn_tree_commit`).
* "copy", "keep": the pages of a cache, all layers in one call: whole pages copied (forks,
  defragmentation; `paged_kv_copy`), the accepted path's rows moved up behind the context
  (`paged_kv_keep`).

Where `own` is false the same is computed in elementary torch operations in 32 bits.
"""
import math

import torch

own = False

HEADS, KV, DIM = 24, 4, 256                          # full attention
GROUP = HEADS // KV
ROPE, THETA, EPS = 64, 1e7, 1e-6
SCALE = DIM ** -0.5
KH, VH, KD, VD, WIDTH = 16, 48, 128, 128, 10240      # gated DeltaNet: q | k | v of WIDTH channels
SHARE = VH // KH
OUT_SCALE = KD ** -0.5
F16, F32, F64, I32 = torch.float16, torch.float32, torch.float64, torch.int32


def listed():
    return [
        # one user's tree in a short chat
        dict(name="tree_1x16_short", kind="tree", seqs=1, tokens=16, fewest=16, shortest=500, longest=500,
             page=16, window=0, sinks=0, kv8=False),
        # a serving batch of unlike contexts and trees over the int8 cache
        dict(name="tree_12x26_ragged_kv8", kind="tree", seqs=12, tokens=26, fewest=5, shortest=100,
             longest=32768, page=64, window=0, sinks=0, kv8=True),
        # the largest trees over long documents: the most products
        dict(name="tree_4x63_long", kind="tree", seqs=4, tokens=63, fewest=63, shortest=20000,
             longest=60000, page=128, window=0, sinks=0, kv8=False),
        # a batch of trees prepared at their depths
        dict(name="axes_12x26_tree", kind="axes", seqs=12, tokens=26, pos=5000, page=64, axes=1,
             interleaved=False),
        # a picture's patches and the text around it: time, height and width
        dict(name="axes_1x4097_picture", kind="axes", seqs=1, tokens=4097, pos=777, page=16, axes=3,
             interleaved=True),
        # one user's tree
        dict(name="gdn_1x16", kind="gdn", seqs=1, tokens=16, fewest=16, fresh=False),
        # a full batch of trees of unlike sizes
        dict(name="gdn_16x37_ragged", kind="gdn", seqs=16, tokens=37, fewest=9, fresh=False),
        # one user's accepted path
        dict(name="commit_1x4", kind="commit", seqs=1, tokens=16, accepted=4),
        # a full batch's, each of its own length
        dict(name="commit_16x7", kind="commit", seqs=16, tokens=37, accepted=7),
        # a fork's private copies of its last pages, int8, with their reading back
        dict(name="copy_3_pages_kv8", kind="copy", layers=1, pool=40, pages=3, page=64, kv8=True),
        # pages moved together in the pools of all layers
        dict(name="copy_150_pages", kind="copy", layers=16, pool=320, pages=150, page=32, kv8=False),
        # the accepted paths of a batch in the pools of all layers
        dict(name="keep_12x5", kind="keep", layers=16, seqs=12, tokens=26, accepted=5, pos=300, page=64,
             kv8=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "tree", "axes", "gdn", "gdn", "commit", "copy", "keep"])
    page = rng.choice([16, 32, 64, 128, 256])
    if kind == "axes":
        axes = rng.choice([1, 2, 3, 3, 4])
        tokens = _log(rng, 1, 4096)
        return dict(kind=kind, seqs=rng.randint(1, max(1, min(24, 4096 // tokens))), tokens=tokens,
                    pos=_log(rng, 1, 100000) - 1, page=page, axes=axes,
                    interleaved=axes > 1 and rng.random() < 0.5)
    if kind == "copy":
        layers, kv8 = rng.choice([1, 2, 5, 16]), rng.random() < 0.4
        if kv8:
            layers = 1
        pages = _log(rng, 1, max(2, 60000 // (layers * page)))
        return dict(kind=kind, layers=layers, pool=2 * pages + rng.randint(1, 40), pages=pages, page=page,
                    kv8=kv8)
    tokens = _log(rng, 1, 64)
    fewest = rng.randint(1, tokens)
    if kind == "gdn":
        return dict(kind=kind, seqs=rng.randint(1, max(1, min(16, 330 // tokens))), tokens=tokens,
                    fewest=fewest, fresh=rng.random() < 0.25)
    if kind == "commit":
        return dict(kind=kind, seqs=rng.randint(1, 16), tokens=tokens,
                    accepted=rng.randint(1, min(tokens, 12)))
    if kind == "keep":
        return dict(kind=kind, layers=rng.choice([1, 4, 16]), seqs=rng.randint(1, 32), tokens=tokens,
                    accepted=rng.randint(1, min(tokens, 12)), pos=_log(rng, 1, 600) - 1, page=page, kv8=False)
    seqs = _log(rng, 1, 48)
    longest = _log(rng, 1, min(100000, max(1, 9000000 // (tokens * seqs))))
    window, sinks = (_log(rng, 4, 16000), rng.choice([0, 1, 4, 100])) if rng.random() < 0.3 else (0, 0)
    return dict(kind=kind, seqs=seqs, tokens=tokens, fewest=fewest, shortest=_log(rng, 1, longest),
                longest=longest, page=page, window=window, sinks=sinks, kv8=rng.random() < 0.5)


def _spread(n, lo, hi):
    """n whole numbers from lo to hi, spread geometrically, not in order."""
    if n == 1:
        return [hi]
    xs = [int(round(lo * (hi / lo) ** (i / (n - 1)))) for i in range(n)]
    step = next(s for s in (5, 7, 11, 1) if math.gcd(s, n) == 1)
    return [xs[i * step % n] for i in range(n)]


def _contexts(case):
    """Context rows of every sequence."""
    if case["kind"] == "tree":
        return _spread(case["seqs"], case["shortest"], case["longest"])
    return [case["pos"] + (13 * i if case["pos"] else 0) for i in range(case["seqs"])]


def _sizes(case):
    """Tokens of every sequence's tree."""
    return list(reversed(_spread(case["seqs"], case.get("fewest", case["tokens"]), case["tokens"])))


# ---------------------------------------------------------------------------
# inputs, from the seed alone
# ---------------------------------------------------------------------------

def _randn(g, *shape, scale=1.0, dtype=F16):
    x = torch.empty(shape, dtype=F32, device="cuda").normal_(0.0, scale, generator=g)
    return x if dtype == F32 else x.to(dtype)


def _pool(g, rows, kv8):
    """A pool of `rows` cached rows of KV heads: fp16 values or the int8 format
    (values [rows, KV, DIM] int8, then scales [rows, KV, DIM / 32] fp16, flat)."""
    if not kv8:
        return _randn(g, rows, KV, DIM)
    vals, scales = rows * KV * DIM, rows * KV * (DIM // 32)
    pool = torch.zeros(vals + 2 * scales, dtype=torch.int8, device="cuda")
    pool[:vals].random_(-127, 128, generator=g)
    pool[vals:] = (_randn(g, scales, dtype=F32).abs() * 0.005 + 0.012).half().view(torch.int8)
    return pool


def _trees(seed, sizes, tokens):
    """parents [B, tokens] on the host: half of the tokens go on from the one before them, as the
    likeliest path does, the others from any earlier one."""
    g = torch.Generator().manual_seed(int(seed) * 104729 + 5)
    parents = torch.full((len(sizes), tokens), -2, dtype=I32)
    for b, n in enumerate(sizes):
        u = torch.rand(2, n, generator=g)
        for i in range(n):
            parents[b, i] = i - 1 if i == 0 or u[0, i] < 0.5 else int(u[1, i] * i)
    return parents


def _depths(parents):
    depth = torch.zeros_like(parents)
    for b in range(parents.shape[0]):
        for i in range(parents.shape[1]):
            p = int(parents[b, i])
            depth[b, i] = depth[b, p] + 1 if p >= 0 else 0
    return depth


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 29)
    kind = case["kind"]
    s = dict(case)
    host = torch.Generator().manual_seed(int(seed) * 31337 + 3)
    if kind == "copy":
        rows = case["pool"] * case["page"]
        for name in ("kpools", "vpools"):
            pools = [_pool(g, rows, case["kv8"]) for _ in range(case["layers"])]
            s[name] = pools if case["kv8"] else [p.view(case["pool"], case["page"], KV, DIM) for p in pools]
        order = torch.randperm(case["pool"], generator=host).to(I32).cuda()
        n = case["pages"]
        s["src"], s["dst"] = order[:n].contiguous(), order[n:2 * n].contiguous()
        s["all"] = torch.arange(case["pool"], dtype=I32, device="cuda")[None]
        s["starts"] = torch.tensor([0, rows], dtype=I32, device="cuda")
        s["zero"] = torch.zeros(1, dtype=I32, device="cuda")
        return s
    B, T = case["seqs"], case["tokens"]
    if kind in ("gdn", "commit"):
        s["x"] = _randn(g, B, T, WIDTH)
        s["a"], s["b"] = _randn(g, B, T, VH, dtype=F32), _randn(g, B, T, VH, dtype=F32)
        s["A_log"], s["dt"] = _randn(g, VH, scale=0.3, dtype=F32), _randn(g, VH, scale=0.3, dtype=F32)
        s["conv_w"] = _randn(g, WIDTH, 4, scale=0.5)
        s["frames"] = [_randn(g, WIDTH, 3) for _ in range(B)]
        s["S"] = [_randn(g, VH, VD, KD, scale=0.05, dtype=F32) for _ in range(B)]
        s["pos0"] = [0 if case.get("fresh") and b % 2 == 0 else 1000 + 7 * b for b in range(B)]
    if kind == "gdn":
        s["z"], s["norm_w"] = _randn(g, B, T, VH * VD), 1.0 + _randn(g, VD, scale=0.2, dtype=F32)
        s["parents"] = _trees(seed, _sizes(case), T).cuda()
        return s
    if kind in ("commit", "keep"):
        # accepted paths, the first tokens at their places already or from behind the path, as
        # wide trees number them (so that a second pass finds the same rows)
        path = torch.full((B, case["accepted"]), -1, dtype=I32)
        for b in range(B):
            n = case["accepted"] - (b * 3) % case["accepted"] if B > 1 else case["accepted"]
            stay = int(torch.randint(0, n + 1, (1,), generator=host))
            far = torch.randperm(T - n, generator=host)[:n - stay].sort().values + n
            stay = n - far.numel()
            path[b, :stay] = torch.arange(stay, dtype=I32)
            path[b, stay:n] = far.to(I32)
        s["path"] = path.cuda()
    if kind == "commit":
        s["S_out"] = [torch.empty_like(x) for x in s["S"]]
        s["frames_out"] = [torch.empty_like(x) for x in s["frames"]]
        return s
    # a paged cache with the sequences' pages in the order that a long-running pool hands them out
    page, kv8 = case["page"], case.get("kv8", False)
    contexts = _contexts(case)
    count = [(c + T + page - 1) // page for c in contexts]
    first = [c // page if kind == "axes" else 0 for c in contexts]
    n_pages = sum(c - f for c, f in zip(count, first)) + 3
    order = torch.randperm(n_pages, generator=host).to(I32)
    pages = torch.full((B, max(count)), -1, dtype=I32)
    at = 0
    for b in range(B):
        n = count[b] - first[b]
        pages[b, first[b]:count[b]] = order[at:at + n]
        at += n
    s["pages"], s["rows"] = pages.cuda(), n_pages * page
    s["pos0"] = torch.tensor(contexts, dtype=I32, device="cuda")
    layers = case.get("layers", 1)
    for name in ("kpools", "vpools"):
        pools = [_pool(g, s["rows"], kv8) for _ in range(layers)]
        s[name] = pools if kv8 else [p.view(n_pages, page, KV, DIM) for p in pools]
    if kind == "tree":
        s["qg"] = _randn(g, B, T, HEADS, 2 * DIM)
        s["parents"] = _trees(seed, _sizes(case), T).cuda()
    if kind == "axes":
        s["qg"], s["k"], s["v"] = (_randn(g, B * T, *d) for d in ((HEADS, 2 * DIM), (KV, DIM), (KV, DIM)))
        s["wq"], s["wk"] = (_randn(g, DIM, scale=0.1, dtype=F32) for _ in range(2))
        s["starts"] = torch.arange(0, B * T + 1, T, dtype=I32, device="cuda")
        s["q_out"] = torch.empty((B * T, HEADS, DIM), dtype=F16, device="cuda")
        axes, pairs = case["axes"], ROPE // 2
        s["sections"] = [pairs - (axes - 1) * (pairs // axes)] + [pairs // axes] * (axes - 1)
        base = torch.tensor(contexts)[:, None]
        i = torch.arange(T)[None].expand(B, T)
        side = max(1, int(math.sqrt(T)))
        if axes == 1:     # a tree's depths
            at = [base + (_depths(_trees(seed, [T] * B, T)) if T <= 64 else i)]
        else:             # time, then the rows and columns of a picture (and a video's frames of it)
            at = [base + i // (side * side), base + i // side % side, base + i % side, base + i // 7][:axes]
        s["positions"] = torch.stack([a.reshape(-1) for a in at]).to(I32).cuda()
    return s


# ---------------------------------------------------------------------------
# the plain forms: elementary operations in 32 bits
# ---------------------------------------------------------------------------

def _row_at(s, b, positions):
    return s["pages"][b].long()[positions // s["page"]] * s["page"] + positions % s["page"]


def _fetch(pool, rows, n, kv8):
    """Cached rows in 32 bits; n: rows of the pool."""
    if not kv8:
        return pool.view(n, KV, DIM)[rows].float()
    cut = n * KV * DIM
    scales = pool[cut:].view(F16).view(n, KV, DIM // 32)[rows].float()
    return pool[:cut].view(n, KV, DIM)[rows].float() * scales.repeat_interleave(32, -1)


def _axis_of(s):
    """The axis of each rotary pair: section after section, or, interleaved, pair j axis j % axes
    as far as that axis' section goes and the first axis behind it."""
    axes, pairs = s["axes"], ROPE // 2
    if s["interleaved"]:
        return [j % axes if j < axes * s["sections"][j % axes] else 0 for j in range(pairs)]
    return [a for a in range(axes) for _ in range(s["sections"][a])]


def _axes(s):
    half = ROPE // 2
    freq = THETA ** (-2.0 * torch.arange(half, dtype=F64, device="cuda") / ROPE)
    angle = s["positions"].double()[torch.tensor(_axis_of(s), device="cuda")].t() * freq
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def heads(x, w):
        x = x.float()
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * (1.0 + w)
        a, b = x[..., :half], x[..., half:ROPE]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., ROPE:]], -1).half()

    T = s["tokens"]
    rows = torch.cat([_row_at(s, b, c + torch.arange(T, device="cuda")) for b, c in enumerate(_contexts(s))])
    s["kpools"][0].view(-1, KV, DIM)[rows] = heads(s["k"], s["wk"])
    s["vpools"][0].view(-1, KV, DIM)[rows] = s["v"]
    return heads(s["qg"][..., :DIM], s["wq"]), s["kpools"][0], s["vpools"][0]


def _family(parents):
    """[T, T] truth values of one tree: row i's ancestors and itself; depths."""
    T = parents.numel()
    line = torch.eye(T, dtype=torch.bool)
    for i in range(T):
        p = int(parents[i])
        if p >= 0:
            line[i] |= line[p]
    return line, line.sum(1) - 1


def _tree(s):
    T, kv8 = s["tokens"], s["kv8"]
    out = torch.zeros((s["seqs"], T, HEADS, DIM), dtype=F16, device="cuda")
    parents = s["parents"].cpu()
    for b, (c, n) in enumerate(zip(_contexts(s), _sizes(s))):
        line, depth = _family(parents[b, :n])
        line, depth = line.cuda(), depth.cuda()
        # the rows' positions, and who sees them
        lowest = max(0, c - s["window"] + 1) if s["window"] else 0
        ctx = torch.cat([torch.arange(min(s["sinks"], lowest), device="cuda"),
                         torch.arange(lowest, c, device="cuda")])
        place = torch.cat([ctx, c + torch.arange(n, device="cuda")])
        at = torch.cat([ctx, c + depth])
        see = torch.cat([torch.ones((n, ctx.numel()), dtype=torch.bool, device="cuda"), line], 1)
        if s["window"]:
            see &= (at[None] > (c + depth)[:, None] - s["window"]) | (at[None] < s["sinks"])
        rows = _row_at(s, b, place)
        k, v = (_fetch(s[p][0], rows, s["rows"], kv8) for p in ("kpools", "vpools"))
        for h in range(KV):
            q = s["qg"][b, :n, h * GROUP:(h + 1) * GROUP, :DIM].float()
            scores = (q.reshape(-1, DIM) @ k[:, h].t()).view(n, GROUP, -1) * SCALE
            scores.masked_fill_(~see[:, None], float("-inf"))
            e = (scores - scores.amax(-1, keepdim=True)).exp()
            z = (e.view(n * GROUP, -1) @ v[:, h]).view(n, GROUP, DIM) / e.sum(-1, keepdim=True)
            gate = s["qg"][b, :n, h * GROUP:(h + 1) * GROUP, DIM:].float()
            out[b, :n, h * GROUP:(h + 1) * GROUP] = (z / (1.0 + (-gate).exp())).half()
    return out


def _conv(s, b, x3, x2, x1, x0):
    """silu of the four taps, and its q, k (unit length) and v."""
    w = s["conv_w"].float()
    y = w[:, 0] * x3 + w[:, 1] * x2 + w[:, 2] * x1 + w[:, 3] * x0
    y = y / (1.0 + (-y).exp())
    q, k, v = y[:KH * KD].view(KH, KD), y[KH * KD:2 * KH * KD].view(KH, KD), y[2 * KH * KD:].view(VH, VD)
    q, k = (t * torch.rsqrt((t * t).sum(-1, keepdim=True) + 1e-6) for t in (q, k))
    return q.repeat_interleave(SHARE, 0), k.repeat_interleave(SHARE, 0), v


def _gates(s):
    pre = s["a"] + s["dt"]
    soft = torch.where(pre > 20.0, pre, pre.clamp(max=20.0).exp().log1p())
    return (-s["A_log"].exp() * soft).exp(), 1.0 / (1.0 + (-s["b"]).exp())


def _first_frames(s, b):
    return list(s["frames"][b].float().unbind(1)) if s["pos0"][b] else [torch.zeros(WIDTH, device="cuda")] * 3


def _step(S, alpha, beta, k, v):
    S = S * alpha[:, None, None]
    delta = (v - (S * k[:, None]).sum(-1)) * beta[:, None]
    return S + delta[..., None] * k[:, None]


def _gdn(s):
    alpha, beta = _gates(s)
    out = torch.zeros((s["seqs"], s["tokens"], VH * VD), dtype=F16, device="cuda")
    parents = s["parents"].cpu()
    for b, n in enumerate(_sizes(s)):
        states, frames = {-1: s["S"][b]}, {-1: _first_frames(s, b)}
        for i in range(n):
            p = int(parents[b, i])
            x0 = s["x"][b, i].float()
            f = frames[p]
            q, k, v = _conv(s, b, *f, x0)
            frames[i] = [f[1], f[2], x0]
            S = states[i] = _step(states[p], alpha[b, i], beta[b, i], k, v)
            o = (S * q[:, None]).sum(-1) * OUT_SCALE
            o = o * torch.rsqrt((o * o).mean(-1, keepdim=True) + 1e-6) * s["norm_w"]
            z = s["z"][b, i].float().view(VH, VD)
            out[b, i] = (o * z / (1.0 + (-z).exp())).half().view(-1)
    return out


def _commit(s):
    alpha, beta = _gates(s)
    path = s["path"].cpu()
    for b in range(s["seqs"]):
        S, f = s["S"][b], _first_frames(s, b)
        for i in (int(i) for i in path[b] if i >= 0):
            x0 = s["x"][b, i].float()
            _, k, v = _conv(s, b, *f, x0)
            f = [f[1], f[2], x0]
            S = _step(S, alpha[b, i], beta[b, i], k, v)
        s["S_out"][b].copy_(S)
        s["frames_out"][b].copy_(torch.stack(f, 1))
    return s["S_out"], s["frames_out"]


def _copy(s):
    src, dst, n = s["src"].long(), s["dst"].long(), s["pool"] * s["page"]
    for pool in s["kpools"] + s["vpools"]:
        if s["kv8"]:
            cut = n * KV * DIM
            for part in (pool[:cut].view(s["pool"], -1), pool[cut:].view(s["pool"], -1)):
                part[dst] = part[src]
        else:
            pool[dst] = pool[src]
    if not s["kv8"]:
        return s["kpools"], s["vpools"]
    rows = torch.arange(n, device="cuda")
    return [_fetch(p, rows, n, True).half() for p in s["kpools"] + s["vpools"]]


def _keep(s):
    path = s["path"].cpu()
    src, dst = [], []
    for b, c in enumerate(_contexts(s)):
        nodes = path[b][path[b] >= 0].long().cuda()
        src.append(_row_at(s, b, c + nodes))
        dst.append(_row_at(s, b, c + torch.arange(nodes.numel(), device="cuda")))
    src, dst = torch.cat(src), torch.cat(dst)
    for pool in s["kpools"] + s["vpools"]:
        flat = pool.view(-1, KV, DIM)
        flat[dst] = flat[src]
    return s["kpools"], s["vpools"]


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    s = state
    kind = s["kind"]
    if not own:
        return dict(axes=_axes, tree=_tree, gdn=_gdn, commit=_commit, copy=_copy, keep=_keep)[kind](s)
    from __graft_entry__ import load_package
    ops = load_package().ops
    if kind == "axes":
        pools = s["kpools"][0], s["vpools"][0]
        ops.attn_prep_axes(s["qg"], s["k"], s["v"], s["wq"], s["wk"], *pools, s["pages"], s["starts"],
                           s["pos0"], s["positions"], page_size=s["page"], sections=s["sections"],
                           interleaved=s["interleaved"], q_out=s["q_out"])
        return s["q_out"], *pools
    if kind == "tree":
        return ops.attn_tree_paged(s["qg"], s["kpools"][0], s["vpools"][0], s["pages"], s["pos0"],
                                   s["parents"], page_size=s["page"], window=s["window"], sinks=s["sinks"])
    if kind == "gdn":
        return ops.gdn_tree_normed(s["x"], s["S"], s["a"], s["b"], s["A_log"], s["dt"], s["z"], s["norm_w"],
                                   s["parents"], pos0s=s["pos0"], conv_w=s["conv_w"], cst_in=s["frames"])
    if kind == "commit":
        ops.gdn_tree_commit(s["x"], s["S"], s["a"], s["b"], s["A_log"], s["dt"], s["path"], s["S_out"],
                            pos0s=s["pos0"], conv_w=s["conv_w"], cst_in=s["frames"], cst_out=s["frames_out"])
        return s["S_out"], s["frames_out"]
    if kind == "keep":
        ops.paged_kv_keep(s["kpools"], s["vpools"], s["pages"], s["pos0"], s["path"], page_size=s["page"])
        return s["kpools"], s["vpools"]
    ops.paged_kv_copy(s["kpools"], s["vpools"], s["src"], s["dst"], page_size=s["page"])
    if not s["kv8"]:
        return s["kpools"], s["vpools"]
    k, v = ops.paged_kv_load(s["kpools"][0], s["vpools"][0], s["all"], s["starts"], s["zero"],
                             T=s["pool"] * s["page"], page_size=s["page"])
    return [k, v]


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    kind, row = case["kind"], 272 if case.get("kv8") else 512       # bytes of a cached head row
    if kind == "copy":
        moved = 4 * case["layers"] * case["pages"] * case["page"] * KV * row
        n = case["pool"] * case["page"] * KV
        return {"bytes": moved + (2 * n * (row + 512) if case["kv8"] else 0),
                "flops": 2 * n * DIM if case["kv8"] else 0}
    B, T = case["seqs"], case["tokens"]
    if kind == "keep":
        return {"bytes": 4 * case["layers"] * B * case["accepted"] * KV * row // 2, "flops": 0}
    if kind == "axes":
        n = B * T
        return {"bytes": 2 * n * HEADS * DIM * 2 + 4 * n * KV * DIM * 2 + 2 * DIM * 4 + 4 * n * case["axes"],
                "flops": 6 * n * (HEADS + KV) * DIM}
    if kind == "commit":
        n = B * (case["accepted"] + 1) / 2 if B > 1 else case["accepted"]
        return {"bytes": int(2 * B * VH * VD * KD * 4 + n * (WIDTH * 2 + 2 * VH * 4) + 2 * B * WIDTH * 6
                             + WIDTH * 8), "flops": int(n * VH * 6 * VD * KD)}
    n = sum(_sizes(case))
    if kind == "gdn":
        return {"bytes": B * VH * VD * KD * 4 + n * (WIDTH * 2 + 2 * VH * 4 + 4) + B * WIDTH * 6 + WIDTH * 8
                + 2 * n * VH * VD * 2 + VD * 4, "flops": n * VH * (4 * VD * KD + 8 * (KD + VD))}
    rows = pairs = 0
    for c, t in zip(_contexts(case), _sizes(case)):
        seen = c if case["window"] == 0 else min(c, case["window"] - 1 + min(case["sinks"], max(0, c - case["window"] + 1)))
        rows += seen + t
        pairs += t * (seen + 1)
    return {"bytes": 3 * n * HEADS * DIM * 2 + 2 * rows * KV * row, "flops": 4 * pairs * HEADS * DIM}


# ---------------------------------------------------------------------------
# from the definition, in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    kind, page = case["kind"], case.get("page", 1)

    def where(b, positions):
        ids = s["pages"][b].long().gather(0, positions.div(page, rounding_mode="floor"))
        return ids * page + positions.remainder(page)

    def cached(pool, index):
        n = s["rows"]
        if not case["kv8"]:
            return pool.reshape(n, KV * DIM)[index].double().unflatten(-1, (KV, DIM))
        values = pool[:n * KV * DIM].reshape(n, KV * DIM)[index].double().unflatten(-1, (-1, 32))
        steps = pool[n * KV * DIM:].view(F16).reshape(n, KV * DIM // 32)[index].double()
        return (values * steps.unsqueeze(-1)).flatten(1).unflatten(-1, (KV, DIM))

    if kind == "copy":
        n = case["pool"] * page
        out = []
        for pool in s["kpools"] + s["vpools"]:
            index = torch.arange(n, device="cuda").view(case["pool"], page)
            index[s["dst"].long()] = index[s["src"].long()]
            s["rows"] = n
            got = cached(pool, index.flatten())
            out.append(got if case["kv8"] else got.reshape(pool.shape))
        L = case["layers"]
        return out if case["kv8"] else (out[:L], out[L:])
    if kind == "keep":
        both = []
        for pools in (s["kpools"], s["vpools"]):
            new = []
            for pool in pools:
                y = pool.double().reshape(-1, KV * DIM)
                z = y.clone()
                for b, c in enumerate(_contexts(case)):
                    for d, i in enumerate(s["path"][b].tolist()):
                        if i >= 0:
                            at = where(b, torch.tensor([c + d, c + i], device="cuda"))
                            z[at[0]] = y[at[1]]
                new.append(z.reshape(pool.shape))
            both.append(new)
        return tuple(both)
    B, T = case["seqs"], case["tokens"]
    if kind == "axes":
        pos, n_axes = s["positions"].double(), case["axes"]
        if case["interleaved"]:
            owner = [0] * (ROPE // 2)
            for a in range(1, n_axes):
                owner[a:n_axes * s["sections"][a]:n_axes] = [a] * len(range(a, n_axes * s["sections"][a], n_axes))
        else:
            owner = sum(([a] * m for a, m in enumerate(s["sections"])), [])

        def heads(x, w):
            x = x.double()
            x = x / (x.square().sum(-1, keepdim=True) / DIM + EPS).sqrt() * (w.double() + 1)
            y = x.clone()
            for j, a in enumerate(owner):
                t = pos[a] * math.pow(THETA, -2 * j / ROPE)
                c, d = torch.cos(t)[:, None], torch.sin(t)[:, None]
                u, v = x[..., j], x[..., j + ROPE // 2]
                y[..., j], y[..., j + ROPE // 2] = u * c - v * d, v * c + u * d
            return y
        index = torch.cat([where(b, torch.arange(c, c + T, device="cuda"))
                           for b, c in enumerate(_contexts(case))])
        out = [heads(s["qg"][..., :DIM], s["wq"])]
        for pool, x in ((s["kpools"][0], heads(s["k"], s["wk"])), (s["vpools"][0], s["v"].double())):
            y = pool.double().reshape(-1, KV, DIM)
            y[index] = x
            out.append(y.reshape(pool.shape))
        return tuple(out)
    if kind == "tree":
        out = torch.zeros((B, T, HEADS, DIM), dtype=F64, device="cuda")
        parents = s["parents"].tolist()
        for b, (c, n) in enumerate(zip(_contexts(case), _sizes(case))):
            index = where(b, torch.arange(c + n, device="cuda"))
            K, V = (cached(s[p][0], index) for p in ("kpools", "vpools"))
            for i in range(n):
                up = [i]
                while parents[b][up[-1]] >= 0:
                    up.append(parents[b][up[-1]])
                p = c + len(up) - 1
                r = torch.arange(c, device="cuda")
                if case["window"]:
                    r = r[(r > p - case["window"]) | (r < case["sinks"])]
                    up = [j for e, j in enumerate(up)
                          if e < case["window"] or p - e < case["sinks"]]
                r = torch.cat([r, c + torch.tensor(up, device="cuda")])
                for h in range(KV):
                    q = s["qg"][b, i, h * GROUP:(h + 1) * GROUP].double()
                    w = torch.softmax(q[:, :DIM] @ K[r, h].T / math.sqrt(DIM), -1)
                    out[b, i, h * GROUP:(h + 1) * GROUP] = (w @ V[r, h]) * torch.sigmoid(q[:, DIM:])
        return out
    # gated DeltaNet: a path's tokens one after the other
    decay = torch.exp(-s["A_log"].double().exp() * torch.nn.functional.softplus(s["a"].double() + s["dt"].double()))
    rate = torch.sigmoid(s["b"].double())
    taps = s["conv_w"].double().T

    def walk(b, S, past, i):
        past = torch.cat([past[1:], s["x"][b, i].double()[None]])
        y = torch.nn.functional.silu((taps * past).sum(0))
        q, k, v = y.split([KH * KD, KH * KD, VH * VD])
        q, k = (t.unflatten(0, (KH, 1, KD)).expand(KH, SHARE, KD).reshape(VH, KD) for t in (q, k))
        q, k = (t / (t.square().sum(-1, keepdim=True) + 1e-6).sqrt() for t in (q, k))
        S = S * decay[b, i].view(VH, 1, 1)
        fix = rate[b, i].unsqueeze(1) * (v.view(VH, VD) - torch.bmm(S, k.unsqueeze(2)).squeeze(2))
        S = S + torch.bmm(fix.unsqueeze(2), k.unsqueeze(1))
        return S, past, torch.bmm(S, q.unsqueeze(2)).squeeze(2) / math.sqrt(KD)

    def root(b):
        past = s["frames"][b].double().T * (1 if s["pos0"][b] else 0)
        return s["S"][b].double(), torch.cat([torch.zeros_like(past[:1]), past])
    if kind == "commit":
        states, frames = [], []
        for b in range(B):
            S, past = root(b)
            for i in s["path"][b].tolist():
                if i >= 0:
                    S, past, _ = walk(b, S, past, i)
            states.append(S)
            frames.append(past[1:].T)
        return states, frames
    out = torch.zeros((B, T, VH * VD), dtype=F64, device="cuda")
    for b in range(B):
        kept = {-1: root(b)}
        for i, p in enumerate(s["parents"][b].tolist()):
            if p < -1:
                continue
            S, past, o = walk(b, *kept[p], i)
            kept[i] = (S, past)
            o = o / (o.square().sum(-1, keepdim=True) / VD + 1e-6).sqrt() * s["norm_w"].double()
            out[b, i] = (o * torch.nn.functional.silu(s["z"][b, i].double().view(VH, VD))).view(-1)
    return out
