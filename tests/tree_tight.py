"""Trees of drafted tokens on which the GDN kernel's operands show: outputs far smaller than the terms
that make them up, so that y's own rounding hides nothing, and the kernel's arithmetic in float64 with
each operand kept to as few bits as asked for."""
import torch

import tree_ref as ref

F16, F32, F64 = torch.float16, torch.float32, torch.float64


def inverse_silu(y):
    """s with silu(s) = y, for y > -0.278, where silu grows."""
    lo, hi = torch.full_like(y, -1.278), y.abs() * 2 + 2
    for _ in range(80):
        mid = (lo + hi) / 2
        low = mid * torch.sigmoid(mid) < y
        lo, hi = torch.where(low, mid, lo), torch.where(low, hi, mid)
    return (lo + hi) / 2


def layer_of(q, k, v, n_v, z_seed=1, device="cpu"):
    """A layer whose conv is its newest tap alone, so that a token's q, k (directions, [B, T, n_k, 128])
    and v ([B, T, n_v, 128], above -0.27) are what is asked for, but for x's rounding. Gates: beta and
    alpha 1 to 2^-40."""
    B, T, n_k, _ = q.shape
    g = torch.Generator().manual_seed(z_seed)
    q, k = (t.double() / t.double().abs().amax(-1, keepdim=True) * 0.2 for t in (q, k))
    y = torch.cat([q.flatten(2), k.flatten(2), v.double().flatten(2)], -1)
    dim = y.shape[-1]
    conv = torch.zeros(dim, 4)
    conv[:, 3] = 1
    to = lambda t, dtype: t.to(dtype).to(device)
    return dict(x=to(inverse_silu(y), F16), S=[to(torch.zeros(n_v, 128, 128), F32) for _ in range(B)],
                a=to(torch.full((B, T, n_v), -30.0), F32), b=to(torch.full((B, T, n_v), 30.0), F32),
                A_log=to(torch.zeros(n_v), F32), dt_bias=to(torch.zeros(n_v), F32),
                z=to(torch.randn((B, T, n_v * 128), generator=g).abs() + 0.5, F16), norm_w=to(torch.ones(128), F32),
                conv_w=to(conv, F16), cst=[to(torch.zeros(dim, 3), F16) for _ in range(B)], n_k=n_k, n_v=n_v)


def rows_of(d, b, i):
    """(q, k [n_k, 128], v [n_v, 128]) of a token, in float64, as the layer above forms them."""
    s = d["x"][b, i].double()
    y, n = s * torch.sigmoid(s), d["n_k"] * 128
    q, k = (t.view(d["n_k"], 128) for t in (y[:n], y[n:2 * n]))
    q, k = (t / (t.square().sum(-1, keepdim=True) + 1e-6).sqrt() for t in (q, k))
    return q, k, y[2 * n:].view(d["n_v"], 128)


def unseen_states(g, B, T, n_k, n_v, near, device="cpu"):
    """States that the tree's q and k are all orthogonal to, with values in a few of their rows alone: what
    S0 k and S0 q leave in the others is their operands' error. near: every q close to its k, so that an
    error of u shows (that of S0 k and S0 q themselves is the same then, and cancels)."""
    r = lambda *s: torch.randn(s, generator=g)
    k, v = r(B, T, n_k, 128), torch.zeros(B, T, n_v, 128)
    v[..., ::16] = 0.05 + 0.2 * torch.rand((B, T, n_v, 8), generator=g)
    d = layer_of(k + 0.3 * r(B, T, n_k, 128) if near else r(B, T, n_k, 128), k, v, n_v, device=device)
    for b in range(B):
        S = r(n_v, 128, 128).double()
        for h in range(n_k):
            Q = torch.linalg.qr(torch.cat([torch.stack([rows_of(d, b, i)[n][h] for i in range(T)])
                                           for n in (0, 1)]).cpu().t())[0]
            for m in range(h * n_v // n_k, (h + 1) * n_v // n_k):
                S[m] -= S[m] @ Q @ Q.t()
        d["S"][b] = S.float().to(device)
    return d


def cancelling_paths(g, B, T, n_k, n_v, device="cpu"):
    """(layer, parents): a root and its children, keys correlated, every head's values one direction (but in
    a few rows), and a child's q orthogonal to what its path's terms add up to: of (q.k0) u0 + (q.k1) u1
    nothing is left there."""
    r = lambda *s: torch.randn(s, generator=g)
    parents = [[-1] + [0] * (T - 1) for _ in range(B)]
    k = r(B, 1, n_k, 128) + 0.5 * r(B, T, n_k, 128)
    w = 0.05 + 0.2 * torch.rand((B, 1, n_v, 128), generator=g)
    v = w * (0.5 + torch.rand((B, T, n_k, 1), generator=g)).repeat_interleave(n_v // n_k, 2)
    v[..., ::16] = 0.05 + 0.2 * torch.rand((B, T, n_v, 8), generator=g)
    d = layer_of(k + 0.3 * r(B, T, n_k, 128), k, v, n_v, device=device)
    plain = torch.arange(128) % 16 != 0
    q = torch.zeros(B, T, n_k, 128, dtype=F64)
    for b in range(B):
        for h in range(n_k):
            m = h * n_v // n_k
            to = w[b, 0, m].double()[plain]
            size = lambda x: x[m].cpu()[plain] @ to / to.square().sum()
            _, k0, v0 = rows_of(d, b, 0)
            k0 = k0[h].cpu()
            for i in range(T):
                qi, ki, vi = rows_of(d, b, i)
                qi, ki = qi[h].cpu(), ki[h].cpu()
                line = k0 * size(v0)
                if i:
                    line = line + ki * (size(vi) - (ki @ k0) * size(v0))
                    qi = qi - line * (qi @ line) / line.square().sum()
                q[b, i, h] = qi
    return layer_of(q, k, v, n_v, device=device), parents


def terms(x, n, unit=1.0):
    """x as n fp16 terms of x * unit (None: as fp32)."""
    if n is None:
        return x.float().double()
    x = x * unit
    hi = x.half().double()
    return (hi if n == 1 else hi + (x - hi).half().double()) / unit


def bits11(x):
    """x with fp16's 11 bits, at any size."""
    m, e = torch.frexp(x)
    return torch.ldexp((m * 2048).round() / 2048, e)


def kernel_form(d, parents, S=2, q=2, k=2, system=None, shared=False):
    """y [B, T, n_v * 128] as the kernel forms it, rounded once: two fp16 terms of q, k (times 2^14) and S0
    (a row's largest number brought to 2^14), u and the coefficients in fp32. S, q, k: terms kept; system:
    "u", "A" or "P" in 11 bits; shared: a state row's S0 and u as two terms of one scale, by the largest v
    of all tokens. (Everything else, sums among it, in float64.)"""
    B, T = len(parents), len(parents[0])
    n_k, n_v, G = d["n_k"], d["n_v"], d["n_v"] // d["n_k"]
    y = torch.zeros(B, T, n_v, 128, dtype=F64, device=d["x"].device)
    few = lambda x, name: bits11(x) if system == name else x.float().double()
    for b in range(B):
        rows = [rows_of(d, b, i) for i in range(T)]
        qs, ks, vs = (torch.stack([r[n] for r in rows]) for n in range(3))
        qs, ks = (terms(t, n, 16384.0).repeat_interleave(G, 1) for t, n in ((qs, q), (ks, k)))
        S0 = d["S"][b].double()
        top = S0.abs().amax(-1, keepdim=True).clamp_min(1e-30)
        if shared:
            top = 32 * (64 * vs.abs().amax(0)[..., None] + 12 * top)
        unit = torch.exp2(14 - top.log2().floor())
        S0 = terms(S0, S, unit)
        trim = (lambda u: terms(u, 2, unit[..., 0])) if shared else (lambda u: few(u, "u"))
        us = []
        for i, line in enumerate(ref.lines(parents[b])):
            if line is None:
                us.append(None)
                continue
            u = vs[i] - (S0 @ ks[i][..., None])[..., 0]
            for j in line[:-1]:
                u = u - few((ks[i] * ks[j]).sum(-1), "A")[:, None] * us[j]
            us.append(trim(u))
            o = (S0 @ qs[i][..., None])[..., 0]
            for j in line:
                o = o + few((qs[i] * ks[j]).sum(-1), "P")[:, None] * us[j]
            o = o * 128 ** -0.5
            z = d["z"][b, i].double().view(n_v, 128)
            y[b, i] = (o / (o.square().mean(-1, keepdim=True) + 1e-6).sqrt() * d["norm_w"].double()
                       * torch.nn.functional.silu(z))
    return y.view(B, T, -1).half().double()
