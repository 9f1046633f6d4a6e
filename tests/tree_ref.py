"""The operators over trees of drafted tokens in float64, and the error that the kernels'
arithmetic allows."""
import torch

F16, F32, F64, I32 = torch.float16, torch.float32, torch.float64, torch.int32
EPS16 = 2.0 ** -11


def lines(parents):
    """Of one sequence's parents (a list): each token's path from the context to itself, None for
    places that hold no token."""
    out = []
    for i, p in enumerate(parents):
        if p == -1:
            out.append([i])
        elif 0 <= p < i and out[p] is not None:
            out.append(out[p] + [i])
        else:
            out.append(None)
    return out


def gdn_layer(g, B, T, n_k=16, n_v=48, extra=0, ab_extra=0, device="cuda"):
    """Random inputs of a GDN layer (g: a CPU generator)."""
    dim = 2 * n_k * 128 + n_v * 128

    def r(*s, scale=1.0, dtype=F32):
        return (torch.randn(s, generator=g) * scale).to(dtype).to(device)
    return dict(x=r(B, T, dim + extra, dtype=F16), S=[r(n_v, 128, 128, scale=0.05) for _ in range(B)],
                a=r(B, T, n_v + ab_extra), b=r(B, T, n_v + ab_extra), A_log=r(n_v, scale=0.3),
                dt_bias=r(n_v, scale=0.3), z=r(B, T, n_v * 128, dtype=F16), norm_w=1 + r(128, scale=0.2),
                conv_w=r(dim, 4, scale=0.5, dtype=F16), cst=[r(dim, 3, dtype=F16) for _ in range(B)],
                n_k=n_k, n_v=n_v)


class Walk:
    """One sequence's paths in float64, with a bound of the error in fp32.

    The kernels solve for u_i = beta (v - (alpha S) k), a row of v apart. A computed u_i is the exact
    one of a step whose sums are off by eps_i = C (|v_i| + |S0| |k_i| + sum_j |k_i.k_j| |u_j|): products
    summed over at most 128 + 64 terms (2^-24 a term, 2^-16.4 of the sums of their magnitudes in the
    worst order), and under it the conv's, norms', gates' and ratios' few 2^-23 each (a decay's
    logarithm along a path of 64: 2^-18). C = 2^-15 holds both. A step (alpha <= 1, |k| <= 1, beta <= 1)
    never enlarges what an earlier one left in a row of the state, so a row of S is off by the sum
    of eps over the path at most, in its Euclidean norm, and beside that by C of its own size."""
    C = 2.0 ** -15

    def __init__(self, d, b, fresh):
        self.d, self.b = d, b
        n_k, n_v = d["n_k"], d["n_v"]
        self.dim = 2 * n_k * 128 + n_v * 128
        f = d["cst"][b].double()
        if fresh:
            f = torch.zeros_like(f)
        self.nodes = {-1: (d["S"][b].double(), list(f.unbind(1)), torch.zeros(n_v, 128, dtype=F64, device=f.device),
                           [], [])}

    def step(self, i, p):
        d, b = self.d, self.b
        n_k, n_v = d["n_k"], d["n_v"]
        S, f, eps, us, ks = self.nodes[p]
        x0 = d["x"][b, i, :self.dim].double()
        w = d["conv_w"].double()
        y = torch.nn.functional.silu(w[:, 0] * f[0] + w[:, 1] * f[1] + w[:, 2] * f[2] + w[:, 3] * x0)
        q, k = (t.view(n_k, 128) for t in (y[:n_k * 128], y[n_k * 128:2 * n_k * 128]))
        q, k = ((t / (t.square().sum(-1, keepdim=True) + 1e-6).sqrt()).repeat_interleave(n_v // n_k, 0)
                for t in (q, k))
        v = y[2 * n_k * 128:].view(n_v, 128)
        alpha = torch.exp(-d["A_log"].double().exp() * torch.nn.functional.softplus(
            d["a"][b, i, :n_v].double() + d["dt_bias"].double()))
        beta = torch.sigmoid(d["b"][b, i, :n_v].double())
        S = S * alpha[:, None, None]
        u = beta[:, None] * (v - (S @ k[..., None])[..., 0])
        size = v.abs() + (d["S"][b].double().abs() @ k.abs()[..., None])[..., 0]
        for uj, kj in zip(us, ks):
            size = size + (k * kj).sum(-1).abs()[:, None] * uj.abs()
        S = S + u[..., None] * k[:, None]
        eps = eps + self.C * size
        self.nodes[i] = (S, [f[1], f[2], x0], eps, us + [u], ks + [k])
        o = (S @ q[..., None])[..., 0]
        size_o = (d["S"][b].double().abs() @ q.abs()[..., None])[..., 0]
        for uj, kj in zip(us + [u], ks + [k]):
            size_o = size_o + (q * kj).sum(-1).abs()[:, None] * uj.abs()
        return o, eps + self.C * size_o


def gdn_tree(d, parents, fresh):
    """(y [B, T, n_v * 128] float64, its error bound): parents a list of lists, fresh a list. An error
    e of o moves y = o / rms(o) w silu(z) by |w silu(z)| / rms (|e| + |o| |e|_2 / |o|_2); y is rounded once."""
    B, T = len(parents), len(parents[0])
    n_v, scale = d["n_v"], 128 ** -0.5
    y = torch.zeros(B, T, n_v, 128, dtype=F64, device=d["x"].device)
    bound = torch.zeros_like(y)
    for b in range(B):
        walk = Walk(d, b, fresh[b])
        for i, line in enumerate(lines(parents[b])):
            if line is None:
                continue
            o, e = walk.step(i, line[-2] if len(line) > 1 else -1)
            o, e = o * scale, e * scale
            inv = 1 / (o.square().mean(-1, keepdim=True) + 1e-6).sqrt()
            z = d["z"][b, i].double().view(n_v, 128)
            gate = d["norm_w"].double() * torch.nn.functional.silu(z)
            y[b, i] = o * inv * gate
            spread = e.norm(dim=-1, keepdim=True) / o.norm(dim=-1, keepdim=True).clamp_min(1e-30)
            bound[b, i] = gate.abs() * inv * (e + o.abs() * spread) + y[b, i].abs() * (EPS16 + 2.0 ** -18) + 2.0 ** -25
    return y.view(B, T, -1), bound.view(B, T, -1)


def accepted(path, T):
    """The tokens of a path, as far as it goes."""
    out = []
    for i in path:
        if i <= (out[-1] if out else -1) or i >= T:
            break
        out.append(i)
    return out


def gdn_commit(d, paths, fresh):
    """Per sequence (S, its error bound, frames) behind a path."""
    out = []
    for b, path in enumerate(paths):
        walk, at = Walk(d, b, fresh[b]), -1
        for i in accepted(path, d["x"].shape[1]):
            walk.step(i, at)
            at = i
        S, f, eps, _, _ = walk.nodes[at]
        out.append((S, eps[..., None] + Walk.C * S.abs(), torch.stack(f, 1).half()))
    return out
