"""Data on which a lost, repeated or swapped tile of cached rows shows, and the error that the
paged attention kernels' roundings allow when the reference starts from the values they form.

Over int8 pools the kernels take K as byte * scale exactly and V as fp16(byte * scale): with
those as the reference's K and V the bound needs no term for the cache's format."""
import torch

import paged_ref as ref

EPS16 = 2.0 ** -11
ONE_TERM, TWO_TERMS = 2.0 ** -11, 2.0 ** -21   # a weight's rounding: one fp16, or that and the rest


def marked_rows(g, n, n_kv):
    """(k, v) [n, n_kv, 256] fp16: k random; v of row r is 0 but for a positive number in one
    dim that goes with its 32-row tile, another one in every kv head. So z[dim] is the weight of
    the tiles of that dim, sum w |v| is z itself, and a tile more or less is a good part of it."""
    r = torch.arange(n)
    k = torch.randn((n, n_kv, 256), generator=g)
    v = torch.zeros(n, n_kv, 256)
    for h in range(n_kv):
        v[r, h, (r // 32 * 5 + 37 * h) % 256] = 1 + (r % 32) / 64
    return k.half(), v.half()


def kernel_values(pool, n_rows, n_kv, exact):
    """A pool's rows in float64 as a kernel takes them (int8: exact, or rounded to fp16)."""
    if pool.dtype != torch.int8:
        return pool.view(n_rows, n_kv, 256).double()
    v = ref.dequant(pool, n_rows, n_kv)
    return v if exact else v.half().double()


def attention(q, K, V, seen, scale, p_rel, gate=None):
    """q [n, Hq, 256], K / V [L, n_kv, 256] as the kernel forms them, seen [n, L] bool: (z [n, Hq,
    256] float64, the elementwise error bound).

    Weights into the product with v: p_rel of each, or 2^-32 of the largest (half the step of a
    subnormal fp16, seven octaves under it). In 32 bits: a score's 16 x 16 products and its
    scaling (at most 40 roundings of its terms' absolute sum d), the exponential (2^-20), the
    sums over the rows (at most L / 8 + 64 additions in sequence, numerator and denominator), the
    sigmoid (2^-21). Then z once to fp16."""
    n, Hq, _ = q.shape
    n_kv, L = K.shape[1], K.shape[0]
    G = Hq // n_kv
    on = seen.any(0)[:, None, None]
    K = torch.where(on, K.double(), torch.zeros((), dtype=torch.float64, device=q.device))
    V = torch.where(on, V.double(), torch.zeros((), dtype=torch.float64, device=q.device))
    z = torch.zeros((n, Hq, 256), dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(z)
    for h in range(n_kv):
        qh = q[:, h * G:(h + 1) * G].double().reshape(n * G, 256)
        see = seen.repeat_interleave(G, 0)
        s = torch.where(see, qh @ K[:, h].t() * scale, -torch.inf)
        w = torch.nan_to_num(torch.softmax(s, -1))               # (sees none: 0)
        size = torch.where(see, scale * (qh.abs() @ K[:, h].abs().t()), 0.0).amax(-1, keepdim=True)
        zh, ah = w @ V[:, h], w @ V[:, h].abs()
        rel = p_rel + 2 * (L / 8 + 64) * 2.0 ** -24 + 2 * size * 40 * 2.0 ** -24 + 2.0 ** -20
        b = ah * rel + 2.0 ** -32 * w.amax(-1, keepdim=True) * (see.double() @ V[:, h].abs())
        if gate is not None:
            sg = torch.sigmoid(gate[:, h * G:(h + 1) * G].double().reshape(n * G, 256))
            zh, b = zh * sg, b * sg + 2.0 ** -21 * (zh * sg).abs()
        z[:, h * G:(h + 1) * G] = zh.view(n, G, 256)
        bound[:, h * G:(h + 1) * G] = (b + EPS16 * (zh.abs() + b) + 2.0 ** -25).view(n, G, 256)
    return z, bound


def int8_pool(values, scales):
    """The flat int8 pool of byte values [rows, n_kv, 256] and fp16 scales [rows, n_kv, 8]."""
    return torch.cat([values.to(torch.int8).flatten(), scales.half().flatten().view(torch.int8)])


def near_ties(L):
    """(k pool, v pool, q row [256]) of L int8 rows of one kv head on which fp16(byte * scale) for
    K is 5 % off: two kinds of rows, alternating, with scores of about 100 a thousandth apart;
    rounded to fp16 the one kind's K goes up by nearly half a step, the other's down. v tells
    the kinds apart (dim 0 and dim 1)."""
    s = (0.09 + 0.03 * torch.arange(512) / 512).half().double().unique()
    off = ((127 * s).half().double() - 127 * s) / (127 * s)
    up, down = s[off.argmax()], s[off.argmin()]
    size = torch.stack([up, down]) * 127                      # a row's k, all dims alike
    scales = torch.stack([up, down]).repeat(L)[:L].view(L, 1, 1).expand(L, 1, 8)
    # scores 0.0625 q 256 k: the dims' q of each kind's own half, so that both come to about 100
    q = torch.zeros(256)
    values = torch.zeros(L, 1, 256)
    for kind in range(2):
        dims = slice(128 * kind, 128 * kind + 128)
        q[dims] = 100 / (0.0625 * 128 * size[kind])
        values[kind::2, :, dims] = 127
    v = torch.zeros(L, 1, 256)
    v[0::2, :, 0], v[1::2, :, 1] = 127, 127
    return int8_pool(values, scales), int8_pool(v, torch.full((L, 1, 8), 1.0 / 128)), q.half()


def one_term_shows(L):
    """(k pool, v pool, q row [256]) of L int8 rows of one kv head: a first row of v = 0 and L - 1
    alike with weights some octaves below, nearly half a step of fp16 away from a value of it.
    In one fp16 term all of them are off by `off` (the fourth value) of themselves, the same way."""
    scales = (1 + torch.arange(1024).double() / 1024) / 4     # fp16 numbers in [1/4, 1/2)
    first = scales[-64:, None] * 2
    gap = 0.0625 * 1.4426950408889634 * 127 * (first - scales)   # q is 1 in dim 0, k 127 scale
    p = 2.0 ** -gap
    off = torch.where((gap > 2) & (gap < 9), (p.half().double() - p).abs() / p, 0.0)
    i = off.argmax().item()
    off, first, rest = off.flatten()[i], first[i // 1024, 0], scales[i % 1024]
    values, sc = torch.zeros(L, 1, 256), torch.zeros(L, 1, 8)
    values[:, :, 0] = 127
    sc[:, :, 0] = rest
    sc[0, :, 0] = first
    v, vs = torch.zeros(L, 1, 256), torch.full((L, 1, 8), 1.0 / 128)
    v[1:] = 1 + torch.arange(256) % 127
    qrow = torch.zeros(256)
    qrow[0] = 1
    return int8_pool(values, sc), int8_pool(v, vs), qrow.half(), off.item()
