"""The paged operators' formulas in float64 torch, and the error that the kernels'
fp16 and fp32 roundings allow, for the paged cache's tests."""
import torch

EPS16 = 2.0 ** -11      # half a step of an fp16 value


def make_pages(g, lens, page_size, spare=2, device="cuda"):
    """Page tables for sequences of `lens` positions over a shuffled pool:
    (pages [B, max_pages] int32, -1 past a sequence's own; n_pages)."""
    count = [(n + page_size - 1) // page_size for n in lens]
    n_pages = max(1, sum(count) + spare)
    order = torch.randperm(n_pages, generator=g).to(torch.int32)
    pages = torch.full((len(lens), max(1, max(count))), -1, dtype=torch.int32)
    at = 0
    for b, c in enumerate(count):
        pages[b, :c] = order[at:at + c]
        at += c
    return pages.to(device), n_pages


def rows_of(pages, b, page_size, positions):
    """Pool rows of a sequence's positions (-1 where the page is absent); positions
    and the table on the CPU."""
    col = positions // page_size
    inside = col < pages.shape[1]
    ids = pages[b].long()[col.clamp(max=pages.shape[1] - 1)]
    return torch.where(inside & (ids >= 0), ids * page_size + positions % page_size,
                       torch.full_like(positions, -1))


def dequant(pool, n_rows, n_kv):
    """The values of a flat int8 pool, [n_rows, n_kv, 256] float64."""
    cut = n_rows * n_kv * 256
    v = pool[:cut].view(n_rows, n_kv, 8, 32).double()
    s = pool[cut:].view(torch.float16).view(n_rows, n_kv, 8).double()
    return (v * s[..., None]).view(n_rows, n_kv, 256)


def attention(q, K, V, pos, seen, scale, q8=False, gate=None):
    """q [n, Hq, 256], K / V [L, n_kv, 256], seen [n, L] bool, all on one device:
    (z [n, Hq, 256] float64, the elementwise error bound).

    The kernels' roundings, each half a step: the weights p to fp16 before the
    product with v (relative 2^-11 of sum w |v|); z to fp16, and once more after
    the gate; over int8 caches k and v to fp16 (v: 2^-11 of sum w |v|; k: every
    score off by at most d = scale 2^-11 sum |q| |k|, every weight by e^(2d) - 1).
    fp32: a score is a sum of 256 products (16 steps of 16, at most 32 roundings),
    its scaling and the exponential a few more; the sums over the rows add at
    most L / 8 + 64 times in sequence, in the numerator and the denominator."""
    n, Hq, _ = q.shape
    n_kv, L = K.shape[1], K.shape[0]
    G = Hq // n_kv
    z = torch.zeros((n, Hq, 256), dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(z)
    any_seen = seen.any(-1)
    for h in range(Hq):
        k, v = K[:, h // G].double(), V[:, h // G].double()
        k = torch.where(seen.any(0)[:, None], k, torch.zeros_like(k))
        v = torch.where(seen.any(0)[:, None], v, torch.zeros_like(v))
        qh = q[:, h].double()
        s = (qh @ k.t()) * scale
        s = torch.where(seen, s, torch.full_like(s, -float("inf")))
        w = torch.where(any_seen[:, None], torch.softmax(s, -1), torch.zeros_like(s))
        zh, ah = w @ v, w @ v.abs()
        size = torch.where(seen, scale * (qh.abs() @ k.abs().t()), torch.zeros_like(s))
        d = size.amax(-1, keepdim=True)
        rel = EPS16 + 2 * (L / 8 + 64) * 2.0 ** -24 + 2 * d * 40 * 2.0 ** -24 + 2.0 ** -20
        if q8:
            rel = rel + EPS16 + torch.expm1(2 * d * EPS16)
        b = ah * rel
        if gate is not None:
            sg = torch.sigmoid(gate[:, h].double())
            zh, b = zh * sg, b * sg + EPS16 * (zh * sg).abs() + EPS16 * b
        z[:, h] = zh
        bound[:, h] = b + EPS16 * (zh.abs() + b) + 2.0 ** -24
    return z, bound
