"""Plain 64-bit forms of the operators over cached sequences
(runtime/seq_ops.py), written from their definitions for the tests.

Tolerances. Inputs are BF16 and exact in both. The attention kernels keep
scores and sums in fp32 and round twice to BF16: the softmax weights before
their product with v (each off by at most 2^-8 of itself, so the output by at
most 2^-8 of the weighted mean of |v|, on top of the sum of the weights, which
is taken in fp32), and the output (2^-8 of itself: half a step is 2^-9 of the
next power of two above, at most 2^-8 of the value). fp32 effects: a score z
of hd products is off by at most hd 2^-24 sum|q d||k d| scale, and the
exponential turns an absolute error of its argument into a relative one of the
weight; with the inputs here (|z| up to about 30) that is below 1e-4, and the
same for the exponential itself (2^-20 covers its approximation). So
    |got - want| <= 2^-8 |want| + (2^-8 + 2e-4) mean|v| + 1e-30
with mean|v| = sum p |v| of the row.
"""
import torch


def attend(q, k, v, seen, scale):
    """q [t, hd], k, v [l, hd], seen bool [t, l], all 64-bit -> (out, sum p |v|)."""
    if k.shape[0] == 0:
        z = q.new_zeros(q.shape)
        return z, z
    s = (q @ k.T) * scale
    s = s.masked_fill(~seen, float("-inf"))
    m = s.amax(-1, keepdim=True)
    p = torch.where(seen, torch.exp(s - torch.where(m == float("-inf"), 0.0, m)), 0.0)
    l = p.sum(-1, keepdim=True)
    p = torch.where(l > 0, p / torch.where(l > 0, l, 1.0), 0.0)
    # an unseen value must not touch the sum, whatever it is: take it out where no row sees it,
    # and row by row where it is not finite
    bad = ~torch.isfinite(v).all(-1)
    vv = torch.where(bad[:, None], 0.0, v)
    out, size = p @ vv, p @ vv.abs()
    for j in torch.nonzero(bad).flatten().tolist():
        rows = seen[:, j]
        out[rows] += p[rows, j:j + 1] * v[j]
        # its finite values count in sum p |v| like all others: without them the sum can lie below |out|, which it bounds
        # (one seen key of weight 0.9 and value 0.35 beside a NaN: |out| 0.35, the sum without it 0.03)
        size[rows] += p[rows, j:j + 1] * torch.where(torch.isfinite(v[j]), v[j].abs(), 0.0)
    return out, size


def prompt(q, k, v, cu_q, scale, cu_k=None, len_k=None):
    """q [N, nh, hd]; packed or cached keys -> (out, size, rows computed)."""
    n, nh, hd = q.shape
    out = torch.zeros(n, nh, hd, dtype=torch.float64)
    size = torch.zeros_like(out)
    rows = torch.zeros(n, dtype=torch.bool)
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    nkv = k.shape[1]
    cu_q = cu_q.tolist()
    for b in range(len(cu_q) - 1):
        m = cu_q[b + 1] - cu_q[b]
        if k.dim() == 4:
            L = int(len_k[b])
            kk, vv = k[b, :, :L], v[b, :, :L]
        else:
            c = cu_q if cu_k is None else cu_k.tolist()
            L = c[b + 1] - c[b]
            kk, vv = k[c[b]:c[b + 1]].transpose(0, 1), v[c[b]:c[b + 1]].transpose(0, 1)
        seen = torch.arange(L)[None] <= (L - m + torch.arange(m))[:, None]
        rows[cu_q[b]:cu_q[b + 1]] = True
        for h in range(nh):
            g = h // (nh // nkv)
            o, s = attend(q[cu_q[b]:cu_q[b + 1], h], kk[g], vv[g], seen, scale)
            out[cu_q[b]:cu_q[b + 1], h], size[cu_q[b]:cu_q[b + 1], h] = o, s
    return out, size, rows


def tree(q, k, v, pos, mask, scale):
    B, T, nh, hd = q.shape
    nkv, rows = k.shape[1], k.shape[2]
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    mask = mask.cpu()
    out = torch.zeros(B, T, nh, hd, dtype=torch.float64)
    size = torch.zeros_like(out)
    for b in range(B):
        p = int(pos[b])
        mb = mask if mask.dim() == 2 else mask[b]
        seen = (torch.arange(rows) < p)[None].repeat(T, 1)
        for j in range(mb.shape[1]):
            if 0 <= p + j < rows:
                seen[:, p + j] = mb[:, j]
        for h in range(nh):
            g = h // (nh // nkv)
            out[b, :, h], size[b, :, h] = attend(q[b, :, h], k[b, g], v[b, g], seen, scale)
    return out, size


def check(got, want, size):
    got = got.double().cpu()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)])
    tol = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2e-4) * size + 1e-30
    off = ((got - want).abs() / tol)[fine]
    assert off.numel() == 0 or float(off.max()) <= 1.0, float(off.max())


def rope(qkv, nh, nkv, hd, cu, start, inv_freq, depth=None, q_norm=None, k_norm=None, eps=1e-6):
    """-> (q, k, v) of every row in 64 bits, slot [N], sequence [N] (-1: none)."""
    x = qkv.double().cpu().view(qkv.shape[0], nh + 2 * nkv, hd)
    cu, start = cu.tolist(), start.tolist()
    N = x.shape[0]
    seq = torch.full((N,), -1, dtype=torch.int64)
    slot = torch.zeros(N, dtype=torch.int64)
    place = torch.zeros(N, dtype=torch.float64)
    for b in range(len(start)):
        for n in range(cu[b], cu[b + 1]):
            seq[n], slot[n] = b, start[b] + n - cu[b]
            place[n] = start[b] + (n - cu[b] if depth is None else int(depth[n]))
    f = inv_freq.double().cpu()
    a = place[:, None] * f[None]
    c, s = torch.cos(a)[:, None], torch.sin(a)[:, None]
    half = hd // 2

    def turned(h, w):
        if w is not None:
            h = h / torch.sqrt(h.square().mean(-1, keepdim=True) + eps) * w.double().cpu()
        lo, hi = h[..., :half], h[..., half:]
        return torch.cat((lo * c - hi * s, hi * c + lo * s), -1), \
            torch.cat((lo.abs() + hi.abs(), lo.abs() + hi.abs()), -1)

    q, q_size = turned(x[:, :nh], q_norm)
    k, k_size = turned(x[:, nh:nh + nkv], k_norm)
    return q, q_size, k, k_size, x[:, nh + nkv:], seq, slot
