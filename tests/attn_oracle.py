"""Plain 64-bit restatements of the attention operators for the tests, and how far a kernel's output may be off.

A bf16 rounding is off by at most half a step, 2^-8 relative; an fp32 one by 2^-24."""
import torch

KEYS, QROWS = 64, 128
BF16_HALF, F32_HALF = 2.0 ** -8, 2.0 ** -24


def softmax_rows(q, k, v, scale, seen=None):
    """(o, a, bound) of one head in 64 bits: o = softmax(scale q k^T) v over the keys that `seen` [rows, n] counts
    (None: each once), a the same with |v|, m the largest sum of |products| behind a score of the row.  Rows without
    a key are zero."""
    q, k, v = q.double(), k.double(), v.double()
    s = scale * (q @ k.T)
    m = (abs(scale) * (q.abs() @ k.abs().T)).amax(1, keepdim=True) if k.shape[0] else q.new_zeros(q.shape[0], 1)
    w = torch.ones_like(s) if seen is None else seen.double()
    s = torch.where(w > 0, s, torch.full_like(s, -torch.inf))
    top = s.amax(1, keepdim=True) if k.shape[0] else s.new_zeros(q.shape[0], 1)
    p = w * torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(1, keepdim=True)
    p = torch.where(total > 0, p / total, torch.zeros_like(p))
    return p @ v, p @ v.abs(), m


def tolerance(o, a, m, n, d, vsum=0.0):
    """Bound on |kernel - o|: the result's rounding to bf16, and, relative to a = sum p |v|: p's rounding to bf16
    before the second product; scores as sums of d products and two factors in fp32, an absolute error of
    (d + 4) 2^-24 m each that moves p and the sum of p by as much; the exponential (2^-20 covers ex2.approx and the
    rounding of its argument at |argument| < 8; larger arguments come with an m that covers them); sums over n keys in
    fp32.  vsum, the sum of |v| over the keys, where p may be rounded to fp16 instead: relative 2^-11, which 2^-8 covers,
    but no less than half of fp16's smallest step, 2^-25.  p is 2^11 there for the key that set the row's reference, so
    the sum of p is 2^11 at least and a weight is off by 2^-36 at most: vsum 2^-36 together."""
    return BF16_HALF * (o.abs() + a * (1 + 2.0 ** -7)) + a * (2 * (d + 4) * F32_HALF * m + 2.0 ** -20 + 2 * n * F32_HALF) \
        + vsum * 2.0 ** -36 + 1e-30


def quantise(x, codes, scales, start):
    """The cache's definition for x [n, H, D] (bf16 values) written at `start` into codes [H, cap, D] and scales
    [H, cap / 64]; fp32 quotients as defined, everything else exact.  Token by token blocks, on the CPU."""
    x, codes, scales = x.float().cpu(), codes.cpu().clone(), scales.cpu().clone()
    n = x.shape[0]
    for b in range(start // KEYS, -(-(start + n) // KEYS)):
        lo, hi = max(start, b * KEYS), min(start + n, (b + 1) * KEYS)
        part = x[lo - start:hi - start].transpose(0, 1)  # [H, m, D]
        bad = ~torch.isfinite(part).all(2).all(1)
        s = part.abs().amax((1, 2)) / torch.tensor(127.0)
        old = codes[:, b * KEYS:lo].float()
        former = scales[:, b]
        if lo > b * KEYS:
            s = torch.where((former > s) | torch.isnan(former), former, s)
            ratio = torch.where(s > 0, former / s, torch.ones_like(s))
            old = (old * ratio[:, None, None]).round()
        c = torch.where(s[:, None, None] > 0, part / s[:, None, None], torch.zeros_like(part)).round().clamp(-127, 127)
        c[bad] = 0
        if lo > b * KEYS:
            old[bad] = 0
            codes[:, b * KEYS:lo] = old.to(torch.int8)
        codes[:, lo:hi] = c.to(torch.int8)
        scales[:, b] = s
    return codes, scales


def means(x, rows):
    """Means of blocks of rows, exact sums rounded once to fp32."""
    out = [x[i:i + rows].double().sum(0) / torch.tensor(float(min(rows, x.shape[0] - i)), dtype=torch.float64)
           for i in range(0, x.shape[0], rows)]
    return torch.stack(out).float() if out else x.new_zeros((0, *x.shape[1:]), dtype=torch.float32)


def select(qm, km, topk):
    """[H, nq, topk] ascending indices of the largest products; ties to the lowest index, NaN last."""
    s = torch.einsum("ihd,jhd->hij", qm.double(), km.double())
    s = torch.where(torch.isnan(s), torch.full_like(s, -torch.inf), s)
    return s.sort(dim=2, descending=True, stable=True)[1][:, :, :topk].sort(dim=2)[0].int()


def sparse(q, k, v, blocks, scale):
    """(o, a, m, n) [rows, H, D] / [rows, H, 1] of block-sparse attention in 64 bits; blocks [H, nq, n] with -1."""
    r, h, d = q.shape
    s = k.shape[0]
    o, a = (torch.zeros(r, h, d, dtype=torch.float64, device=q.device) for _ in "oa")
    m = torch.zeros(r, h, 1, dtype=torch.float64, device=q.device)
    for i in range(h):
        for b in range(-(-r // QROWS)):
            rows = slice(b * QROWS, min(r, (b + 1) * QROWS))
            count = torch.zeros(s, device=q.device)
            for j in blocks[i, b].tolist():
                if 0 <= j * KEYS < s:
                    count[j * KEYS:(j + 1) * KEYS] += 1
            at = count.nonzero()[:, 0]
            seen = count[at][None].expand(rows.stop - rows.start, -1)
            o[rows, i], a[rows, i], m[rows, i] = softmax_rows(q[rows, i], k[at, i], v[at, i], scale, seen)
    return o, a, m
