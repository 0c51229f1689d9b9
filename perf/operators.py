"""The measured cases of the attention operators: the 8-bit key/value cache and block-sparse attention.

With `own` false, `run` computes an operator in its plain form (elementary torch operations); with `own` true it makes
the calls that a user makes of h3b.  Three kinds of case:

  write   KV8Cache.write of n new tokens at `start`, then KV8Cache.read of what that changed
  cached  kv8_attention: queries [rows, heads, dim] over a cache of `tokens` tokens held in 8 bits
  sparse  sparse_attention: each block of 128 query rows attends the `topk` blocks of 64 keys that the products of the
          blocks' means put first; with `means` the program keeps the key blocks' means between its calls

The model's sizes are those of the benchmark's block: 40 heads of 128, 512 text tokens, 128000 latent tokens (16000 per
GPU at 8, with 5 heads each after the exchange), 4128 tokens a latent frame.
"""
import math
import os
import sys

import torch

own = False

BLOCK = 64    # tokens of the cache that share a scale, and keys of a sparse block
QROWS = 128   # query rows that share a selection


def _h3b():
    root = os.path.join(os.getcwd(), "minimax-h3-multi-dgx-spark_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import h3b
    return h3b


def listed():
    return [
        # one token appended to a cache in the middle of a block: latency
        {"name": "write 1 token", "kind": "write", "heads": 40, "dim": 128, "start": 1000, "n": 1},
        # the text context of a prompt, written once for all denoising steps
        {"name": "write 512 text tokens", "kind": "write", "heads": 40, "dim": 128, "start": 0, "n": 512},
        # eight latent frames appended behind an odd prefix
        {"name": "write 33024 tokens at 77", "kind": "write", "heads": 40, "dim": 128, "start": 77, "n": 33024},
        # one query token over a short cache: latency
        {"name": "cached 1 x 512", "kind": "cached", "heads": 40, "dim": 128, "rows": 1, "tokens": 512},
        # one query token over a long cache of odd length: bandwidth
        {"name": "cached 1 x 131071", "kind": "cached", "heads": 40, "dim": 128, "rows": 1, "tokens": 131071},
        # a frame's rows over the frames before it, on one of eight GPUs
        {"name": "cached 4128 x 33024", "kind": "cached", "heads": 5, "dim": 128, "rows": 4128, "tokens": 33024},
        # cross-attention of one of eight GPUs' rows to the cached text
        {"name": "cached 16000 x 512", "kind": "cached", "heads": 40, "dim": 128, "rows": 16000, "tokens": 512},
        # cross-attention of the whole sequence to the cached text: the largest
        {"name": "cached 128000 x 512", "kind": "cached", "heads": 40, "dim": 128, "rows": 128000, "tokens": 512},
        # one query token over kept means
        {"name": "sparse 1 x 16389", "kind": "sparse", "heads": 40, "dim": 128, "rows": 1, "keys": 16389, "topk": 16,
         "means": True},
        # a small model's odd sizes
        {"name": "sparse 1000 heads of 64", "kind": "sparse", "heads": 16, "dim": 64, "rows": 1000, "keys": 1000,
         "topk": 5, "means": False},
        # a frame of latent tokens, all heads
        {"name": "sparse 4128", "kind": "sparse", "heads": 40, "dim": 128, "rows": 4128, "keys": 4128, "topk": 16,
         "means": False},
        # the whole sequence with one of eight GPUs' heads
        {"name": "sparse 128000", "kind": "sparse", "heads": 5, "dim": 128, "rows": 128000, "keys": 128000, "topk": 64,
         "means": False},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["write", "cached", "sparse"])
    heads, dim = rng.choice([1, 3, 5, 8, 10, 16, 20, 40]), rng.choice([64, 128, 128])
    if kind == "write":
        n = _log(rng, 1, 33024)
        return {"kind": kind, "heads": heads, "dim": dim, "start": rng.choice([0, rng.randint(1, 4200)]), "n": n}
    most = 128000 * 512 * 40 // 2  # scores of a pass, half the largest listed case's
    if kind == "cached":
        rows = 1 if rng.random() < 0.25 else _log(rng, 1, 128000)
        return {"kind": kind, "heads": heads, "dim": dim, "rows": rows,
                "tokens": _log(rng, 1, min(131071, most // (rows * heads)))}
    if rng.random() < 0.25:
        rows, keys, means = rng.randint(1, 4), _log(rng, 64, 131071), True
    else:
        rows = keys = _log(rng, 64, 65536)
        means = False
    nq = -(-rows // QROWS)
    topk = _log(rng, 1, max(1, min(96, most // (heads * nq * QROWS * BLOCK), -(-keys // BLOCK))))
    return {"kind": kind, "heads": heads, "dim": dim, "rows": rows, "keys": keys, "topk": topk, "means": means}


def work(case):
    h, d = case["heads"], case["dim"]
    if case["kind"] == "write":
        e, nb = case["n"] * h * d, _blocks(case["start"] % BLOCK + case["n"])
        # K and V: bf16 in, codes and scales written, bf16 read back
        return {"bytes": 2 * (2 + 1 + 2) * e + 2 * 4 * nb * h, "flops": 0}
    if case["kind"] == "cached":
        r, t = case["rows"], case["tokens"]
        return {"bytes": 2 * t * h * d + 2 * 4 * _blocks(t) * h + 4 * r * h * d, "flops": 4 * r * t * h * d}
    r, s, topk = case["rows"], case["keys"], min(case["topk"], _blocks(case["keys"]))
    nq, nk = -(-r // QROWS), _blocks(s)
    attended = h * r * min(s, topk * BLOCK)
    kv = 2 * 2 * s * h * d if not case["means"] else 2 * 2 * h * d * min(s, nq * topk * BLOCK) + 4 * nk * h * d
    return {"bytes": kv + 4 * r * h * d + 4 * h * nq * topk, "flops": 4 * attended * d + 2 * nq * nk * h * d}


def _blocks(n):
    return -(-n // BLOCK)


# ---------------------------------------------------------------------------
# inputs


def _rand(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    h, d = case["heads"], case["dim"]
    if case["kind"] == "write":
        start, n = case["start"], case["n"]
        cap = _blocks(start + n) * BLOCK
        # keys carry a few large channels; values are plainer
        k = (_rand(g, n, h, d) * (1 + 3 * _rand(g, 1, h, d).abs())).bfloat16()
        v = _rand(g, n, h, d).bfloat16()
        kq, vq = (torch.randint(-127, 128, (h, cap, d), generator=g, device="cuda", dtype=torch.int8) for _ in "kv")
        ks, vs = (0.01 + 0.04 * torch.rand(h, cap // BLOCK, generator=g, device="cuda") for _ in "kv")
        return {"case": case, "k": k, "v": v, "kq": kq, "vq": vq, "ks": ks, "vs": vs}
    if case["kind"] == "cached":
        t = case["tokens"]
        cap = _blocks(t) * BLOCK
        # codes as a quantiser leaves them: a normal variable whose largest of a block is near 127
        kq, vq = ((_rand(g, h, cap, d) * 32).round_().clamp_(-127, 127).to(torch.int8) for _ in "kv")
        ks, vs = (0.02 + 0.02 * torch.rand(h, cap // BLOCK, generator=g, device="cuda") for _ in "kv")
        return {"case": case, "q": _rand(g, case["rows"], h, d).bfloat16(), "kq": kq, "vq": vq, "ks": ks, "vs": vs}
    r, s = case["rows"], case["keys"]
    # neighbouring tokens are alike, which is what a block's mean stands for
    k = _rand(g, s, h, d)
    k.add_(0.5 * _rand(g, _blocks(s), h, d).repeat_interleave(BLOCK, 0)[:s])
    q = _rand(g, r, h, d)
    q.add_(0.5 * _rand(g, -(-r // QROWS), h, d).repeat_interleave(QROWS, 0)[:r])
    k, q, v = k.bfloat16(), q.bfloat16(), _rand(g, s, h, d).bfloat16()
    return {"case": case, "q": q, "k": k, "v": v, "km": _means(k, BLOCK) if case["means"] else None}


# ---------------------------------------------------------------------------
# one pass


def run(state):
    case = state["case"]
    if case["kind"] == "write":
        start, n = case["start"], case["n"]
        lo = start // BLOCK * BLOCK
        if own:
            cache = _h3b().KV8Cache.wrap(state["kq"], state["vq"], state["ks"], state["vs"], start)
            cache.write(state["k"], state["v"])
            k, v = cache.read(lo)
        else:
            k = _write(state["k"], state["kq"], state["ks"], start)
            v = _write(state["v"], state["vq"], state["vs"], start)
        b0, b1 = lo // BLOCK, _blocks(start + n)
        return {"k": k, "v": v, "ks": state["ks"][:, b0:b1], "vs": state["vs"][:, b0:b1]}
    if case["kind"] == "cached":
        if own:
            h3b = _h3b()
            cache = h3b.KV8Cache.wrap(state["kq"], state["vq"], state["ks"], state["vs"], case["tokens"])
            return h3b.kv8_attention(state["q"], cache)
        return _cached(state["q"], state["kq"], state["vq"], state["ks"], state["vs"], case["tokens"])
    if own:
        o, blocks = _h3b().sparse_attention(state["q"], state["k"], state["v"], case["topk"], k_means=state["km"],
                                            return_blocks=True)
        return {"o": o, "blocks": blocks}
    return _sparse(state["q"], state["k"], state["v"], case["topk"], state["km"])


def _write(x, codes, scales, start):
    """x [n, H, D] quantised into codes [H, cap, D] / scales [H, cap / BLOCK] at `start`; the touched blocks' values."""
    n, h, d = x.shape
    lo = start // BLOCK * BLOCK
    old, b0, nb = start - lo, lo // BLOCK, _blocks(start - lo + n)
    new = torch.zeros(h, nb * BLOCK, d, device=x.device)
    new[:, old:old + n] = x.transpose(0, 1).float()
    s = new.view(h, nb, BLOCK * d).abs().amax(2) / torch.full((1, 1), 127.0, device=x.device)
    had = torch.zeros(h, nb * BLOCK, d, device=x.device)
    if old:
        had[:, :old] = codes[:, lo:start].float()
        before = scales[:, b0].clone()
        s[:, 0] = torch.maximum(s[:, 0], before)
        had[:, :old] = (had[:, :old] * (before / s[:, 0])[:, None, None]).round()
    each = s.repeat_interleave(BLOCK, 1)[:, :, None]
    c = torch.where(each > 0, new / each, torch.zeros_like(new)).round().clamp(-127, 127) + had
    codes[:, lo:start + n] = c[:, :old + n].to(torch.int8)
    scales[:, b0:b0 + nb] = s
    return (c * each)[:, :old + n].transpose(0, 1).bfloat16()


def _cached(q, kq, vq, ks, vs, t):
    if t == 0:
        return torch.zeros_like(q)
    k = kq[:, :t].float() * ks.repeat_interleave(BLOCK, 1)[:, :t, None]
    v = vq[:, :t].float() * vs.repeat_interleave(BLOCK, 1)[:, :t, None]
    s = torch.matmul(q.transpose(0, 1).float() * q.shape[2] ** -0.5, k.transpose(1, 2))
    s.sub_(s.amax(2, keepdim=True)).exp_()
    total = s.sum(2, keepdim=True)
    return (torch.matmul(s, v) / total).transpose(0, 1).bfloat16()


def _means(x, rows):
    """The mean of each block of `rows` rows of x [S, H, D], summed in 64 bits."""
    s, h, d = x.shape
    nb = -(-s // rows)
    pad = torch.zeros(nb * rows, h, d, dtype=x.dtype, device=x.device)
    pad[:s] = x
    count = torch.full((nb, 1, 1), float(rows), dtype=torch.float64, device=x.device)
    count[-1] = s - (nb - 1) * rows
    return (pad.view(nb, rows, h, d).sum(1, dtype=torch.float64) / count).float()


def _sparse(q, k, v, topk, km):
    (r, h, d), s = q.shape, k.shape[0]
    nq, nk = -(-r // QROWS), _blocks(s)
    topk = min(topk, nk)
    qm = _means(q, QROWS).double().transpose(0, 1)
    km = (_means(k, BLOCK) if km is None else km).double().transpose(0, 1)
    # 64 bits: a selection hangs on differences that sums in 32 bits do not hold
    score = torch.matmul(qm, km.transpose(1, 2))
    blocks = score.sort(dim=2, descending=True, stable=True)[1][:, :, :topk].sort(dim=2)[0]  # [H, nq, topk]
    pick = (torch.arange(h, device=q.device)[:, None, None], blocks)

    def gathered(x):
        pad = torch.zeros(nk * BLOCK, h, d, dtype=x.dtype, device=x.device)
        pad[:s] = x
        return pad.view(nk, BLOCK, h, d).permute(2, 0, 1, 3)[pick].reshape(h, nq, topk * BLOCK, d).float()

    qp = torch.zeros(nq * QROWS, h, d, device=q.device)
    qp[:r] = q.float() * d ** -0.5
    p = torch.matmul(qp.view(nq, QROWS, h, d).permute(2, 0, 1, 3), gathered(k).transpose(2, 3))
    at = blocks[..., None] * BLOCK + torch.arange(BLOCK, device=q.device)
    p.masked_fill_((at >= s).reshape(h, nq, 1, topk * BLOCK), -math.inf)
    p.sub_(p.amax(3, keepdim=True)).exp_()
    total = p.sum(3, keepdim=True)
    o = (torch.matmul(p, gathered(v)) / total).permute(1, 2, 0, 3).reshape(nq * QROWS, h, d)[:r].bfloat16()
    return {"o": o, "blocks": blocks.int()}


# ---------------------------------------------------------------------------
# the definitions in 64 bits


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "write":
        start, n, h = case["start"], case["n"], case["heads"]
        out = {}
        for name in "kv":
            x, codes, scales = st[name].double(), st[name + "q"].double(), st[name + "s"].double()
            values, kept = [], []
            for b in range(start // BLOCK, _blocks(start + n)):
                lo, hi = b * BLOCK, min((b + 1) * BLOCK, start + n)
                first = max(lo, start)
                part = x[first - start:hi - start]                        # [m, H, D]
                # scale and quotient are numbers of 32 bits by definition
                s = (part.abs().amax((0, 2)) / 127).float().double()
                have = codes[:, lo:first].transpose(0, 1)
                if first > lo:
                    s = torch.maximum(s, scales[:, b])
                    ratio = (scales[:, b] / s).float().double()
                    have = (have * ratio[None, :, None]).float().double().round()
                per = s[None, :, None]
                c = torch.where(per > 0, (part / per).float().double(), torch.zeros_like(part)).round().clamp(-127, 127)
                values.append(torch.cat([have, c]) * per)
                kept.append(s)
            out[name], out[name + "s"] = torch.cat(values), torch.stack(kept, 1)
        return out
    if case["kind"] == "cached":
        t, d = case["tokens"], case["dim"]
        each = torch.arange(t, device="cuda") // BLOCK
        out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
        for i in range(case["heads"]):
            k = st["kq"][i, :t].double() * st["ks"][i].double()[each, None]
            v = st["vq"][i, :t].double() * st["vs"][i].double()[each, None]
            for j in range(0, case["rows"], 8192):
                s = st["q"][j:j + 8192, i].double() @ k.T / math.sqrt(d)
                out[j:j + 8192, i] = (s - torch.logsumexp(s, 1, keepdim=True)).exp() @ v
        return out
    s, d, r, h = case["keys"], case["dim"], case["rows"], case["heads"]
    nq, nk = -(-r // QROWS), _blocks(s)
    topk = min(case["topk"], nk)
    out = torch.zeros(r, h, d, dtype=torch.float64, device="cuda")

    def pooled(x, rows):  # a mean is a number of 32 bits by definition
        where = torch.arange(x.shape[0], device="cuda") // rows
        total = torch.zeros(int(where[-1]) + 1, d, dtype=torch.float64, device="cuda").index_add_(0, where, x)
        return (total / torch.bincount(where)[:, None].double()).float().double()

    lane = torch.arange(BLOCK, device="cuda")
    for i in range(h):
        q, k, v = (st[name][:, i].double() for name in "qkv")
        km = pooled(k, BLOCK) if st["km"] is None else st["km"][:, i].double()
        chosen = torch.topk(pooled(q, QROWS) @ km.T, topk, dim=1)[1]     # [nq, topk]
        for j in range(0, nq, 128):
            keys = (chosen[j:j + 128, :, None] * BLOCK + lane).flatten(1)  # [m, topk * BLOCK]
            kg, vg = k[keys.clamp(max=s - 1)], v[keys.clamp(max=s - 1)]
            qp = torch.zeros(keys.shape[0] * QROWS, d, dtype=torch.float64, device="cuda")
            part = q[j * QROWS:(j + 128) * QROWS]
            qp[:part.shape[0]] = part
            a = torch.einsum("mrd,mcd->mrc", qp.view(-1, QROWS, d), kg) / math.sqrt(d)
            a = torch.where((keys < s)[:, None], a, torch.full_like(a, -math.inf)).softmax(2)
            out[j * QROWS:j * QROWS + part.shape[0], i] = (a @ vg).reshape(-1, d)[:part.shape[0]]
    return {"o": out, "blocks": None}
