"""The 8-bit key/value cache and block-sparse attention on the GPU, against plain 64-bit restatements."""
import pytest
import torch

from attn_oracle import means, quantise, select, softmax_rows, sparse, tolerance
from gpu_util import gen

pytestmark = pytest.mark.gpu

h3b = pytest.importorskip("h3b")
from h3b import model as hm  # noqa: E402

DEV = torch.device("cuda", 0)
INF, NAN = float("inf"), float("nan")


def randn(*shape, seed, scale=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, generator=gen(seed)) * scale).to(dtype).to(DEV)


def same(a, b):
    return torch.equal(a.cpu(), b.cpu())


def near(got, o, a, m, n, d, vsum=0.0):
    over = (got.double() - o).abs() - tolerance(o, a, m, n, d, vsum)
    assert torch.isfinite(got).all()
    assert over.max().item() <= 0, f"off by {(got.double() - o).abs().max().item():.3g}, {over.max().item():.3g} over the bound"


# ---------------------------------------------------------------------------
# the cache


def filled(H, cap, D, length, seed, spread=0.0):
    """A cache of random codes and scales, poisoned behind `length`: codes of 127 and NaN scales of the blocks there."""
    g = gen(seed)
    nb = cap // 64
    kq, vq = (torch.randint(-127, 128, (H, cap, D), generator=g, dtype=torch.int8) for _ in "kv")
    ks, vs = ((0.01 + 0.02 * torch.rand(H, nb, generator=g)) * torch.exp(spread * torch.randn(H, nb, generator=g))
              for _ in "kv")
    for c, s in ((kq, ks), (vq, vs)):
        c[:, length:] = 127
        s[:, -(-length // 64):] = NAN
    return h3b.KV8Cache.wrap(kq.to(DEV), vq.to(DEV), ks.to(DEV), vs.to(DEV), length)


def values(cache):
    n = cache.length
    return [(c[:, :n].double() * s.double().repeat_interleave(64, 1)[:, :n, None]).transpose(0, 1)
            for c, s in ((cache.kq, cache.ks), (cache.vq, cache.vs))]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,start,n", [(1, 0, 1), (3, 0, 64), (2, 63, 1), (2, 64, 1), (5, 17, 300), (1, 100, 27),
                                       (40, 1000, 1), (2, 5, 59), (2, 5, 60), (3, 0, 1025)])
def test_write_matches_the_definition(D, H, start, n):
    cap = -(-(start + n) // 64) * 64 + 64
    c = filled(H, cap, D, start, seed=n)
    k = randn(n, H, D, seed=1) * torch.logspace(-3, 3, n, dtype=torch.float32)[:, None, None].to(DEV).bfloat16()
    v = randn(n, H, D, seed=2, scale=0.1)  # smaller than the staying scale: a partial block keeps it
    want = [quantise(x, q, s, start) for x, q, s in ((k, c.kq, c.ks), (v, c.vq, c.vs))]
    assert c.write(k, v) is c and c.length == start + n
    for (q, s), gq, gs in zip(want, (c.kq, c.vq), (c.ks, c.vs)):
        assert same(q, gq) and torch.equal(torch.nan_to_num(s, -1.0), torch.nan_to_num(gs.cpu(), -1.0))
    # reading back, in both types, whole and from the middle of a block
    kd, vd = values(c)
    for dtype in (torch.float32, torch.bfloat16):
        for lo, hi in ((0, c.length), (start, start + n), (start + n - 1, start + n), (start, start)):
            gk, gv = c.read(lo, hi, dtype)
            assert gk.shape == (hi - lo, H, D) and gk.dtype == dtype
            assert same(gk, kd[lo:hi].float().to(dtype)) and same(gv, vd[lo:hi].float().to(dtype))


def test_written_values_lie_within_half_a_step():
    k = randn(500, 4, 128, seed=3)
    c = h3b.KV8Cache(500, 4, 128, DEV).write(k, -k)
    gk, gv = c.read(dtype=torch.float32)
    step = c.ks.repeat_interleave(64, 1)[:, :500].T[:, :, None]
    # half a step of the code, and fp32 roundings of the scale, the quotient and the product at 127 steps
    assert ((gk - k.float()).abs() <= step * (0.5 + 3 * 127 * 2.0 ** -24)).all()
    assert same(gv, -gk)


def test_write_token_by_token_rewind_and_no_tokens():
    k, v = randn(130, 2, 128, seed=5), randn(130, 2, 128, seed=6)
    c = h3b.KV8Cache(130, 2, 128, DEV)
    assert c.capacity == 192
    kq, ks, vq, vs = (t.clone() for t in (c.kq, c.ks, c.vq, c.vs))
    for t in range(130):
        kq, ks = quantise(k[t:t + 1], kq, ks, t)
        vq, vs = quantise(v[t:t + 1], vq, vs, t)
        c.write(k[t:t + 1], v[t:t + 1])
    for a, b in ((c.kq, kq), (c.vq, vq)):
        assert same(a[:, :130], b[:, :130])
    assert same(c.ks, ks) and same(c.vs, vs)
    assert c.write(k[:0], v[:0]).length == 130
    kq, ks = quantise(v[:7], c.kq, c.ks, 70)
    assert c.write(v[:7], k[:7], start=70).length == 77  # the tokens behind 70 are dropped
    assert same(c.kq[:, :77], kq[:, :77]) and same(c.ks, ks)
    assert c.write(v[:0], k[:0], start=0).length == 0
    assert c.read()[0].shape == (0, 2, 128)


def test_zero_blocks_and_non_finite_tokens():
    k = torch.zeros(192, 2, 64, dtype=torch.bfloat16, device=DEV)
    v = randn(192, 2, 64, seed=7)
    v[70, 0, 3], v[150, 1, 0] = INF, NAN
    c = h3b.KV8Cache(192, 2, 64, DEV).write(k, v)
    gk, gv = c.read()
    assert (gk == 0).all() and (c.ks == 0).all()
    bad = torch.zeros(192, 2, dtype=torch.bool, device=DEV)
    bad[64:128, 0], bad[128:, 1] = True, True
    assert torch.isnan(gv[bad]).all() and torch.isfinite(gv[~bad]).all()
    # a block made non-finite by a later token loses its older ones too, and a rewrite from its start mends it
    c = h3b.KV8Cache(64, 2, 64, DEV).write(v[:10], v[:10]).write(v[70:71], v[70:71])
    assert torch.isnan(c.read()[0][:, 0]).all() and torch.isfinite(c.read()[0][:, 1]).all()
    assert torch.isfinite(c.write(v[:10], v[:10], start=0).read()[0]).all()
    # a scale of zero grows with the first value
    c = h3b.KV8Cache(64, 2, 64, DEV).write(k[:5], k[:5]).write(v[:5], v[:5])
    assert (c.read()[0][:5] == 0).all() and (c.read()[0][5:].abs().amax((0, 2)) > 0).all()


def test_write_of_strided_views():
    qkv = randn(200, 3 * 256, seed=8)
    k, v = qkv[:, 256:512].view(200, 2, 128), qkv[:, 512:].view(200, 2, 128)
    a = h3b.KV8Cache(200, 2, 128, DEV).write(k, v)
    b = h3b.KV8Cache(200, 2, 128, DEV).write(k.contiguous(), v.contiguous())
    t = h3b.KV8Cache(200, 2, 128, DEV).write(k.transpose(0, 1).contiguous().transpose(0, 1), v)
    for x in (a, t):
        assert same(x.kq[:, :200], b.kq[:, :200]) and same(x.vq[:, :200], b.vq[:, :200]) and same(x.ks, b.ks)


# ---------------------------------------------------------------------------
# attention over the cache


def check_cached(q, c, scale=None):
    got = h3b.kv8_attention(q, c, scale)
    assert got.shape == q.shape and got.is_contiguous()
    d = q.shape[2]
    k, v = values(c)
    for h in range(q.shape[1]):
        o, a, m = softmax_rows(q[:, h], k[:, h], v[:, h], d ** -0.5 if scale is None else scale)
        near(got[:, h], o, a, m, c.length, d, v[:, h].abs().sum(0))
    return got


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rows,tokens,H", [(1, 1, 1), (1, 63, 2), (1, 64, 3), (1, 65, 40), (1, 5000, 3), (2, 127, 2),
                                           (7, 129, 1), (16, 300, 2), (17, 300, 2), (64, 64, 2), (127, 128, 1),
                                           (128, 191, 2), (129, 257, 3), (300, 512, 4), (1000, 77, 2), (511, 1000, 5)])
def test_cached_attention(D, rows, tokens, H):
    check_cached(randn(rows, H, D, seed=rows + tokens), filled(H, -(-tokens // 64) * 64 + 128, D, tokens, seed=tokens))


@pytest.mark.parametrize("rows", [1, 20, 150])
def test_cached_attention_over_wide_scales_and_scores(rows):
    """Scales that differ by e^±6 between blocks, and scores in the hundreds: a softmax near a single key."""
    c = filled(3, 640, 128, 600, seed=9, spread=2.0)
    check_cached(randn(rows, 3, 128, seed=10), c)
    check_cached(randn(rows, 3, 128, seed=11, scale=8.0), c, scale=0.5)
    check_cached(randn(rows, 3, 128, seed=12), c, scale=0.0)
    check_cached(randn(rows, 3, 128, seed=13), c, scale=-0.3)


@pytest.mark.parametrize("rows", [1, 16, 40, 200])
def test_cached_attention_rising_maximum(rows):
    """Keys whose scores rise all along the cache, so the running maximum moves in every tile."""
    D, n = 128, 1000
    c = filled(1, 1024, D, n, seed=14)
    c.kq.zero_()
    c.kq[:, :, 0] = 127
    c.ks[0, :16] = torch.linspace(0.01, 2.0, 16, device=DEV)
    q = torch.zeros(rows, 1, D, dtype=torch.bfloat16, device=DEV)
    q[:, 0, 0] = torch.linspace(-4, 4, rows, device=DEV).bfloat16() if rows > 1 else 3.0
    check_cached(q, c)


def test_cached_attention_empty_and_no_rows():
    c = filled(2, 64, 64, 0, seed=15)
    for rows in (0, 1, 200):
        got = h3b.kv8_attention(randn(rows, 2, 64, seed=16), c)
        assert got.shape == (rows, 2, 64) and (got == 0).all()


@pytest.mark.parametrize("rows", [1, 200])
def test_cached_attention_non_finite_blocks_stay_in_their_head(rows):
    x = randn(200, 3, 128, seed=17)
    bad = x.clone()
    bad[100, 1, 5] = INF
    q = randn(rows, 3, 128, seed=18)
    good = h3b.kv8_attention(q, h3b.KV8Cache(200, 3, 128, DEV).write(x, x))
    for k, v in ((bad, x), (x, bad)):
        got = h3b.kv8_attention(q, h3b.KV8Cache(200, 3, 128, DEV).write(k, v))
        assert torch.isnan(got[:, 1]).all() and same(got[:, ::2], good[:, ::2])
    qn = q.clone()
    qn[rows - 1, 0, 0] = NAN
    got = h3b.kv8_attention(qn, h3b.KV8Cache(200, 3, 128, DEV).write(x, x))
    assert torch.isnan(got[rows - 1, 0]).all() and same(got[:rows - 1], good[:rows - 1]) and same(got[:, 1:], good[:, 1:])


@pytest.mark.parametrize("rows", [1, 300])
def test_cached_attention_of_strided_queries(rows):
    c = filled(4, 320, 128, 300, seed=19)
    wide = randn(rows, 3 * 512, seed=20)
    q = wide[:, 512:1024].view(rows, 4, 128)
    assert same(h3b.kv8_attention(q, c), h3b.kv8_attention(q.contiguous(), c))
    t = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert same(h3b.kv8_attention(t, c), h3b.kv8_attention(q.contiguous(), c))


def test_long_cache_offsets_pass_32_bits():
    """A cache whose last head's codes lie behind 2^32 bytes: 40 heads, 860000 tokens (4.4 GB of codes each)."""
    H, n, D = 40, 860000, 128
    g = torch.Generator(device=DEV).manual_seed(21)
    c = h3b.KV8Cache(n, H, D, DEV)
    for t in (c.kq, c.vq):
        t.random_(-127, 128, generator=g)
    c.ks.fill_(0.02)
    c.vs.fill_(0.02)
    c.length = n - 3
    assert c.kq.numel() > 2 ** 32
    last = randn(3, H, D, seed=22)
    want, scale = quantise(last, c.kq[:, -64:], c.ks[:, -1:], 29)  # token 859997 is the 29th of the last block
    c.write(last, last)
    gk, gv = c.read(n - 3, n, torch.float32)
    k, v = (x[:, -64:].double() * s[:, -1].double()[:, None, None] for x, s in ((c.kq, c.ks), (c.vq, c.vs)))
    assert same(gk, k[:, 29:32].transpose(0, 1).float()) and same(gv, v[:, 29:32].transpose(0, 1).float())
    assert same(c.kq[:, -35:-32], want[:, 29:32]) and same(c.ks[:, -1:], scale)
    q = randn(2, H, D, seed=23)
    got = h3b.kv8_attention(q, c)
    for h in (0, H - 1):
        k, v = (x[h, :n].double() * s[h].double().repeat_interleave(64)[:n, None] for x, s in ((c.kq, c.ks), (c.vq, c.vs)))
        o, a, m = softmax_rows(q[:, h], k, v, D ** -0.5)
        near(got[:, h], o, a, m, n, D, v.abs().sum(0))
    del c, k, v
    torch.cuda.empty_cache()


# ---------------------------------------------------------------------------
# selection


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,H,rows", [(1, 1, 64), (63, 2, 64), (64, 3, 64), (65, 2, 128), (1000, 5, 64), (1000, 5, 128)])
def test_block_means(D, n, H, rows):
    x = randn(n, H, D, seed=n) * torch.logspace(-4, 4, n, dtype=torch.float32)[:, None, None].to(DEV).bfloat16()
    assert same(h3b.block_means(x, rows), means(x, rows))
    wide = torch.cat([x, x], 2).view(n, 2 * H, D)[:, ::2]
    assert same(h3b.block_means(wide, rows), means(wide, rows))
    if n > rows:
        out = means(x, rows).to(DEV)
        want = out.clone()
        out[1:] = 0
        h3b.block_means(x[rows:], rows, out=out[1:])
        assert same(out, want)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("nq,nk,H", [(1, 1, 1), (1, 257, 5), (3, 64, 2), (70, 65, 3), (129, 300, 2), (2, 5000, 1)])
def test_select_blocks(D, nq, nk, H):
    qm, km = randn(nq, H, D, seed=1, dtype=torch.float32), randn(nk, H, D, seed=2, dtype=torch.float32)
    for topk in sorted({0, 1, min(7, nk), nk // 2, nk}):
        got = h3b.select_blocks(qm, km, topk)
        assert got.shape == (H, nq, topk) and same(got, select(qm, km, topk))
    assert h3b.select_blocks(qm, km, nk + 5).shape == (H, nq, nk)


def test_select_blocks_ties_zeros_and_non_numbers():
    km = torch.zeros(300, 2, 64, device=DEV)
    qm = randn(5, 2, 64, seed=3, dtype=torch.float32)
    assert same(h3b.select_blocks(qm, km, 9), torch.arange(9, dtype=torch.int32).expand(2, 5, 9))
    km[:] = -0.0
    km[::2] = 0.0  # products of -0 and +0: equal
    assert same(h3b.select_blocks(qm, km, 9), torch.arange(9, dtype=torch.int32).expand(2, 5, 9))
    km = randn(40, 2, 64, seed=4, dtype=torch.float32)[torch.arange(300, device=DEV) % 40].contiguous()  # each 7 or 8 times
    for topk in (1, 7, 8, 9, 100):
        assert same(h3b.select_blocks(qm, km, topk), select(qm, km, topk))
    km[11], km[200] = NAN, INF
    assert same(h3b.select_blocks(qm, km, 299), select(qm, km, 299))
    qm[2] = NAN
    assert same(h3b.select_blocks(qm, km, 3)[:, 2], torch.arange(3, dtype=torch.int32).expand(2, 3))


def test_select_blocks_in_several_rounds():
    """A selection whose scores pass through the workspace in more than one round."""
    nq, nk, H = 1500, 9000, 3
    qm, km = randn(nq, H, 64, seed=5, dtype=torch.float32), randn(nk, H, 64, seed=6, dtype=torch.float32)
    assert nq * nk * H * 8 > h3b.lib.h3b_select_blocks_workspace(nq, nk, H) > 0
    assert same(h3b.select_blocks(qm, km, 50), select(qm, km, 50))


# ---------------------------------------------------------------------------
# block-sparse attention


def check_sparse(q, k, v, blocks, scale=None):
    d = q.shape[2]
    got = h3b.block_sparse_attention(q, k, v, blocks, scale)
    assert got.shape == q.shape and got.is_contiguous()
    o, a, m = sparse(q, k, v, blocks, d ** -0.5 if scale is None else scale)
    near(got, o, a, m, blocks.shape[2] * 64, d)
    return got


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rows,keys,H,topk", [(1, 1, 1, 1), (1, 1000, 4, 3), (3, 64, 2, 1), (128, 128, 2, 2), (129, 65, 3, 2),
                                              (300, 1000, 3, 5), (1000, 1000, 2, 16), (1, 9000, 2, 130), (260, 640, 40, 4)])
def test_sparse_attention(D, rows, keys, H, topk):
    q, k, v = randn(rows, H, D, seed=1), randn(keys, H, D, seed=2), randn(keys, H, D, seed=3)
    topk = min(topk, -(-keys // 64))
    o, blocks = h3b.sparse_attention(q, k, v, topk, return_blocks=True)
    assert same(blocks, select(means(q, 128), means(k, 64), topk))
    assert same(o, check_sparse(q, k, v, blocks))
    assert same(o, h3b.sparse_attention(q, k, v, topk, k_means=h3b.block_means(k)))


def test_sparse_attention_over_all_blocks_is_attention():
    q, k, v = (randn(333, 3, 128, seed=s) for s in (4, 5, 6))
    got = h3b.sparse_attention(q, k, v, 99)
    for h in range(3):
        o, a, m = softmax_rows(q[:, h], k[:, h], v[:, h], 128 ** -0.5)
        near(got[:, h], o, a, m, 333, 128)


@pytest.mark.parametrize("rows", [1, 500])
def test_sparse_attention_lists_with_gaps_repeats_and_bad_indices(rows):
    H, D, keys = 3, 128, 1000
    q, k, v = randn(rows, H, D, seed=7), randn(keys, H, D, seed=8), randn(keys, H, D, seed=9)
    nq = -(-rows // 128)
    blocks = torch.randint(-1, 16, (H, nq, 9), generator=gen(10)).int()
    blocks[0, 0] = -1                                                # rows without a key
    blocks[1, 0] = torch.tensor([15, -1, -1, 15, 3, 3, 3, -1, 0])    # repeats, the short last block among them
    check_sparse(q, k, v, blocks.to(DEV))
    assert (h3b.block_sparse_attention(q, k, v, blocks.to(DEV))[:128, 0] == 0).all()
    assert h3b.status() == 0
    wrong = blocks.clone()
    wrong[2, 0, :3] = torch.tensor([16, -2, 2 ** 31 - 1])
    clean = wrong.clone()
    clean[2, 0, :3] = -1
    assert same(h3b.block_sparse_attention(q, k, v, wrong.to(DEV)), h3b.block_sparse_attention(q, k, v, clean.to(DEV)))
    assert h3b.status() == 3
    h3b.clear_status()


def test_sparse_attention_without_keys_or_lists():
    q, k = randn(200, 2, 64, seed=11), randn(0, 2, 64, seed=12)
    o, blocks = h3b.sparse_attention(q, k, k, 4, return_blocks=True)
    assert blocks.shape == (2, 2, 0) and (o == 0).all()
    k = randn(100, 2, 64, seed=13)
    assert (h3b.sparse_attention(q, k, k, 0) == 0).all()
    assert h3b.sparse_attention(q[:0], k, k, 1).shape == (0, 2, 64)


@pytest.mark.parametrize("rows", [1, 300])
def test_sparse_attention_reads_nothing_else(rows):
    """NaN and infinities in the keys and values of blocks that are not selected, and behind the last key, stay out."""
    H, D, keys = 2, 128, 500
    kbig, vbig = randn(keys + 200, H, D, seed=14), randn(keys + 200, H, D, seed=15)
    q = randn(rows, H, D, seed=16)
    blocks = torch.tensor([1, 4, 7], dtype=torch.int32, device=DEV).expand(H, -(-rows // 128), 3).contiguous()
    want = check_sparse(q, kbig[:keys], vbig[:keys], blocks)
    out = torch.ones(keys + 200, dtype=torch.bool, device=DEV)
    for b in (1, 4, 7):
        out[b * 64:min((b + 1) * 64, keys)] = False
    kbig[out], vbig[out] = NAN, INF
    assert same(h3b.block_sparse_attention(q, kbig[:keys], vbig[:keys], blocks), want)


def test_sparse_attention_of_strided_views():
    rows, H, D = 300, 4, 128
    qkv = randn(rows, 3 * H * D, seed=17)
    q, k, v = (qkv[:, i * H * D:(i + 1) * H * D].view(rows, H, D) for i in range(3))
    want = h3b.sparse_attention(*(t.contiguous() for t in (q, k, v)), 3)
    assert same(h3b.sparse_attention(q, k, v, 3), want)
    q, k, v = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v))
    assert same(h3b.sparse_attention(q, k, v, 3), want)


# ---------------------------------------------------------------------------
# refusals, streams, graphs, the model


def test_refusals():
    q = randn(4, 2, 128, seed=1)
    c = filled(2, 128, 128, 100, seed=2)
    cases = [lambda: h3b.kv8_attention(q.float(), c), lambda: h3b.kv8_attention(q[:, :1], c),
             lambda: h3b.kv8_attention(q[..., :64], c), lambda: h3b.kv8_attention(q[0], c),
             lambda: h3b.kv8_attention(q.transpose(1, 2).contiguous().transpose(1, 2), c),
             lambda: h3b.kv8_attention(q[:, :1].expand(4, 2, 128), c),
             lambda: c.write(q, q, start=101), lambda: c.write(q, q[:3]), lambda: c.write(q, q, start=-1),
             lambda: c.write(randn(29, 2, 128, seed=3), randn(29, 2, 128, seed=3)),
             lambda: c.read(0, 101), lambda: c.read(5, 4), lambda: c.read(dtype=torch.float16),
             lambda: h3b.block_means(q, 32), lambda: h3b.block_means(q, out=torch.zeros(1, 2, 64, device=DEV)),
             lambda: h3b.select_blocks(q.float(), q.float()[:, :1].contiguous(), 1),
             lambda: h3b.select_blocks(q, q, 1), lambda: h3b.select_blocks(q.float(), q.float(), -1),
             lambda: h3b.sparse_attention(q, q, q[:3], 1),
             lambda: h3b.sparse_attention(q, q, q, 1, k_means=torch.zeros(2, 2, 128, device=DEV)),
             lambda: h3b.block_sparse_attention(q, q, q, torch.zeros(2, 2, 1, dtype=torch.int32, device=DEV)),
             lambda: h3b.block_sparse_attention(q, q, q, torch.zeros(2, 1, 1, dtype=torch.int64, device=DEV))]
    for i, call in enumerate(cases):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"case {i} was taken")
    assert c.length == 100
    with pytest.raises(TypeError):
        h3b.kv8_attention(q.cpu(), c)


def test_side_streams_run_side_by_side():
    """The same operators on two streams at once, each with its own workspaces, equal to one after the other."""
    q, k, v = (randn(700, 4, 128, seed=s) for s in (1, 2, 3))
    c = filled(4, 4096, 128, 4000, seed=4)
    one = randn(1, 4, 128, seed=5)
    want = [h3b.sparse_attention(q, k, v, 4), h3b.kv8_attention(q, c), h3b.kv8_attention(one, c),
            h3b.sparse_attention(one, k, v, 8)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                got.append([h3b.sparse_attention(q, k, v, 4), h3b.kv8_attention(q, c), h3b.kv8_attention(one, c),
                            h3b.sparse_attention(one, k, v, 8)])
    torch.cuda.synchronize()
    for g in got:
        assert all(same(a, b) for a, b in zip(g, want))


def test_captured_graphs_share_a_pool_and_follow_their_inputs():
    c = filled(4, 2048, 128, 2000, seed=6)
    kv = randn(40, 4, 128, seed=7)
    q, k, v = (randn(300, 4, 128, seed=s) for s in (8, 9, 10))
    one = randn(1, 4, 128, seed=11)

    def first():
        c.write(kv, kv, start=1990)
        return h3b.kv8_attention(one, c), h3b.kv8_attention(q, c)

    def second():
        return h3b.sparse_attention(q, k, v, 3), h3b.sparse_attention(one, k, v, 3)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        first(), second()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for f in (first, second):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0].pool() if graphs else None, stream=side):
            outs.append(f())
        graphs.append(g)
    for seed in (20, 30):
        for t, s in ((q, 0), (k, 1), (v, 2), (one, 3), (kv, 4)):
            t.copy_(randn(*t.shape, seed=seed + s))
        for order in ((0, 1), (1, 0)):
            c.length = 2000
            kept = c.kq.clone(), c.ks.clone()
            want = [first(), second()]
            c.kq.copy_(kept[0]), c.ks.copy_(kept[1])
            c.length = 2030
            for i in order:
                graphs[i].replay()
                torch.cuda.synchronize()
                assert all(same(a, b) for a, b in zip(outs[i], want[i]))


def test_model_with_text_cache_and_sparse_attention():
    """Two blocks over cached text equal the same blocks given the values that the cache stands for, and selecting
    every block equals dense attention, both to the rounding of attention outputs (which the INT8 linears behind it
    turn into code steps: the comparison is of the whole output's norm).  Each branch that is not asked for is bitwise
    what it was."""
    cfg = hm.DiTConfig(dim=512, heads=4, head_dim=128, ffn=1024, n_blocks=2, text_len=77)
    dit = hm.SynthDiT(cfg, DEV, seed=3)
    S = 700
    x, text = randn(S, 512, seed=1), randn(77, 512, seed=2)
    ridx = torch.zeros(S, dtype=torch.int32, device=DEV)
    plain = dit.forward(x.clone(), ridx, None, text)
    caches = dit.text_cache(text)
    assert [c.length for c in caches] == [77, 77]
    y = dit.forward(x.clone(), ridx, None, caches)
    assert same(y, dit.forward(x.clone(), ridx, None, caches))

    def with_values(p, cache):
        def cross(cfg_, p_, hq, text_):
            q = hm._lin_q(hq, p_.cq).view(S, 4, 128)
            k, v = cache.read(dtype=torch.float32)
            o = torch.softmax(torch.einsum("qhd,khd->hqk", q.float(), k) * 128 ** -0.5, 2)
            return hm._lin(torch.einsum("hqk,khd->qhd", o, v).bfloat16().reshape(S, 512), p_.cout)
        return cross
    ref = x.clone()
    keep = hm.cross_attention
    try:
        for p, c in zip(dit.params, caches):
            hm.cross_attention = with_values(p, c)
            ref = hm.block_forward(cfg, p, ref, ridx, None, text)
    finally:
        hm.cross_attention = keep
    rel = lambda a, b: ((a.float() - b.float()).norm() / b.float().norm()).item()  # noqa: E731
    # attention outputs within a bf16 step move int8 codes by at most one of 127: a few parts in a thousand here
    assert rel(y, ref) < 0.01
    assert rel(y, plain) < 0.05  # 8-bit keys and values
    with pytest.raises(ValueError):
        dit.forward(x.clone(), ridx, None, caches[:1])
    dense = hm.SynthDiT(cfg, DEV, seed=3)
    dense.cfg = hm.DiTConfig(**{**cfg.__dict__, "attn_topk": 11})
    assert rel(dense.forward(x.clone(), ridx, None, text), plain) < 0.01
    dense.cfg = hm.DiTConfig(**{**cfg.__dict__, "attn_topk": 3})
    y = dense.forward(x.clone(), ridx, None, caches)
    assert torch.isfinite(y).all() and not same(y, plain)
    assert h3b.status() == 0


@pytest.mark.parametrize("rows,tokens,H", [(300, 70, 40), (900, 200, 40), (16000 // 8 - 40, 512, 40), (130, 1500, 150)])
def test_cached_attention_with_an_odd_number_of_tiles_over_many_items(rows, tokens, H):
    """More pairs of row tiles than SMs, and a head's last pair with one tile only: CTAs that go from item to item."""
    c = filled(H, -(-tokens // 64) * 64, 128, tokens, seed=rows)
    q = randn(rows, H, 128, seed=tokens)
    got = h3b.kv8_attention(q, c)
    k, v = values(c)
    for h in (0, 1, H // 2, H - 1):
        o, a, m = softmax_rows(q[:, h], k[:, h], v[:, h], 128 ** -0.5)
        near(got[:, h], o, a, m, tokens, 128)
    assert same(got[:, ::7], h3b.kv8_attention(q, c)[:, ::7])
    assert h3b.status() == 0


@pytest.mark.parametrize("rows,H", [(129, 150), (640, 40), (385, 149)])
def test_sparse_attention_over_many_items(rows, H):
    q, k, v = randn(rows, H, 64, seed=1), randn(400, H, 64, seed=2), randn(400, H, 64, seed=3)
    o, blocks = h3b.sparse_attention(q, k, v, 3, return_blocks=True)
    heads = [0, H // 3, H - 1]
    ref, a, m = sparse(q[:, heads], k[:, heads], v[:, heads], blocks[heads], 64 ** -0.5)
    near(o[:, heads], ref, a, m, 192, 64)
    assert h3b.status() == 0


def test_cached_attention_widens_its_heads_in_groups():
    """Codes of 9 heads that widen to 645 MB, in launches of 5 and 4: more than the workspace takes at a time."""
    H, n, D, rows = 9, 140000, 128, 70
    c = filled(H, -(-n // 64) * 64, D, n, seed=31)
    assert 2 * n * D * 2 * H > 512 << 20
    q = randn(rows, H, D, seed=32)
    got = h3b.kv8_attention(q, c)
    k, v = values(c)
    for h in range(H):
        o, a, m = softmax_rows(q[:, h], k[:, h], v[:, h], D ** -0.5)
        near(got[:, h], o, a, m, n, D)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rows,H,topk", [(300, 3, 40), (128, 1, 70), (513, 60, 30)])
def test_sparse_attention_over_long_lists(D, rows, H, topk):
    """Items of 24 steps or more, whose tiles' exponentials take turns, with and without a tile at the end that has no
    partner."""
    q, k, v = randn(rows, H, D, seed=1), randn(5000, H, D, seed=2), randn(5000, H, D, seed=3)
    o, blocks = h3b.sparse_attention(q, k, v, topk, return_blocks=True)
    heads = sorted({0, H // 2, H - 1})
    ref, a, m = sparse(q[:, heads], k[:, heads], v[:, heads], blocks[heads], D ** -0.5)
    near(o[:, heads], ref, a, m, topk * 64, D)
    assert h3b.status() == 0


@pytest.mark.parametrize("rows,tokens,H", [(16000, 512, 4), (1000, 64, 40), (700, 4000, 7), (200, 129, 3)])
def test_repeated_calls_are_bitwise_equal(rows, tokens, H):
    """Nothing depends on which of the kernel's warps comes first: fifty runs, other work on another stream meanwhile."""
    c = filled(H, -(-tokens // 64) * 64, 128, tokens, seed=41)
    q = randn(rows, H, 128, seed=42)
    want = h3b.kv8_attention(q, c)
    sq = h3b.sparse_attention(q, q, q, 5)
    side = torch.cuda.Stream()
    a = randn(2048, 2048, seed=43)
    torch.cuda.synchronize()
    for _ in range(50):
        with torch.cuda.stream(side):
            a @ a
        assert torch.equal(h3b.kv8_attention(q, c), want) and torch.equal(h3b.sparse_attention(q, q, q, 5), sq)
    assert h3b.status() == 0


@pytest.mark.parametrize("rows", [8, 9, 64, 65])
@pytest.mark.parametrize("tokens", [200, 3000])
def test_cached_attention_where_the_kernels_change(rows, tokens):
    """Row counts on both sides of each choice of kernel: a row's output does not depend on it beyond its rounding."""
    c = filled(3, -(-tokens // 64) * 64, 128, tokens, seed=rows)
    check_cached(randn(rows, 3, 128, seed=tokens), c)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rows", [1, 20, 300])
def test_cached_attention_over_negative_scales(D, rows):
    """Scales of a wrapped cache may be of either sign, and zero."""
    c = filled(3, 704, D, 650, seed=51)
    sign = torch.tensor([1.0, -1.0, -1.0, 0.0, 1.0, -1.0, 1.0, 1.0, -1.0, 0.0, -1.0], device=DEV)
    c.ks.mul_(sign)
    c.vs.mul_(sign.flip(0))
    check_cached(randn(rows, 3, D, seed=52, scale=4.0), c)
    check_cached(randn(rows, 3, D, seed=53, scale=4.0), c, scale=-0.2)


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
@pytest.mark.parametrize("rows,topk", [(1, 3), (300, 3), (300, 40)])
def test_sparse_attention_of_other_scales(rows, topk, scale):
    q, k, v = randn(rows, 3, 128, seed=54), randn(2700, 3, 128, seed=55), randn(2700, 3, 128, seed=56)
    blocks = h3b.select_blocks(h3b.block_means(q, 128), h3b.block_means(k), topk)
    check_sparse(q, k, v, blocks, scale)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rows", [65, 300])
def test_cached_attention_to_a_single_token_rounds_once(D, rows):
    """p and its sum are 1 up to 2^-24 of a score's reference (below 2^6 here), so the output is the token's value
    rounded to bf16: half a step and less than 2^-16 beside it."""
    c = filled(5, 64, D, 1, seed=61)
    got = h3b.kv8_attention(randn(rows, 5, D, seed=62), c).double()
    want = values(c)[1].expand(rows, -1, -1)
    assert ((got - want).abs() <= 2.0 ** -8 * (1 + 2.0 ** -8) * want.abs()).all()


def items_of_a_head(rows):
    """Pairs of row tiles of a head; the last has one tile only if the tiles are odd."""
    return -(-rows // 256)


def takes_a_single_tile_before_a_pair(rows, tokens, H, D):
    """A CTA goes from an item with one tile to an item with both, and writes both to o itself (nothing is split)."""
    each, sms = items_of_a_head(rows), torch.cuda.get_device_properties(DEV).multi_processor_count
    whole = h3b.lib.h3b_attn_workspace(1, rows, H, D, -(-tokens // 64)) == 4 * H * -(-tokens // 64) * 64 * D
    single = [i % each == each - 1 for i in range(each * H)]
    return whole and -(-rows // 128) % 2 == 1 and any(a and not b for a, b in zip(single, single[sms:]))


@pytest.mark.parametrize("tokens", [64, 77, 100, 128, 192, 256, 320])
@pytest.mark.parametrize("rows,H,D", [(16000, 40, 128), (4128, 40, 128), (8000, 40, 128), (600, 100, 128), (600, 100, 64)])
def test_cached_attention_outputs_after_an_item_with_a_single_tile(rows, tokens, H, D):
    """Heads with an odd number of row tiles over short caches: both tiles of a CTA write their outputs through one
    place, and after an item with tile 0 alone tile 1 is free to run ahead of it."""
    assert takes_a_single_tile_before_a_pair(rows, tokens, H, D)
    c = filled(H, -(-tokens // 64) * 64, D, tokens, seed=rows + tokens)
    q = torch.randn(rows, H, D, generator=torch.Generator(device=DEV).manual_seed(tokens), device=DEV).bfloat16()
    got = h3b.kv8_attention(q, c)
    k, v = values(c)
    for h in range(H):
        o, a, m = softmax_rows(q[:, h], k[:, h], v[:, h], D ** -0.5)
        near(got[:, h], o, a, m, tokens, D)
    for _ in range(10):
        assert torch.equal(h3b.kv8_attention(q, c), got)
    assert h3b.status() == 0


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("start,n", [(17, 1), (100, 28), (63, 200)])
def test_write_behind_scales_of_either_sign(D, start, n):
    """The staying tokens' scale is kept if it is larger in magnitude, of whichever sign, and gives way if it is not."""
    H, block = 8, start // 64
    c = filled(H, -(-(start + n) // 64) * 64, D, start, seed=71)
    k, v = randn(n, H, D, seed=72), randn(n, H, D, seed=73)
    factor = torch.tensor([0.5, -0.5, 2.0, -2.0, -1.0, -0.01, 30.0, -30.0])
    before, want = [], []
    for x, codes, scales in ((k, c.kq, c.ks), (v, c.vq, c.vs)):
        here = x[:64 - start % 64].float().cpu().transpose(0, 1)  # the new tokens of the block that holds older ones
        new = here.abs().amax((1, 2)) / torch.tensor(127.0)
        former = new * factor
        scales[:, block] = former.to(DEV)
        old = codes[:, block * 64:start].float().cpu()
        s = torch.where(former.abs() > new, former, new)
        kept = torch.where((s == former)[:, None, None], old, (old * (former / s)[:, None, None]).round())
        before.append(old.double() * former.double()[:, None, None])
        want.append((torch.cat([kept, (here / s[:, None, None]).round()], 1), s))
    c.write(k, v)
    end = min(start + n, block * 64 + 64)
    for codes, scales, (q, s), was, x in zip((c.kq, c.vq), (c.ks, c.vs), want, before, (k, v)):
        assert same(codes[:, block * 64:end].float(), q) and same(scales[:, block], s)
        # what is held is off by half a step of the code and three fp32 roundings at 127 steps
        step = s.double().abs()[:, None, None] * (0.5 + 3 * 127 * 2.0 ** -24)
        got = codes[:, block * 64:end].double().cpu() * s.double()[:, None, None]
        now = torch.cat([was, x[:end - start].double().cpu().transpose(0, 1)], 1)
        assert ((got - now).abs() <= step).all()
    check_cached(randn(3, H, D, seed=74), c)
    check_cached(randn(70, H, D, seed=75), c)


@pytest.mark.parametrize("former", [-0.0, -INF, NAN])
def test_write_behind_scales_that_are_no_numbers(former):
    c = filled(2, 64, 64, 10, seed=76)
    c.ks[0], c.vs[0] = former, former
    x = randn(5, 2, 64, seed=77)
    gk, gv = c.write(x, x).read(dtype=torch.float32)
    for g in (gk, gv):
        if former == 0:
            assert (g[:10, 0] == 0).all() and (g[10:, 0] != 0).any()
        else:
            assert torch.isnan(g[10:, 0]).all() and not torch.isfinite(g[:10, 0]).any()
        assert torch.isfinite(g[:, 1]).all()


@pytest.mark.parametrize("rows", [1, 20, 70, 300])
@pytest.mark.parametrize("tokens", [1, 64, 3000])
def test_cached_attention_of_rows_whose_scores_are_all_minus_infinity(rows, tokens):
    """A softmax over nothing but -infinity is NaN, whole and split over the keys; a row that has keys is never zeros."""
    c = filled(2, -(-tokens // 64) * 64, 128, tokens, seed=81)
    c.kq[:, :tokens, 0] = -5
    q = randn(rows, 2, 128, seed=82)
    want = h3b.kv8_attention(q, c)
    q[rows // 2, 1, 0] = INF
    got = h3b.kv8_attention(q, c)
    assert torch.isnan(got[rows // 2, 1]).all()
    got[rows // 2, 1] = want[rows // 2, 1]
    assert same(got, want)


@pytest.mark.parametrize("rows,topk", [(1, 3), (1, 130), (300, 3), (300, 40)])
def test_sparse_attention_over_scores_of_minus_infinity(rows, topk):
    """Keys with a score of -infinity weigh nothing beside others; rows that have no other are NaN, rows that have no key
    at all zero."""
    H, D, keys, nq = 2, 128, 9000, -(-rows // 128)
    q, k, v = randn(rows, H, D, seed=83), randn(keys, H, D, seed=84), randn(keys, H, D, seed=85)
    q[:, :, 0] = 1.0
    k[64:, 1, 0] = -INF  # all blocks of head 1 but the first
    blocks = torch.arange(topk, dtype=torch.int32, device=DEV).expand(H, nq, topk).contiguous()
    got = h3b.block_sparse_attention(q, k, v, blocks)
    alone = torch.full_like(blocks, -1)
    alone[0], alone[1, :, 0] = blocks[0], 0
    o, a, m = sparse(q, k, v, alone, D ** -0.5)
    near(got, o, a, m, topk * 64, D)
    blocks[1, :, 0] = -1
    got = h3b.block_sparse_attention(q, k, v, blocks)
    assert torch.isnan(got[:, 1]).all() and torch.isfinite(got[:, 0]).all()
    blocks[1] = -1
    assert (h3b.block_sparse_attention(q, k, v, blocks)[:, 1] == 0).all()
    assert h3b.status() == 0


@pytest.mark.parametrize("rows", [64, 128])
def test_block_means_of_any_order_within_their_exact_range(rows):
    """Values within a factor of 2^38 add up to 53 bits at most (8 + 38 + 7), so a block's mean is that of its rows in any
    order."""
    x = randn(rows, 3, 128, seed=91).float().sign() * (1 + torch.rand(rows, 3, 128, generator=gen(92))).to(DEV)
    x = (x * 2.0 ** torch.randint(-19, 19, (rows, 3, 128), generator=gen(93)).to(DEV)).bfloat16()
    want = h3b.block_means(x, rows)
    assert same(want, means(x, rows))
    for seed in range(5):
        assert torch.equal(h3b.block_means(x[torch.randperm(rows, generator=gen(94 + seed)).to(DEV)], rows), want)


@pytest.mark.parametrize("rows,H,groups,topk", [(700, 4, 2, 3), (20000, 40, 8, 4)])
def test_sparse_attention_of_head_groups_selects_the_same_blocks(rows, H, groups, topk):
    """Calls of some heads each, on views of one buffer as a head group's exchange delivers them: the blocks are those of
    the call of all heads; the outputs are right, if not bitwise the same (a call's split over the keys goes by its heads)."""
    hc, D = H // groups, 64
    buf = [randn(rows * H * D, seed=s) for s in (101, 102, 103)]
    views = [[b[g * rows * hc * D:(g + 1) * rows * hc * D].view(rows, hc, D) for b in buf] for g in range(groups)]
    q, k, v = (torch.cat([views[g][i] for g in range(groups)], 1) for i in range(3))
    o, blocks = h3b.sparse_attention(q, k, v, topk, return_blocks=True)
    for g in (0, groups - 1):
        og, bg = h3b.sparse_attention(*views[g], topk, return_blocks=True)
        assert same(bg, blocks[g * hc:(g + 1) * hc])
        ref, a, m = sparse(*(t[:, :1] for t in views[g]), bg[:1], D ** -0.5)
        near(og[:, :1], ref, a, m, topk * 64, D)
        near(o[:, g * hc:g * hc + 1], ref, a, m, topk * 64, D)
    assert h3b.status() == 0
