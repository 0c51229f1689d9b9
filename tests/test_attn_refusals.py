"""Refusals of the attention operators, without a GPU: the C entry points before any device work, and the Python checks."""
import ctypes

import pytest
import torch

import h3b
from h3b._lib import lib

P0 = ctypes.c_void_p(0)
P16 = ctypes.c_void_p(4096)  # aligned, never dereferenced: each call is refused for another reason
P2 = ctypes.c_void_p(4098)


def refused(name, rc, word):
    assert rc == -1, f"{name} returned {rc}"
    msg = lib.h3b_last_error().decode()
    assert name in msg and word in msg, msg


def write(k=P16, kld=128, khs=128, start=0, n=1, H=1, D=128, kq=P16, cap=64):
    return lib.h3b_kv8_write(k, kld, khs, P16, 128, 128, start, n, H, D, kq, P16, P16, P16, cap, P0)


def test_write_refusals():
    refused("h3b_kv8_write", write(D=96), "head_dim")
    refused("h3b_kv8_write", write(H=0), "heads")
    refused("h3b_kv8_write", write(cap=65), "capacity")
    refused("h3b_kv8_write", write(start=64), "outside")
    refused("h3b_kv8_write", write(start=-1), "outside")
    refused("h3b_kv8_write", write(n=-1), "outside")
    refused("h3b_kv8_write", write(start=1, n=2 ** 63 - 1), "outside")
    refused("h3b_kv8_write", write(kq=P0), "NULL")
    refused("h3b_kv8_write", write(k=P0), "NULL")
    refused("h3b_kv8_write", write(k=P2), "aligned")
    refused("h3b_kv8_write", write(kld=129), "strides")
    assert write(n=0) == 0  # nothing to do, nothing launched


def test_read_refusals():
    def read(start=0, n=1, D=128, out=P16):
        return lib.h3b_kv8_read(P16, P16, P16, P16, 64, start, n, 1, D, out, P16, 0, P0)
    refused("h3b_kv8_read", read(D=32), "head_dim")
    refused("h3b_kv8_read", read(start=60, n=5), "outside")
    refused("h3b_kv8_read", read(out=P0), "NULL")
    refused("h3b_kv8_read", read(out=P2), "aligned")
    assert read(n=0) == 0


def test_attention_refusals():
    def cached(q=P16, qld=128, Sq=1, H=1, D=128, kq=P16, cap=64, length=64, o=P16):
        return lib.h3b_kv8_attn(q, qld, 128, Sq, H, D, kq, P16, P16, P16, cap, length, 1.0, o, 128, 128, P0, 0, P0)
    refused("h3b_kv8_attn", cached(length=65), "length")
    refused("h3b_kv8_attn", cached(length=-1), "length")
    refused("h3b_kv8_attn", cached(cap=100), "capacity")
    refused("h3b_kv8_attn", cached(kq=P0), "NULL")
    refused("h3b_kv8_attn", cached(H=0), "heads")
    refused("h3b_kv8_attn", cached(D=256), "head_dim")
    refused("h3b_kv8_attn", cached(q=P2), "aligned")
    refused("h3b_kv8_attn", cached(o=P0), "NULL")
    refused("h3b_kv8_attn", cached(qld=100), "strides")
    refused("h3b_kv8_attn", cached(Sq=2 ** 40), "range")
    refused("h3b_kv8_attn", cached(qld=0), "strides")
    refused("h3b_kv8_attn", cached(cap=4096, length=4096), "workspace")
    assert lib.h3b_attn_workspace(1, 1, 1, 128, 64) > 0 and lib.h3b_attn_workspace(1, 0, 1, 128, 64) == 0
    assert lib.h3b_attn_workspace(0, 100000, 40, 128, 64) == 0 and lib.h3b_attn_workspace(1, 5, 1, 128, 0) == 0
    # a cache's widened heads: 512 MiB at most, or one head
    assert lib.h3b_attn_workspace(1, 100000, 40, 128, 1 << 14) >= 2 ** 20 * 512
    assert cached(Sq=0) == 0

    def sparse(k=P16, kld=128, Sk=64, blocks=P16, topk=1, D=128):
        return lib.h3b_block_sparse_attn(P16, 128, 128, 1, 1, D, k, kld, 128, P16, 128, 128, Sk, blocks, topk, 1.0, P16,
                                         128, 128, P0, 0, P0)
    refused("h3b_block_sparse_attn", sparse(topk=-1), "topk")
    refused("h3b_block_sparse_attn", sparse(topk=2 ** 26), "topk")
    refused("h3b_block_sparse_attn", sparse(blocks=P0), "blocks")
    refused("h3b_block_sparse_attn", sparse(k=P2), "aligned")
    refused("h3b_block_sparse_attn", sparse(kld=4), "strides")
    refused("h3b_block_sparse_attn", sparse(Sk=-1), "range")
    refused("h3b_block_sparse_attn", sparse(D=80), "head_dim")


def test_sparse_attention_refusals():
    def sparse(q=P16, Sq=200, Sk=100, H=2, D=128, topk=2, ws=P16, size=1 << 30, k=P16):
        return lib.h3b_sparse_attn(q, 256, 128, Sq, H, D, k, 256, 128, P16, 256, 128, Sk, P0, topk, 1.0, P16, P16, 256, 128,
                                   ws, size, P0)
    refused("h3b_sparse_attn", sparse(D=32), "head_dim")
    refused("h3b_sparse_attn", sparse(H=0), "heads")
    refused("h3b_sparse_attn", sparse(Sq=-1), "rows")
    refused("h3b_sparse_attn", sparse(topk=-1), "topk")
    refused("h3b_sparse_attn", sparse(ws=P0), "workspace")
    refused("h3b_sparse_attn", sparse(size=100), "workspace")
    refused("h3b_sparse_attn", sparse(k=P2), "aligned")
    # query means, key means (unless kept) and the scores
    assert lib.h3b_sparse_attn_workspace(200, 100, 2, 128, 2, 0) == 2048 + 2048 + 2 * 64 * 2 * 8
    assert lib.h3b_sparse_attn_workspace(200, 100, 2, 128, 2, 1) == 2048 + 2 * 64 * 2 * 8
    assert lib.h3b_sparse_attn_workspace(200, 100, 2, 96, 2, 1) == 0


def test_selection_refusals():
    def means(D=128, rows=64, x=P16, ld=128):
        return lib.h3b_block_means(x, ld, 128, 5, 1, D, rows, P16, P0)
    refused("h3b_block_means", means(D=16), "head_dim")
    refused("h3b_block_means", means(rows=96), "rows")
    refused("h3b_block_means", means(x=P0), "NULL")
    refused("h3b_block_means", means(ld=12), "strides")

    def select(nq=1, nk=4, topk=2, D=64, ws=P16, size=1 << 20):
        return lib.h3b_select_blocks(P16, P16, nq, nk, 1, D, topk, P16, ws, size, P0)
    refused("h3b_select_blocks", select(topk=5), "topk")
    refused("h3b_select_blocks", select(topk=-1), "topk")
    refused("h3b_select_blocks", select(D=72), "head_dim")
    refused("h3b_select_blocks", select(ws=P0), "NULL")
    refused("h3b_select_blocks", select(size=100), "workspace")
    assert select(nq=0) == 0 and select(topk=0) == 0
    assert lib.h3b_select_blocks_workspace(0, 5, 1) == 0
    # one unit is 64 query blocks of a head; a workspace holds at least one, and at most 256 MiB beyond it
    assert lib.h3b_select_blocks_workspace(65, 10, 3) == 2 * 3 * 64 * 10 * 8
    assert lib.h3b_select_blocks_workspace(1, 1 << 20, 1) == 64 * (1 << 20) * 8


def test_python_checks_on_the_cpu():
    """No CPU path: CPU tensors raise TypeError, malformed caches ValueError."""
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(TypeError):
        h3b.block_means(x)
    with pytest.raises(TypeError):
        h3b.sparse_attention(x, x, x, 1)
    with pytest.raises(TypeError):
        h3b.KV8Cache(64, 2, 64, device="cpu")
    with pytest.raises(ValueError):
        h3b.KV8Cache(64, 2, 96)
    with pytest.raises(ValueError):
        h3b.KV8Cache(-1, 2, 64)
    kq, ks = torch.zeros(2, 128, 64, dtype=torch.int8), torch.zeros(2, 2)
    for bad in ((kq.float(), kq, ks, ks, 0), (kq[:, :100], kq[:, :100], ks, ks, 0), (kq, kq[:1], ks, ks, 0),
                (kq, kq, ks[:, :1], ks, 0), (kq, kq, ks, ks.double(), 0), (kq, kq, ks, ks, 129), (kq, kq, ks, ks, -1),
                (kq.transpose(0, 1).contiguous().transpose(0, 1), kq, ks, ks, 0)):
        with pytest.raises(ValueError):
            h3b.KV8Cache.wrap(*bad)
    with pytest.raises(TypeError):
        h3b.KV8Cache.wrap(kq, kq, ks, ks, 0)


def test_strides_must_be_positive():
    for stride in (0, -128):
        refused("h3b_kv8_write", write(kld=stride), "strides")
        refused("h3b_kv8_write", write(khs=stride), "strides")
        refused("h3b_kv8_write", lib.h3b_kv8_write(P16, 128, 128, P16, stride, 128, 0, 1, 1, 128, P16, P16, P16, P16, 64, P0),
                "strides")
        refused("h3b_kv8_write", lib.h3b_kv8_write(P16, 128, 128, P16, 128, stride, 0, 1, 1, 128, P16, P16, P16, P16, 64, P0),
                "strides")
        refused("h3b_block_means", lib.h3b_block_means(P16, stride, 128, 5, 1, 128, 64, P16, P0), "strides")
        refused("h3b_block_means", lib.h3b_block_means(P16, 128, stride, 5, 1, 128, 64, P16, P0), "strides")


def test_sparse_attention_is_refused_before_any_of_its_steps():
    """The attention's own checks come before the means and the selection are enqueued (no device here to run them)."""
    def sparse(q=P16, k=P16, v=P16, o=P16, blocks=P16, **stride):
        st = {**dict.fromkeys(("qld", "kld", "vld", "old"), 256), **dict.fromkeys(("qhs", "khs", "vhs", "ohs"), 128), **stride}
        return lib.h3b_sparse_attn(q, st["qld"], st["qhs"], 200, 2, 128, k, st["kld"], st["khs"], v, st["vld"], st["vhs"], 100,
                                   P0, 2, 1.0, blocks, o, st["old"], st["ohs"], P16, 1 << 30, P0)
    for bad in (P0, P2):
        for name in "qkvo":
            refused("h3b_sparse_attn", sparse(**{name: bad}), "aligned")
    refused("h3b_sparse_attn", sparse(blocks=P0), "blocks")
    for name in ("qld", "qhs", "kld", "khs", "vld", "vhs", "old", "ohs"):
        for stride in (0, -256, 132):
            refused("h3b_sparse_attn", sparse(**{name: stride}), "strides")


def test_a_single_text_cache_is_not_taken_for_several_blocks():
    """A cache holds one block's keys and values: given alone it would serve every block with those."""
    from h3b import model as hm

    dit = object.__new__(hm.SynthDiT)
    dit.cfg, dit.params = None, [None, None]
    cache = object.__new__(h3b.KV8Cache)
    for text in (cache, [cache], (cache,) * 3):
        with pytest.raises(ValueError, match="text caches for 2 blocks"):
            dit.forward(None, None, None, text)
