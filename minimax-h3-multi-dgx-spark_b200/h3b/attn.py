"""Attention operators next to the block's SDPA: a key/value cache held in 8 bits, and block-sparse attention.

  KV8Cache                 K/V of one sequence as int8 codes with an fp32 scale per 64 tokens and head
    .write(k, v)             quantise new tokens into it;  .read() gives them back as bf16 / fp32
  kv8_attention(q, cache)  softmax(scale * q K^T) V over the cached tokens
  block_means(x, rows)     fp32 means of blocks of rows
  select_blocks(qm, km, k) the k key blocks whose means have the largest products with a query block's mean
  block_sparse_attention   softmax attention of each block of 128 query rows over its own blocks of 64 keys
  sparse_attention         the three in a row

They take the place of the attention between the qkv and the out projection of sp_attention
(comfyui_nodes/minimax-h3-sp/minimax_sp/sp_forward.py:276-318), tensors being [tokens, heads, head_dim] with
head_dim 64 or 128 as everywhere in h3b.  h3b.model uses them for a cached text context (SynthDiT.text_cache) and for
sparse self-attention (DiTConfig.attn_topk).  Inputs may be strided over tokens and heads (multiples of 8 elements,
16-byte aligned, unit stride over the head's channels); outputs are allocated with PyTorch's caching allocator on the
input's device and the kernels run on its current stream.  No operator synchronises; under stream capture the sizes
(a cache's length among them) are those of the capture.  There is no backward pass: the framework does not train.
"""
import contextlib

import torch

from ._lib import check, lib, require_cuda
from .trace import span

BF16 = torch.bfloat16
KEYS = 64    # tokens per scale of the cache, keys per sparse block
QROWS = 128  # query rows that share a selection of key blocks


_HERE = contextlib.nullcontext()


def _on(device):
    """Makes `device` the current one for the launches inside (nothing to do when it is)."""
    return _HERE if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _stream(device):
    # (the handle alone: a torch.cuda.Stream object costs as much as the rest of a call's checks)
    return torch._C._cuda_getCurrentRawStream(device.index)


def _rows(name, t, like=None):
    """(token stride, head stride) of t [n, H, D] bf16 in elements; raises if the kernels cannot read it."""
    if t.dtype != BF16 or t.dim() != 3:
        raise ValueError(f"{name} must be a bf16 [tokens, heads, head_dim] tensor, got {t.dtype} {tuple(t.shape)}")
    n, h, d = t.shape
    if d != 128 and d != 64:
        raise ValueError(f"{name}: head_dim {d} is not covered (64 or 128)")
    if h == 0:
        raise ValueError(f"{name}: no heads")
    if like is not None and (t.shape[1:] != like.shape[1:] or t.device != like.device):
        raise ValueError(f"{name} {tuple(t.shape)} on {t.device} does not go with {tuple(like.shape)} on {like.device}")
    ld, hs, cs = t.stride()
    # the stride over a single token or head says nothing
    if n <= 1:
        ld = h * d
    if h == 1:
        hs = d
    if n and (cs != 1 or ld % 8 or hs % 8 or ld <= 0 or hs <= 0 or t.data_ptr() % 16):
        raise ValueError(f"{name}: strides {t.stride()} need a unit channel stride, positive token and head strides that "
                         "are multiples of 8 elements, and a 16-byte aligned start; pass a contiguous copy")
    return ld, hs


def _scale(scale, d):
    return d ** -0.5 if scale is None else float(scale)


def _workspace(cache, q, segments):
    """(tensor or None, bytes): where the parts of a split over the keys meet and a cache's codes are widened."""
    n = lib.h3b_attn_workspace(cache, q.shape[0], q.shape[1], q.shape[2], segments)
    return (torch.empty(n, dtype=torch.uint8, device=q.device) if n else None), n


def _ptr(t):
    return None if t is None else t.data_ptr()


class KV8Cache:
    """Keys and values of up to `capacity` tokens in 8 bits.

    kq, vq: int8 codes [heads, capacity, head_dim]; ks, vs: fp32 scales [heads, capacity / 64], one per block of 64
    tokens and head (capacity is rounded up to whole blocks).  `length` tokens are held; what lies behind them is
    never read.  A token costs 2 * heads * (head_dim + 4 / 64) bytes, about half of bf16."""

    def __init__(self, capacity, heads, head_dim, device="cuda"):
        if capacity < 0 or heads <= 0 or head_dim not in (64, 128):
            raise ValueError(f"KV8Cache: capacity {capacity}, heads {heads}, head_dim {head_dim} (64 or 128)")
        cap = -(-int(capacity) // KEYS) * KEYS
        kw = dict(device=device)
        self._take(torch.empty((heads, cap, head_dim), dtype=torch.int8, **kw),
                   torch.empty((heads, cap, head_dim), dtype=torch.int8, **kw),
                   torch.empty((heads, cap // KEYS), dtype=torch.float32, **kw),
                   torch.empty((heads, cap // KEYS), dtype=torch.float32, **kw), 0)

    @classmethod
    def wrap(cls, kq, vq, ks, vs, length):
        """A cache over existing codes and scales (contiguous, laid out as above), of which `length` tokens are held."""
        shape = kq.shape
        if len(shape) != 3 or kq.dtype != torch.int8 or shape[0] == 0 or shape[2] not in (64, 128) or shape[1] % KEYS:
            raise ValueError("KV8Cache.wrap: kq must be int8 [heads, capacity, head_dim], capacity a multiple of "
                             f"{KEYS} and head_dim 64 or 128; got {kq.dtype} {tuple(shape)}")
        scales = (shape[0], shape[1] // KEYS)
        if vq.shape != shape or vq.dtype != torch.int8 or ks.shape != scales or vs.shape != scales or \
                ks.dtype != torch.float32 or vs.dtype != torch.float32:
            raise ValueError(f"KV8Cache.wrap: vq must match kq, ks and vs must be fp32 {scales}")
        for t in (kq, vq, ks, vs):
            if not t.is_contiguous() or t.device != kq.device or t.data_ptr() % 16:
                raise ValueError("KV8Cache.wrap: codes and scales must be contiguous, 16-byte aligned and on one device")
        if not 0 <= length <= shape[1]:
            raise ValueError(f"KV8Cache.wrap: length {length} outside the capacity {shape[1]}")
        self = cls.__new__(cls)
        self._take(kq, vq, ks, vs, int(length))
        return self

    def _take(self, kq, vq, ks, vs, length):
        require_cuda(kq)
        self.kq, self.vq, self.ks, self.vs, self.length = kq, vq, ks, vs, length

    @property
    def heads(self):
        return self.kq.shape[0]

    @property
    def capacity(self):
        return self.kq.shape[1]

    @property
    def head_dim(self):
        return self.kq.shape[2]

    def _goes_with(self, name, t):
        if t.shape[1] != self.heads or t.shape[2] != self.head_dim or t.device != self.kq.device:
            raise ValueError(f"{name} {tuple(t.shape)} on {t.device} does not go with a cache of {self.heads} heads of "
                             f"{self.head_dim} on {self.kq.device}")

    def write(self, k, v, start=None):
        """Quantise k, v [n, heads, head_dim] (bf16) into tokens start .. start + n (start <= length, by default the
        end); tokens that lay at and behind start are dropped.  A block's scale is its new tokens' absmax / 127, or
        its former scale where older tokens stay in it and that is larger in magnitude; staying codes are requantised
        when the scale changes.  A NaN or infinity makes its block and head NaN.  Returns the cache."""
        require_cuda(k, v)
        start = self.length if start is None else int(start)
        (kld, khs), (vld, vhs) = _rows("k", k), _rows("v", v, k)
        self._goes_with("k", k)
        n = k.shape[0]
        if v.shape[0] != n:
            raise ValueError(f"KV8Cache.write: {n} keys and {v.shape[0]} values")
        if not 0 <= start <= self.length or start + n > self.capacity:
            raise ValueError(f"KV8Cache.write: tokens {start} .. {start + n} do not follow the {self.length} held "
                             f"within the capacity {self.capacity}")
        H, D = self.heads, self.head_dim
        if n:
            with _on(k.device), span("kv8_write", 6 * n * H * D):
                check(lib.h3b_kv8_write(_ptr(k), kld, khs, _ptr(v), vld, vhs, start, n, H, D, _ptr(self.kq), _ptr(self.vq),
                                        _ptr(self.ks), _ptr(self.vs), self.capacity, _stream(k.device)), "h3b_kv8_write")
        self.length = start + n
        return self

    def read(self, start=0, stop=None, dtype=BF16):
        """(k, v) [stop - start, heads, head_dim] of the held tokens: code * scale, rounded once more to bf16 unless
        dtype is float32."""
        stop = self.length if stop is None else int(stop)
        start = int(start)
        if not 0 <= start <= stop <= self.length:
            raise ValueError(f"KV8Cache.read: tokens {start} .. {stop} are not among the {self.length} held")
        if dtype not in (BF16, torch.float32):
            raise ValueError(f"KV8Cache.read: dtype {dtype} is not covered (bfloat16 or float32)")
        n, H, D = stop - start, self.heads, self.head_dim
        k, v = (torch.empty((n, H, D), dtype=dtype, device=self.kq.device) for _ in "kv")
        if n:
            with _on(k.device), span("kv8_read", 2 * n * H * D * (1 + k.element_size())):
                check(lib.h3b_kv8_read(_ptr(self.kq), _ptr(self.vq), _ptr(self.ks), _ptr(self.vs), self.capacity, start, n,
                                       H, D, _ptr(k), _ptr(v), int(dtype == torch.float32), _stream(k.device)), "h3b_kv8_read")
        return k, v


def kv8_attention(q, cache, scale=None):
    """softmax(scale * q K^T) V of q [rows, heads, head_dim] over the tokens held in `cache` -> bf16 like q
    (contiguous); scale defaults to head_dim ** -0.5.  An empty cache gives zeros."""
    require_cuda(q)
    ld, hs = _rows("q", q)
    cache._goes_with("q", q)
    sq, H, D = q.shape
    o = torch.empty((sq, H, D), dtype=BF16, device=q.device)
    if sq:
        ws, nbytes = _workspace(1, q, -(-cache.length // KEYS))
        with _on(q.device), span("kv8_attn", 4.0 * sq * cache.length * H * D):
            check(lib.h3b_kv8_attn(_ptr(q), ld, hs, sq, H, D, _ptr(cache.kq), _ptr(cache.vq), _ptr(cache.ks), _ptr(cache.vs),
                                   cache.capacity, cache.length, _scale(scale, D), _ptr(o), H * D, D,
                                   _ptr(ws), nbytes, _stream(q.device)), "h3b_kv8_attn")
    return o


def block_means(x, rows=KEYS, out=None):
    """fp32 [ceil(n / rows), heads, head_dim]: the mean of each block of `rows` (64 or 128) rows of x
    [n, heads, head_dim] bf16, the last block's over the rows it has.  Summed in 64 bits and rounded once: exact sums
    where a block's nonzero values lie within a factor of 2^38, a fixed order otherwise.  out (optional, contiguous) takes the result: a program that appends keys keeps the means
    and renews those of the blocks it touched, block_means(k[64 * b:], out=means[b:])."""
    require_cuda(x)
    ld, hs = _rows("x", x)
    if rows not in (64, 128):
        raise ValueError(f"block_means: rows {rows} is not covered (64 or 128)")
    n, H, D = x.shape
    shape = (-(-n // rows), H, D)
    if out is None:
        out = torch.empty(shape, dtype=torch.float32, device=x.device)
    elif tuple(out.shape) != shape or out.dtype != torch.float32 or not out.is_contiguous() or out.device != x.device:
        raise ValueError(f"block_means: out must be contiguous fp32 {shape} on {x.device}")
    if n:
        with _on(x.device), span("block_means", 2 * x.numel()):
            check(lib.h3b_block_means(_ptr(x), ld, hs, n, H, D, rows, _ptr(out), _stream(x.device)), "h3b_block_means")
    return out


def select_blocks(qm, km, topk):
    """int32 [heads, nq, min(topk, nk)]: for each head and row of qm [nq, heads, head_dim] (fp32 means of query
    blocks) the rows of km [nk, heads, head_dim] with the largest products, ascending.  Products are summed in 64
    bits (in an order of their own up to 4 query blocks: scores that differ by no more than its rounding may rank
    either way); ties go to the lowest index, a NaN product ranks below every number."""
    require_cuda(qm, km)
    if qm.dim() != 3 or km.dim() != 3 or qm.shape[1:] != km.shape[1:] or qm.device != km.device:
        raise ValueError(f"select_blocks: means {tuple(qm.shape)} and {tuple(km.shape)} do not go together")
    if any(t.dtype != torch.float32 or not t.is_contiguous() for t in (qm, km)):
        raise ValueError("select_blocks: means must be contiguous fp32 [blocks, heads, head_dim]")
    (nq, H, D), nk = qm.shape, km.shape[0]
    if D not in (64, 128) or H == 0:
        raise ValueError(f"select_blocks: heads {H}, head_dim {D} (64 or 128)")
    if topk < 0:
        raise ValueError(f"select_blocks: topk {topk}")
    topk = min(int(topk), nk)
    blocks = torch.empty((H, nq, topk), dtype=torch.int32, device=qm.device)
    if nq and topk:
        ws = torch.empty(lib.h3b_select_blocks_workspace(nq, nk, H), dtype=torch.uint8, device=qm.device)
        with _on(qm.device), span("select_blocks", 2.0 * nq * nk * H * D, launches=2):
            check(lib.h3b_select_blocks(_ptr(qm), _ptr(km), nq, nk, H, D, topk, _ptr(blocks), _ptr(ws), ws.numel(),
                                        _stream(qm.device)), "h3b_select_blocks")
    return blocks


def block_sparse_attention(q, k, v, blocks, scale=None):
    """softmax(scale * q K^T) V where query rows 128 i .. of head h see the keys of blocks[h, i, :] only, block b being
    keys 64 b .. 64 b + 63 (those that exist).  q [rows, H, D], k / v [keys, H, D] bf16, blocks int32 [H,
    ceil(rows / 128), n] contiguous; -1 stands for no block, a block named twice counts twice, and rows without a key
    are zero.  An index outside -1 .. ceil(keys / 64) - 1 is skipped and recorded in the device status."""
    require_cuda(q, k, v, blocks)
    (qld, qhs), (kld, khs), (vld, vhs) = _rows("q", q), _rows("k", k, q), _rows("v", v, q)
    sq, H, D = q.shape
    nq = -(-sq // QROWS)
    if v.shape[0] != k.shape[0]:
        raise ValueError(f"block_sparse_attention: {k.shape[0]} keys and {v.shape[0]} values")
    if blocks.dtype != torch.int32 or blocks.dim() != 3 or tuple(blocks.shape[:2]) != (H, nq) or \
            not blocks.is_contiguous() or blocks.device != q.device:
        raise ValueError(f"block_sparse_attention: blocks must be contiguous int32 [{H}, {nq}, n] on {q.device}, got "
                         f"{blocks.dtype} {tuple(blocks.shape)}")
    n = blocks.shape[2]
    o = torch.empty((sq, H, D), dtype=BF16, device=q.device)
    if sq:
        ws, nbytes = _workspace(0, q, n)
        with _on(q.device), span("sparse_attn", 4.0 * sq * n * KEYS * H * D):
            check(lib.h3b_block_sparse_attn(_ptr(q), qld, qhs, sq, H, D, _ptr(k), kld, khs, _ptr(v), vld, vhs, k.shape[0],
                                            _ptr(blocks), n, _scale(scale, D), _ptr(o), H * D, D,
                                            _ptr(ws), nbytes, _stream(q.device)), "h3b_block_sparse_attn")
    return o


def sparse_attention(q, k, v, topk, scale=None, k_means=None, return_blocks=False):
    """block_sparse_attention over the topk blocks of 64 keys that select_blocks finds for each block of 128 query
    rows.  k_means: block_means(k) if the program keeps it.  With return_blocks, (o, blocks)."""
    require_cuda(q, k, v, k_means)
    (qld, qhs), (kld, khs), (vld, vhs) = _rows("q", q), _rows("k", k, q), _rows("v", v, q)
    (sq, H, D), sk = q.shape, k.shape[0]
    nk = -(-sk // KEYS)
    if v.shape[0] != sk:
        raise ValueError(f"sparse_attention: {sk} keys and {v.shape[0]} values")
    if topk < 0:
        raise ValueError(f"sparse_attention: topk {topk}")
    if k_means is not None and (k_means.shape != (nk, H, D) or k_means.dtype != torch.float32 or
                                not k_means.is_contiguous() or k_means.device != q.device):
        raise ValueError(f"sparse_attention: k_means must be contiguous fp32 {(nk, H, D)} on {q.device}, got "
                         f"{k_means.dtype} {tuple(k_means.shape)}")
    topk = min(int(topk), nk)
    blocks = torch.empty((H, -(-sq // QROWS), topk), dtype=torch.int32, device=q.device)
    o = torch.empty((sq, H, D), dtype=BF16, device=q.device)
    if sq:
        has = int(k_means is not None)
        nbytes = lib.h3b_sparse_attn_workspace(sq, sk, H, D, topk, has)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
        with _on(q.device), span("sparse_attn", 4.0 * sq * topk * KEYS * H * D, launches=4):
            check(lib.h3b_sparse_attn(_ptr(q), qld, qhs, sq, H, D, _ptr(k), kld, khs, _ptr(v), vld, vhs, sk, _ptr(k_means),
                                      topk, _scale(scale, D), _ptr(blocks), _ptr(o), H * D, D, _ptr(ws), nbytes,
                                      _stream(q.device)), "h3b_sparse_attn")
    return (o, blocks) if return_blocks else o
