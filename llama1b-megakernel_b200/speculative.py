"""Speculative decoding: drafted tokens verified in one pass over a paged cache.

The reference decodes one token per step over a bf16 cache
(nki_kernels/attention.py:77-492). Here several drafted tokens of a sequence go
through the layers together, and the cache may hold 8-bit rows. The operators,
each one C entry point of ``include/mk.h``:

* ``kv_write``: rotate the q/k/v rows of new tokens, store their K/V (bf16, or
  e4m3 codes with one power-of-two scale byte per row) and write q;
* ``kv_read``: rows of a sequence back as contiguous bf16;
* ``tree_attention``: every drafted node attends its sequence's committed
  positions and the drafted nodes its mask allows (its ancestors; for a chunk
  of a prompt, the nodes before it). One node per sequence is a decode step;
* ``token_logprobs``: log probabilities of given tokens, entropy and the most
  likely alternatives of rows of logits.

All run asynchronously on the current stream of their tensors' device, allocate
outputs and workspaces that are not passed in from PyTorch's allocator, and raise
``ValueError`` on arguments that do not fit. What only the device can see (a page
id, a length or a token out of range) sets the caller's ``error`` word, an int32
tensor of one zero that the caller reads when it synchronises.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib


def _check(t: torch.Tensor, dtype, name: str, dev, shape=None) -> int:
    """The tensor's address, once its type, device, layout and shape fit."""
    if t.dtype is not dtype and t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if t.device != dev:
        raise ValueError(f"{name} is on {t.device}, the cache or logits on {dev}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    return t.data_ptr()


def _call(fn, dev: torch.device, *args) -> None:
    """Run an entry point on the current stream of ``dev``."""
    if dev.index == torch.cuda.current_device():
        _lib.check(fn(*args, torch.cuda.current_stream(dev).cuda_stream))
    else:
        with torch.cuda.device(dev):
            _lib.check(fn(*args, torch.cuda.current_stream(dev).cuda_stream))


def _error_word(error: torch.Tensor | None, dev) -> torch.Tensor:
    return torch.zeros(1, dtype=torch.int32, device=dev) if error is None else error


class KVLayer:
    """One layer of a paged cache, as the operators take it: pages [num_pages, nkv,
    page_size, 64] (bf16, or ``torch.float8_e4m3fn`` with uint8 scale bytes
    [num_pages, nkv, page_size]) and block tables [batch, max_blocks] int32.
    Holds references to the tensors; make it once per layer
    (``PagedKVCache.layer``) or per call."""

    __slots__ = ("k_pages", "v_pages", "block_tables", "k_scales", "v_scales", "device", "batch",
                 "num_kv_heads", "page_size", "max_blocks", "struct", "ref")

    def __init__(self, k_pages, v_pages, block_tables, k_scales=None, v_scales=None):
        if k_pages.dim() != 4 or k_pages.shape[3] != 64:
            raise ValueError(f"pages must be [num_pages, kv heads, page_size, 64], got "
                             f"{tuple(k_pages.shape)}")
        dev = k_pages.device
        if dev.type != "cuda":
            raise ValueError("the cache must be on a CUDA device")
        if k_scales is None and v_scales is None:
            fmt, dtype, ks, vs = _lib.MK_KV_BF16, torch.bfloat16, None, None
        elif k_scales is None or v_scales is None:
            raise ValueError("an 8-bit cache needs both k_scales and v_scales")
        else:
            fmt, dtype = _lib.MK_KV_E4M3, torch.float8_e4m3fn
            ks = _check(k_scales, torch.uint8, "k_scales", dev, k_pages.shape[:3])
            vs = _check(v_scales, torch.uint8, "v_scales", dev, k_pages.shape[:3])
        k = _check(k_pages, dtype, "k_pages", dev)
        v = _check(v_pages, dtype, "v_pages", dev, k_pages.shape)
        if block_tables.dim() != 2:
            raise ValueError("block_tables must be [batch, max_blocks]")
        t = _check(block_tables, torch.int32, "block_tables", dev)
        self.k_pages, self.v_pages, self.block_tables = k_pages, v_pages, block_tables
        self.k_scales, self.v_scales, self.device = k_scales, v_scales, dev
        pages, self.num_kv_heads, self.page_size, _ = k_pages.shape
        self.batch, self.max_blocks = block_tables.shape
        self.struct = _lib.MkKVLayer(k, v, ks, vs, t, fmt, pages, self.page_size,
                                     self.num_kv_heads, self.max_blocks)
        self.ref = ctypes.byref(self.struct)


def kv_write(layer: KVLayer, qkv, rope_cos, rope_sin, seqs, slots, positions, q_out,
             error=None) -> torch.Tensor:
    """Rotate ``qkv`` [rows, (nq + 2 nkv) * 64] (bf16, packed RoPE-pair order), store
    each row's K/V at place ``slots[r]`` of sequence ``seqs[r]`` (int32; slot -1: a
    padding row) and write its q into ``q_out`` [rows, nq, 64]; ``positions`` are
    the RoPE positions. Returns ``q_out``."""
    dev = layer.device
    rows, nq = q_out.shape[0], q_out.shape[1]
    q = _check(q_out, torch.bfloat16, "q_out", dev, (rows, nq, 64))
    x = _check(qkv, torch.bfloat16, "qkv", dev, (rows, (nq + 2 * layer.num_kv_heads) * 64))
    rope_len = rope_cos.shape[0]
    c = _check(rope_cos, torch.bfloat16, "rope_cos", dev, (rope_len, 64))
    s = _check(rope_sin, torch.bfloat16, "rope_sin", dev, (rope_len, 64))
    sq = _check(seqs, torch.int32, "seqs", dev, (rows,))
    sl = _check(slots, torch.int32, "slots", dev, (rows,))
    ps = _check(positions, torch.int32, "positions", dev, (rows,))
    error = _error_word(error, dev)
    _call(_lib.load().mk_kv_write, dev, layer.ref, layer.batch, x, c, s, rope_len, sq, sl, ps, rows, nq, q,
          _check(error, torch.int32, "error", dev))
    return q_out


def kv_read(layer: KVLayer, lengths, max_len: int, k_out=None, v_out=None, error=None):
    """Positions [0, lengths[b]) of every sequence as bf16 [batch, nkv, max_len, 64]
    (K, V), zeros behind them."""
    dev = layer.device
    n = lengths.shape[0]
    if n > layer.batch:
        raise ValueError(f"{n} lengths for a table of {layer.batch} sequences")
    shape = (n, layer.num_kv_heads, max_len, 64)
    if k_out is None:
        k_out = torch.empty(shape, dtype=torch.bfloat16, device=dev)
    if v_out is None:
        v_out = torch.empty(shape, dtype=torch.bfloat16, device=dev)
    error = _error_word(error, dev)
    _call(_lib.load().mk_kv_read, dev, layer.ref, _check(lengths, torch.int32, "lengths", dev, (n,)), n, max_len,
          _check(k_out, torch.bfloat16, "k_out", dev, shape),
          _check(v_out, torch.bfloat16, "v_out", dev, shape), _check(error, torch.int32, "error", dev))
    return k_out, v_out


def tree_attention(q, layer: KVLayer, cu_nodes, mask, prefix_lens, max_nodes: int, max_len: int,
                   scale: float | None = None, out=None, lse=None, workspace=None, error=None):
    """Attention of the drafted nodes ``q`` [rows, nq, 64] (rotated, bf16) over the
    cache: sequence b has ``prefix_lens[b]`` committed positions and the nodes
    ``cu_nodes[b]`` .. ``cu_nodes[b + 1] - 1``, whose K/V rows are already stored
    behind them. ``mask`` [rows, ceil(max_nodes / 64)] int64: bit j of a node's row
    set when it sees node j of its sequence. ``max_nodes`` (<= 256) and ``max_len``
    bound every sequence's nodes and prefix + nodes. Returns (out [rows, nq, 64]
    bf16, lse [rows, nq] fp32); a node that sees nothing gets 0 and -inf."""
    dev = layer.device
    rows, nq = q.shape[0], q.shape[1]
    shape = (rows, nq, 64)
    n = prefix_lens.shape[0]
    if n > layer.batch:
        raise ValueError(f"{n} sequences for a table of {layer.batch}")
    if out is None:
        out = torch.empty(shape, dtype=torch.bfloat16, device=dev)
    if lse is None:
        lse = torch.empty((rows, nq), dtype=torch.float32, device=dev)
    error = _error_word(error, dev)
    lib = _lib.load()
    nbytes = lib.mk_tree_attention_workspace(n, nq, layer.num_kv_heads, max_nodes, max_len)
    if workspace is None and nbytes:
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    wp, wn = (0, 0) if workspace is None else (_check(workspace, torch.uint8, "workspace", dev),
                                               workspace.numel())
    _call(lib.mk_tree_attention, dev, _check(q, torch.bfloat16, "q", dev, shape), layer.ref,
          _check(cu_nodes, torch.int32, "cu_nodes", dev, (n + 1,)),
          _check(mask, torch.int64, "mask", dev, (rows, (max_nodes + 63) // 64)),
          _check(prefix_lens, torch.int32, "prefix_lens", dev), n, rows, max_nodes, max_len, nq,
          0.125 if scale is None else scale, wp, wn, _check(out, torch.bfloat16, "out", dev, shape),
          _check(lse, torch.float32, "lse", dev, (rows, nq)), _check(error, torch.int32, "error", dev))
    return out, lse


def token_logprobs(logits, targets=None, top: int = 0, logprobs=None, entropy=None, top_ids=None,
                   top_logprobs=None, workspace=None, error=None):
    """From ``logits`` [rows, vocab] (fp32 or bf16; rows may be strided): the log
    probabilities of ``targets`` [rows, n] (int32, negative: no token, 0), the
    entropy of every row in nats, and the ``top`` (<= 32) most likely ids with
    their log probabilities (ties to the lower id). Returns (logprobs [rows, n],
    entropy [rows], top_ids [rows, top] int32, top_logprobs [rows, top])."""
    dev = logits.device
    if dev.type != "cuda":
        raise ValueError("logits must be on a CUDA device")
    if logits.dim() != 2 or (logits.shape[0] > 1 and logits.stride(0) < logits.shape[1]) or logits.stride(1) != 1:
        raise ValueError("logits must be [rows, vocab] with contiguous, non-overlapping rows")
    if logits.dtype == torch.float32:
        dtype = _lib.MK_F32
    elif logits.dtype == torch.bfloat16:
        dtype = _lib.MK_BF16
    else:
        raise ValueError(f"logits must be fp32 or bf16, got {logits.dtype}")
    rows, vocab = logits.shape
    n = 0 if targets is None else targets.shape[1]
    f32 = dict(dtype=torch.float32, device=dev)
    if logprobs is None:
        logprobs = torch.empty((rows, n), **f32)
    if entropy is None:
        entropy = torch.empty(rows, **f32)
    if top_ids is None:
        top_ids = torch.empty((rows, top), dtype=torch.int32, device=dev)
    if top_logprobs is None:
        top_logprobs = torch.empty((rows, top), **f32)
    error = _error_word(error, dev)
    lib = _lib.load()
    nbytes = lib.mk_token_logprobs_workspace(rows, vocab, top)
    if workspace is None and nbytes:
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    wp, wn = (0, 0) if workspace is None else (_check(workspace, torch.uint8, "workspace", dev),
                                               workspace.numel())
    _call(lib.mk_token_logprobs, dev, logits.data_ptr(), dtype, rows, vocab,
          max(logits.stride(0), vocab) if rows < 2 else logits.stride(0),
          _check(targets, torch.int32, "targets", dev, (rows, n)) if n else None, n, top, wp, wn,
          _check(logprobs, torch.float32, "logprobs", dev, (rows, n)) if n else None,
          _check(entropy, torch.float32, "entropy", dev, (rows,)),
          _check(top_ids, torch.int32, "top_ids", dev, (rows, top)) if top else None,
          _check(top_logprobs, torch.float32, "top_logprobs", dev, (rows, top)) if top else None,
          _check(error, torch.int32, "error", dev))
    return logprobs, entropy, top_ids, top_logprobs
