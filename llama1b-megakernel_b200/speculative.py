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


_raw_stream = torch._C._cuda_getCurrentRawStream  # the current stream of a device index, as a number
_BF16, _F32, _I32, _I64, _U8 = torch.bfloat16, torch.float32, torch.int32, torch.int64, torch.uint8


def _check(t: torch.Tensor, dtype, name: str, index: int, shape=None) -> int:
    """The tensor's address, once its type, device, layout and shape fit."""
    if t.dtype is dtype and t.get_device() == index and t.is_contiguous() and (shape is None or t.shape == shape):
        return t.data_ptr()
    if t.dtype is not dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if t.get_device() != index:
        raise ValueError(f"{name} is on {t.device}, the cache or logits on cuda:{index}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")


def _call(fn, index: int, *args) -> None:
    """Run an entry point on the current stream of device ``index``."""
    if index == torch.cuda.current_device():
        status = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = fn(*args, _raw_stream(index))
    if status:
        _lib.check(status)


def _error_word(error: torch.Tensor | None, dev) -> torch.Tensor:
    return torch.zeros(1, dtype=_I32, device=dev) if error is None else error


class KVLayer:
    """One layer of a paged cache, as the operators take it: pages [num_pages, nkv,
    page_size, 64] (bf16, or ``torch.float8_e4m3fn`` with uint8 scale bytes
    [num_pages, nkv, page_size]) and block tables [batch, max_blocks] int32.
    Holds references to the tensors; make it once per layer
    (``PagedKVCache.layer``) or per call."""

    __slots__ = ("k_pages", "v_pages", "block_tables", "k_scales", "v_scales", "device", "index",
                 "batch", "num_kv_heads", "page_size", "struct", "ref")

    def __init__(self, k_pages, v_pages, block_tables, k_scales=None, v_scales=None):
        shape = k_pages.shape
        if len(shape) != 4 or shape[3] != 64:
            raise ValueError(f"pages must be [num_pages, kv heads, page_size, 64], got {tuple(shape)}")
        index = k_pages.get_device()
        if index < 0:
            raise ValueError("the cache must be on a CUDA device")
        pages, heads, page_size, _ = shape
        if k_scales is None and v_scales is None:
            fmt, dtype, ks, vs = _lib.MK_KV_BF16, _BF16, None, None
        elif k_scales is None or v_scales is None:
            raise ValueError("an 8-bit cache needs both k_scales and v_scales")
        else:
            fmt, dtype = _lib.MK_KV_E4M3, torch.float8_e4m3fn
            ks = _check(k_scales, _U8, "k_scales", index, (pages, heads, page_size))
            vs = _check(v_scales, _U8, "v_scales", index, (pages, heads, page_size))
        k = _check(k_pages, dtype, "k_pages", index)
        v = _check(v_pages, dtype, "v_pages", index, shape)
        t = _check(block_tables, _I32, "block_tables", index)
        if block_tables.dim() != 2:
            raise ValueError("block_tables must be [batch, max_blocks]")
        self.k_pages, self.v_pages, self.block_tables = k_pages, v_pages, block_tables
        self.k_scales, self.v_scales, self.device, self.index = k_scales, v_scales, k_pages.device, index
        self.num_kv_heads, self.page_size = heads, page_size
        self.batch, max_blocks = block_tables.shape
        self.struct = _lib.MkKVLayer(k, v, ks, vs, t, fmt, pages, page_size, heads, max_blocks)
        self.ref = ctypes.byref(self.struct)


def kv_write(layer: KVLayer, qkv, rope_cos, rope_sin, seqs, slots, positions, q_out,
             error=None) -> torch.Tensor:
    """Rotate ``qkv`` [rows, (nq + 2 nkv) * 64] (bf16, packed RoPE-pair order), store
    each row's K/V at place ``slots[r]`` of sequence ``seqs[r]`` (int32; slot -1: a
    padding row) and write its q into ``q_out`` [rows, nq, 64]; ``positions`` are
    the RoPE positions. Returns ``q_out``."""
    index = layer.index
    rows, nq, _ = shape = q_out.shape
    per_row = (rows,)
    rope_len = rope_cos.shape[0]
    if shape[2] != 64:
        raise ValueError(f"q_out must be [rows, query heads, 64], got {tuple(shape)}")
    error = _error_word(error, layer.device)
    _call(_lib.load().mk_kv_write, index, layer.ref, layer.batch,
          _check(qkv, _BF16, "qkv", index, (rows, (nq + 2 * layer.num_kv_heads) * 64)),
          _check(rope_cos, _BF16, "rope_cos", index, (rope_len, 64)),
          _check(rope_sin, _BF16, "rope_sin", index, (rope_len, 64)), rope_len,
          _check(seqs, _I32, "seqs", index, per_row), _check(slots, _I32, "slots", index, per_row),
          _check(positions, _I32, "positions", index, per_row), rows, nq,
          _check(q_out, _BF16, "q_out", index), _check(error, _I32, "error", index))
    return q_out


def kv_read(layer: KVLayer, lengths, max_len: int, k_out=None, v_out=None, error=None):
    """Positions [0, lengths[b]) of every sequence as bf16 [batch, nkv, max_len, 64]
    (K, V), zeros behind them."""
    index, dev = layer.index, layer.device
    n = lengths.shape[0]
    if n > layer.batch:
        raise ValueError(f"{n} lengths for a table of {layer.batch} sequences")
    shape = (n, layer.num_kv_heads, max_len, 64)
    if k_out is None:
        k_out = torch.empty(shape, dtype=_BF16, device=dev)
    if v_out is None:
        v_out = torch.empty_like(k_out)
    error = _error_word(error, dev)
    _call(_lib.load().mk_kv_read, index, layer.ref, _check(lengths, _I32, "lengths", index, (n,)), n, max_len,
          _check(k_out, _BF16, "k_out", index, shape), _check(v_out, _BF16, "v_out", index, shape),
          _check(error, _I32, "error", index))
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
    index, dev = layer.index, layer.device
    rows, nq, _ = shape = q.shape
    if shape[2] != 64:
        raise ValueError(f"q must be [rows, query heads, 64], got {tuple(shape)}")
    n = prefix_lens.shape[0]
    if n > layer.batch:
        raise ValueError(f"{n} sequences for a table of {layer.batch}")
    at = _check(q, _BF16, "q", index)
    if out is None:
        out = torch.empty_like(q)
    if lse is None:
        lse = q.new_empty((rows, nq), dtype=_F32)
    error = _error_word(error, dev)
    lib = _lib.load()
    if workspace is None:
        nbytes = lib.mk_tree_attention_workspace(n, nq, layer.num_kv_heads, max_nodes, max_len)
        wp = 0
        if nbytes:
            workspace = torch.empty(nbytes, dtype=_U8, device=dev)
            wp = workspace.data_ptr()
    else:
        wp, nbytes = _check(workspace, _U8, "workspace", index), workspace.numel()
    _call(lib.mk_tree_attention, index, at, layer.ref, _check(cu_nodes, _I32, "cu_nodes", index, (n + 1,)),
          _check(mask, _I64, "mask", index, (rows, (max_nodes + 63) // 64)),
          _check(prefix_lens, _I32, "prefix_lens", index), n, rows, max_nodes, max_len, nq,
          0.125 if scale is None else scale, wp, nbytes, _check(out, _BF16, "out", index, shape),
          _check(lse, _F32, "lse", index, (rows, nq)), _check(error, _I32, "error", index))
    return out, lse


def token_logprobs(logits, targets=None, top: int = 0, logprobs=None, entropy=None, top_ids=None,
                   top_logprobs=None, workspace=None, error=None):
    """From ``logits`` [rows, vocab] (fp32 or bf16; rows may be strided): the log
    probabilities of ``targets`` [rows, n] (int32, negative: no token, 0), the
    entropy of every row in nats, and the ``top`` (<= 32) most likely ids with
    their log probabilities (ties to the lower id). Returns (logprobs [rows, n],
    entropy [rows], top_ids [rows, top] int32, top_logprobs [rows, top])."""
    index = logits.get_device()
    if index < 0:
        raise ValueError("logits must be on a CUDA device")
    if logits.dim() != 2:
        raise ValueError(f"logits must be [rows, vocab], got {tuple(logits.shape)}")
    rows, vocab = logits.shape
    ld, step = logits.stride()
    if rows < 2:
        ld = vocab
    if step != 1 and vocab > 1 or ld < vocab:
        raise ValueError("logits must have contiguous, non-overlapping rows")
    if logits.dtype is _F32:
        dtype = _lib.MK_F32
    elif logits.dtype is _BF16:
        dtype = _lib.MK_BF16
    else:
        raise ValueError(f"logits must be fp32 or bf16, got {logits.dtype}")
    n = 0 if targets is None else targets.shape[1]
    if logprobs is None:
        logprobs = logits.new_empty((rows, n), dtype=_F32)
    if entropy is None:
        entropy = logits.new_empty(rows, dtype=_F32)
    if top_ids is None:
        top_ids = logits.new_empty((rows, top), dtype=_I32)
    if top_logprobs is None:
        top_logprobs = logits.new_empty((rows, top), dtype=_F32)
    error = _error_word(error, logits.device)
    lib = _lib.load()
    if workspace is None:
        nbytes = lib.mk_token_logprobs_workspace(rows, vocab, top)
        wp = 0
        if nbytes:
            workspace = logits.new_empty(nbytes, dtype=_U8)
            wp = workspace.data_ptr()
    else:
        wp, nbytes = _check(workspace, _U8, "workspace", index), workspace.numel()
    _call(lib.mk_token_logprobs, index, logits.data_ptr(), dtype, rows, vocab, ld,
          _check(targets, _I32, "targets", index, (rows, n)) if n else None, n, top, wp, nbytes,
          _check(logprobs, _F32, "logprobs", index, (rows, n)) if n else None,
          _check(entropy, _F32, "entropy", index, (rows,)),
          _check(top_ids, _I32, "top_ids", index, (rows, top)) if top else None,
          _check(top_logprobs, _F32, "top_logprobs", index, (rows, top)) if top else None,
          _check(error, _I32, "error", index))
    return logprobs, entropy, top_ids, top_logprobs
