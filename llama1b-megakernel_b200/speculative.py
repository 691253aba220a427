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

``SpeculativeDecoder`` runs them together: prompts and drafted trees go through a
model's layers (the projections, norms and SwiGLU are the batched step's kernels),
every node is scored for its children, and accepted nodes stay in the cache.

All run asynchronously on the current stream of their tensors' device, allocate
outputs and workspaces that are not passed in from PyTorch's allocator, and raise
``ValueError`` on tensors that do not fit and ``MkError`` on sizes that the library
refuses. What only the device can see (a page id, a length or a token out of range)
sets the caller's ``error`` word, an int32 tensor of one zero that the caller reads
when it synchronises; a call without one has nobody to tell, and such a row is wrong
without a word.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from functools import lru_cache

import torch

from . import _lib
from .kv_cache import PagedKVCache, QuantizedPagedKVCache


# A call of these operators is a few microseconds of host time beside as much of kernel,
# so its Python is kept short: tensors made here are not checked again, and new_empty
# takes its sizes one by one (0.6 us less than as a tuple).
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


@lru_cache(maxsize=256)
def _tree_workspace(batch: int, nq: int, nkv: int, max_nodes: int, max_len: int, index: int) -> int:
    """Bytes; of the sizes (and the device's SMs) alone, as every argument that it is given."""
    with torch.cuda.device(index):
        return _lib.load().mk_tree_attention_workspace(batch, nq, nkv, max_nodes, max_len)


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
    n, = lengths.shape
    if n > layer.batch:
        raise ValueError(f"{n} lengths for a table of {layer.batch} sequences")
    shape = (n, layer.num_kv_heads, max_len, 64)
    at = _check(lengths, _I32, "lengths", index, (n,))
    if k_out is None:
        k_out = lengths.new_empty(*shape, dtype=_BF16)
        kp = k_out.data_ptr()
    else:
        kp = _check(k_out, _BF16, "k_out", index, shape)
    if v_out is None:
        v_out = torch.empty_like(k_out)
        vp = v_out.data_ptr()
    else:
        vp = _check(v_out, _BF16, "v_out", index, shape)
    error = _error_word(error, dev)
    _call(_lib.load().mk_kv_read, index, layer.ref, at, n, max_len, kp, vp, _check(error, _I32, "error", index))
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
    n, = prefix_lens.shape
    if n > layer.batch:
        raise ValueError(f"{n} sequences for a table of {layer.batch}")
    at = _check(q, _BF16, "q", index)
    if out is None:
        out = torch.empty_like(q)
        op = out.data_ptr()
    else:
        op = _check(out, _BF16, "out", index, shape)
    if lse is None:
        lse = q.new_empty(rows, nq, dtype=_F32)
        lp = lse.data_ptr()
    else:
        lp = _check(lse, _F32, "lse", index, (rows, nq))
    error = _error_word(error, dev)
    lib = _lib.load()
    if workspace is None:
        nbytes, wp = _tree_workspace(n, nq, layer.num_kv_heads, max_nodes, max_len, index), 0
        if nbytes:
            workspace = q.new_empty(nbytes, dtype=_U8)
            wp = workspace.data_ptr()
    else:
        wp, nbytes = _check(workspace, _U8, "workspace", index), workspace.numel()
    _call(lib.mk_tree_attention, index, at, layer.ref, _check(cu_nodes, _I32, "cu_nodes", index, (n + 1,)),
          _check(mask, _I64, "mask", index, (rows, (max_nodes + 63) // 64)),
          _check(prefix_lens, _I32, "prefix_lens", index), n, rows, max_nodes, max_len, nq,
          0.125 if scale is None else scale, wp, nbytes, op, lp, _check(error, _I32, "error", index))
    return out, lse


def token_logprobs(logits, targets=None, top: int = 0, logprobs=None, entropy=None, top_ids=None,
                   top_logprobs=None, error=None):
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
    _, n = (rows, 0) if targets is None else targets.shape
    if logprobs is None:
        logprobs = logits.new_empty(rows, n, dtype=_F32)
        lp = logprobs.data_ptr()
    else:
        lp = _check(logprobs, _F32, "logprobs", index, (rows, n)) if n else None
    if entropy is None:
        entropy = logits.new_empty(rows, dtype=_F32)
        ep = entropy.data_ptr()
    else:
        ep = _check(entropy, _F32, "entropy", index, (rows,))
    if top_ids is None:
        top_ids = logits.new_empty(rows, top, dtype=_I32)
        ip = top_ids.data_ptr()
    else:
        ip = _check(top_ids, _I32, "top_ids", index, (rows, top)) if top else None
    if top_logprobs is None:
        top_logprobs = logits.new_empty(rows, top, dtype=_F32)
        tp = top_logprobs.data_ptr()
    else:
        tp = _check(top_logprobs, _F32, "top_logprobs", index, (rows, top)) if top else None
    error = _error_word(error, logits.device)
    _call(_lib.load().mk_token_logprobs, index, logits.data_ptr(), dtype, rows, vocab, ld,
          _check(targets, _I32, "targets", index, (rows, n)) if n else None, n, top, None, 0,
          lp if n else None, ep, ip if top else None, tp if top else None, _check(error, _I32, "error", index))
    return logprobs, entropy, top_ids, top_logprobs


# ---------------------------------------------------------------- drafts
class DraftTree:
    """Drafted tokens of one sequence: ``tokens[i]`` continues ``tokens[parents[i]]``, or
    the committed sequence where the parent is -1; a parent comes before its
    children. ``DraftTree.chain(tokens)`` is a plain continuation."""

    def __init__(self, tokens, parents):
        self.tokens = [int(t) for t in tokens]
        self.parents = [int(p) for p in parents]
        if len(self.tokens) != len(self.parents):
            raise ValueError(f"{len(self.tokens)} tokens, {len(self.parents)} parents")
        for i, p in enumerate(self.parents):
            if not -1 <= p < i:
                raise ValueError(f"node {i}: parent {p} is neither -1 nor a node before it")

    @classmethod
    def chain(cls, tokens) -> "DraftTree":
        tokens = list(tokens)
        return cls(tokens, range(-1, len(tokens) - 1))

    def __len__(self) -> int:
        return len(self.tokens)

    def depths(self) -> list[int]:
        out: list[int] = []
        for p in self.parents:
            out.append(0 if p < 0 else out[p] + 1)
        return out

    def masks(self) -> list[int]:
        """Bit j of node i's mask: j is i or an ancestor of it."""
        out: list[int] = []
        for i, p in enumerate(self.parents):
            out.append((out[p] if p >= 0 else 0) | 1 << i)
        return out

    def children(self) -> list[list[int]]:
        """The children of every node, and of the committed sequence at the end of the list."""
        out: list[list[int]] = [[] for _ in range(len(self) + 1)]
        for i, p in enumerate(self.parents):
            out[p].append(i)
        return out


def mask_words(masks: list[int], max_nodes: int) -> torch.Tensor:
    """Masks as ``tree_attention`` takes them: [nodes, ceil(max_nodes / 64)] int64 (CPU)."""
    words = (max_nodes + 63) // 64
    rows = []
    for m in masks:
        row = [(m >> (64 * w)) & 0xFFFFFFFFFFFFFFFF for w in range(words)]
        rows.append([x - (1 << 64) if x >> 63 else x for x in row])
    return torch.tensor(rows, dtype=torch.int64).reshape(len(masks), words)


@dataclass
class TreeScores:
    """What a pass over drafted trees gives, a row per node, sequences one after the
    other (``first[b]`` is sequence b's first row)."""

    first: list[int]
    logits: torch.Tensor         # [rows, vocab] fp32, after each node
    child_logprobs: torch.Tensor  # [rows, most children] of the node's children, in order (0: none)
    entropy: torch.Tensor        # [rows]
    top_ids: torch.Tensor        # [rows, top]
    top_logprobs: torch.Tensor   # [rows, top]


class SpeculativeDecoder:
    """Decoding several drafted tokens per pass with the weights of ``model`` (a
    single-GPU ``MegakernelLlamaForCausalLM``), over a cache of its own: 8-bit rows
    (``cache="e4m3"``) or bf16.

    ``score`` takes one tree of at most ``max_nodes`` nodes per sequence (128 nodes
    over all sequences), runs them through the model and returns every node's
    logits, the log probabilities of its children, its entropy and ``top``
    alternatives; the nodes' K/V rows then lie behind the committed ones.
    ``commit`` keeps an accepted path of them, ``accept_greedy`` finds the longest
    one the model itself would have taken. ``prefill`` runs prompts as causal
    chains, ``generate`` is greedy decoding with a drafting function."""

    MAX_ROWS = 128  # the GEMM's largest padded row count

    def __init__(self, model, max_batch: int, max_seq_len: int, max_nodes: int = 64, page_size: int = 64,
                 num_pages: int | None = None, cache: str = "e4m3", top: int = 4):
        if getattr(model, "tp_world", 1) != 1:
            raise NotImplementedError("SpeculativeDecoder runs on a single-GPU model")
        if not 1 <= max_nodes <= self.MAX_ROWS:
            raise ValueError(f"max_nodes {max_nodes} outside [1, {self.MAX_ROWS}]")
        if not 1 <= top <= 32:
            raise ValueError(f"top {top} outside [1, 32]")
        if max_seq_len > model.rope_len:
            raise ValueError(f"max_seq_len {max_seq_len} exceeds the model's RoPE table ({model.rope_len} positions)")
        kinds = {"e4m3": QuantizedPagedKVCache, "bf16": PagedKVCache}
        if cache not in kinds:
            raise ValueError(f"cache must be one of {sorted(kinds)}, got {cache!r}")
        self.m, self.cfg, self.lib, self.dev = model, model.cfg, model.lib, model.device
        self.max_batch, self.max_seq_len, self.max_nodes, self.top = max_batch, max_seq_len, max_nodes, top
        self.kv = kinds[cache](self.cfg, max_batch, max_seq_len, page_size, num_pages, device=self.dev)
        self.layers = [self.kv.layer(i) for i in range(self.cfg.num_layers)]
        self.err = torch.zeros(1, dtype=torch.int32, device=self.dev)
        c, z = self.cfg, lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device=self.dev)  # noqa: E731
        R, nh = self.MAX_ROWS, c.num_q_heads + 2 * c.num_kv_heads
        # the first three feed GEMMs, whose padded rows have to be finite: they start as zeros
        self._h, self._attn, self._act = z(R, c.hidden), z(R, c.num_q_heads * 64), z(R, c.intermediate)
        self._qkv, self._q, self._gu = z(R, nh * 64), z(R, c.num_q_heads, 64), z(R, 2 * c.intermediate)
        self._pending: list[DraftTree | None] = [None] * max_batch

    # ------------------------------------------------------------------ one pass
    def _admit(self, tokens: list[list[int]]) -> None:
        """Pages for each sequence's new tokens behind its committed positions. What does not
        fit is refused before anything has changed."""
        lengths = [self.kv.seq_lens[b] + len(t) for b, t in enumerate(tokens)]
        for b, (t, n) in enumerate(zip(tokens, lengths)):
            if n > self.max_seq_len:
                raise ValueError(f"sequence {b}: {n - len(t)} + {len(t)} positions exceed max_seq_len {self.max_seq_len}")
            if t and not 0 <= min(t) <= max(t) < self.cfg.vocab:
                raise ValueError(f"sequence {b}: token id outside the vocabulary")
        self.kv.reserve_all(lengths)

    def _gemm(self, w, x, rows, out=None, out_f32=None, residual=None):
        n, k = w.shape
        pad = 16 if rows <= 16 else 32 if rows <= 32 else 64 if rows <= 64 else 128
        _lib.check(self.lib.mk_gemm_bf16(
            w.data_ptr(), n, k, x.data_ptr(), rows, pad, residual.data_ptr() if residual is not None else None,
            out.data_ptr() if out is not None else None, out_f32.data_ptr() if out_f32 is not None else None,
            None, 0, self.err.data_ptr(), torch.cuda.current_stream(self.dev).cuda_stream))

    @torch.no_grad()
    def _forward(self, trees: list[DraftTree]) -> torch.Tensor:
        """The nodes of one tree per sequence (after ``_admit``) through the layers, their K/V
        behind the committed positions; the residual stream [rows, hidden] after the last."""
        c, pw, lib, kv, dev = self.cfg, self.m.packed, self.lib, self.kv, self.dev
        sizes = [len(t) for t in trees]
        rows = sum(sizes)
        base = [kv.seq_lens[b] for b in range(len(trees))]
        T = max(sizes)
        max_len = max(p + n for p, n in zip(base, sizes))
        seqs = [b for b, n in enumerate(sizes) for _ in range(n)]
        slots = [base[b] + i for b, n in enumerate(sizes) for i in range(n)]
        positions = [base[b] + d for b, t in enumerate(trees) for d in t.depths()]
        tokens = [x for t in trees for x in t.tokens]
        cu = [sum(sizes[:b]) for b in range(len(sizes) + 1)]
        ints = torch.tensor(tokens + seqs + slots + positions + cu + base, dtype=torch.int32).to(dev)
        tokens, seqs, slots, positions = (ints[i * rows:(i + 1) * rows] for i in range(4))
        cu, prefix = ints[4 * rows:4 * rows + len(cu)], ints[4 * rows + len(cu):]
        mask = mask_words([m for t in trees for m in t.masks()], T).to(dev)
        st = torch.cuda.current_stream(dev).cuda_stream
        H, I, eps = c.hidden, c.intermediate, ctypes.c_float(c.rms_eps)
        x = pw.embed[tokens.long()].contiguous()
        qkv, q, attn = self._qkv[:rows], self._q[:rows], self._attn[:rows].view(rows, c.num_q_heads, 64)
        nbytes = lib.mk_tree_attention_workspace(len(trees), c.num_q_heads, c.num_kv_heads, T, max_len)
        work = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=dev)
        lse = torch.empty(rows, c.num_q_heads, dtype=torch.float32, device=dev)
        for i, layer in enumerate(self.layers):
            _lib.check(lib.mk_rmsnorm_rows(x.data_ptr(), pw.norm_attn[i].data_ptr(), eps, rows, H,
                                           self._h.data_ptr(), st))
            self._gemm(pw.w_qkv[i].view(-1, H), self._h, rows, out=qkv)
            kv_write(layer, qkv, pw.rope_cos, pw.rope_sin, seqs, slots, positions, q, error=self.err)
            tree_attention(q, layer, cu, mask, prefix, T, max_len, scale=c.head_dim ** -0.5, out=attn, lse=lse,
                           workspace=work, error=self.err)
            self._gemm(pw.w_o[i], self._attn, rows, out=x, residual=x)
            _lib.check(lib.mk_rmsnorm_rows(x.data_ptr(), pw.norm_mlp[i].data_ptr(), eps, rows, H,
                                           self._h.data_ptr(), st))
            self._gemm(pw.w_gate_up[i].view(2 * I, H), self._h, rows, out=self._gu)
            _lib.check(lib.mk_swiglu(self._gu.data_ptr(), rows * I, self._act.data_ptr(), st))
            self._gemm(pw.w_down[i], self._act, rows, out=x, residual=x)
        return x

    def _logits(self, x: torch.Tensor) -> torch.Tensor:
        """fp32 logits of the rows of x, as many at a time as the buffer of normed rows holds."""
        c, pw = self.cfg, self.m.packed
        logits = torch.empty(x.shape[0], c.vocab, dtype=torch.float32, device=self.dev)
        for rows, out in zip(x.split(self.MAX_ROWS), logits.split(self.MAX_ROWS)):
            _lib.check(self.lib.mk_rmsnorm_rows(
                rows.data_ptr(), pw.norm_final.data_ptr(), ctypes.c_float(c.rms_eps), len(rows), c.hidden,
                self._h.data_ptr(), torch.cuda.current_stream(self.dev).cuda_stream))
            self._gemm(pw.embed, self._h, len(rows), out_f32=out)
        return logits

    # ------------------------------------------------------------------ API
    def prefill(self, prompts) -> torch.Tensor:
        """Commit one prompt per sequence (a list of 1-D token tensors or lists, any
        lengths), continuing from what each has; returns the fp32 logits [B, vocab]
        after each prompt's last token. Prompts that do not fit (``max_seq_len``, the
        page pool, the vocabulary) are refused before any is taken."""
        prompts = [torch.as_tensor(p).reshape(-1).tolist() for p in prompts]
        if not 1 <= len(prompts) <= self.max_batch or not all(prompts):
            raise ValueError(f"prefill takes 1 to {self.max_batch} prompts with at least one token each")
        if any(self._pending):
            raise ValueError("commit or drop the scored trees first")
        self._admit(prompts)
        done = [0] * len(prompts)
        last = torch.empty(len(prompts), self.cfg.hidden, dtype=torch.bfloat16, device=self.dev)
        while any(d < len(p) for d, p in zip(done, prompts)):
            room, trees = self.MAX_ROWS, []
            for p, d in zip(prompts, done):  # as many rows as the GEMM takes
                n = min(room, len(p) - d)
                trees.append(DraftTree.chain(p[d:d + n]))
                room -= n
            x = self._forward(trees)
            at = 0
            for b, t in enumerate(trees):
                at += len(t)
                done[b] += len(t)
                self.kv.seq_lens[b] += len(t)
                if len(t) and done[b] == len(prompts[b]):
                    last[b] = x[at - 1]
        return self._logits(last)

    def score(self, trees: list[DraftTree]) -> TreeScores:
        """Run one tree per sequence (at least one node each; usually node 0 is the
        last accepted token and the rest are drafts) and score it."""
        if not 1 <= len(trees) <= self.max_batch:
            raise ValueError(f"{len(trees)} trees for a cache of {self.max_batch} sequences")
        sizes = [len(t) for t in trees]
        if min(sizes) < 1 or max(sizes) > self.max_nodes or sum(sizes) > self.MAX_ROWS:
            raise ValueError(f"trees of {sizes} nodes: 1 to {self.max_nodes} each, {self.MAX_ROWS} together")
        self._admit([t.tokens for t in trees])
        logits = self._logits(self._forward(trees))
        kids = [t.children() for t in trees]
        most = max(1, max(len(k) for ks in kids for k in ks[:-1]))
        targets = [[t.tokens[j] for j in ks[i]] + [-1] * (most - len(ks[i]))
                   for t, ks in zip(trees, kids) for i in range(len(t))]
        targets = torch.tensor(targets, dtype=torch.int32).to(self.dev)
        lp, ent, ids, top = token_logprobs(logits, targets, min(self.top, self.cfg.vocab), error=self.err)
        self._pending[:len(trees)] = trees
        return TreeScores([sum(sizes[:b]) for b in range(len(sizes))], logits, lp, ent, ids, top)

    def commit(self, seq: int, path: list[int]) -> None:
        """Keep the nodes ``path`` (root first, each the parent of the next) of the tree
        scored for sequence ``seq``: their rows move to the next positions of the
        sequence. An empty path drops the tree."""
        tree = self._pending[seq]
        if tree is None:
            raise ValueError(f"sequence {seq} has no scored tree")
        for i, (node, parent) in enumerate(zip(path, [-1, *path])):
            if not 0 <= node < len(tree) or tree.parents[node] != parent:
                raise ValueError(f"path {path}: {node} is not a child of {parent}")
        kv, ps, base = self.kv, self.kv.page_size, self.kv.seq_lens[seq]
        moved = [(base + n, base + i) for i, n in enumerate(path) if n != i]
        if moved:
            table = kv.pages_of(seq)
            index = torch.tensor([[table[s // ps], s % ps, table[d // ps], d % ps] for s, d in moved]).to(self.dev)
            sp, so, dp, do = index.unbind(1)
            pools = [kv.k_pages, kv.v_pages]
            if isinstance(kv, QuantizedPagedKVCache):
                pools = [kv.k_pages.view(torch.uint8), kv.v_pages.view(torch.uint8), kv.k_scales, kv.v_scales]
            for pool in pools:  # the right side is a copy, so the moves do not meet
                pool[:, dp, :, do] = pool[:, sp, :, so]
        kv.seq_lens[seq] += len(path)
        self._pending[seq] = None

    def accept_greedy(self, scores: TreeScores, seq: int) -> tuple[list[int], int]:
        """The path of the tree scored for ``seq`` that greedy decoding takes, its first
        root included, and the token that follows it."""
        tree = self._pending[seq]
        if tree is None:
            raise ValueError(f"sequence {seq} has no scored tree")
        first = scores.first[seq]
        best = scores.top_ids[first:first + len(tree), 0].tolist()
        kids = tree.children()
        path = [0]
        while True:
            nxt = next((j for j in kids[path[-1]] if tree.tokens[j] == best[path[-1]]), None)
            if nxt is None:
                return path, best[path[-1]]
            path.append(nxt)

    def generate(self, prompt, max_new_tokens: int, draft=None) -> tuple[list[int], int]:
        """Greedy tokens after ``prompt`` (sequence 0, from an empty cache):
        ``draft(tokens)`` proposes a ``DraftTree`` of continuations of the tokens so
        far (None or empty: no draft). Returns (tokens, passes). What does not fit in
        ``max_seq_len`` or the page pool is refused before the first pass."""
        if self.kv.seq_lens[0]:
            raise ValueError("sequence 0 is not empty: release it first")
        tokens = torch.as_tensor(prompt).reshape(-1).tolist()
        start = len(tokens)
        most = start + max(max_new_tokens, 1) - 1  # the last token has no row in the cache
        if most > self.max_seq_len:
            raise ValueError(f"{start} + {max_new_tokens} tokens exceed max_seq_len {self.max_seq_len}")
        self.kv.reserve(0, most)
        tokens.append(int(self.prefill([tokens])[0].argmax()))
        passes = 1
        while len(tokens) - start < max_new_tokens:
            room = min(self.max_nodes - 1, min(self.max_seq_len, self.kv.room(0)) - self.kv.seq_lens[0] - 1)
            proposal = draft(tokens) if draft is not None else None
            if proposal is not None and len(proposal) and room > 0:
                n = min(len(proposal), room)  # parents come first, so a cut tree is a tree
                tree = DraftTree([tokens[-1], *proposal.tokens[:n]], [-1, *(p + 1 for p in proposal.parents[:n])])
            else:
                tree = DraftTree.chain(tokens[-1:])
            path, following = self.accept_greedy(self.score([tree]), 0)
            passes += 1
            tokens += [tree.tokens[i] for i in path[1:]] + [following]
            self.commit(0, path)
        self.check()
        return tokens[start:start + max_new_tokens], passes

    def release(self, seq: int) -> None:
        """Forget a sequence."""
        self.kv.release(seq)
        self._pending[seq] = None

    def check(self) -> None:
        """Wait for the device and raise ``MkError`` if it reported a failure."""
        torch.cuda.synchronize(self.dev)
        code = int(self.err[0])
        if code:
            self.err.zero_()
            what = ("a page id, length or token is out of range" if code == 1 else
                    f"a device-side wait ran out (code {code})")
            raise _lib.MkError(_lib.MK_EDEVICE, f"speculative pass: {what}")


def lookup_draft(tokens: list[int], longest: int = 3, count: int = 8) -> DraftTree | None:
    """Draft by looking the last tokens up in what came before: the continuation of
    the latest earlier occurrence of the last ``longest`` (or fewer) tokens."""
    for n in range(min(longest, len(tokens) - 1), 0, -1):
        tail = tokens[-n:]
        for i in range(len(tokens) - n - 1, -1, -1):
            if tokens[i:i + n] == tail:
                return DraftTree.chain(tokens[i + n:i + n + count])
    return None
