"""Paged bf16 KV cache: the ``past_key_values`` object of the decode path.

The reference keeps one contiguous [1, 8, S_MAX=1024, 64] cache per layer in
NxDI's KV manager, a flat list [K0, V0, K1, V1, ...] that its kernel updates in
place (llama_with_megakernel.py:134-139, nki_kernels/attention.py:450-492).
Here the cache is paged so context length is bounded by the pool, not by a
per-sequence S_MAX:

* ``k_pages`` / ``v_pages``: [num_layers, num_pages, num_kv_heads, page_size,
  head_dim] bf16. One page holds ``page_size`` consecutive positions of one
  sequence for every kv head; a head's rows in a page are contiguous, so the
  kernel fetches them with a single bulk copy.
* ``block_tables``: [max_batch, max_blocks] int32, logical block -> page id,
  shared by all layers. Position p of sequence b is slot p % page_size of
  page ``block_tables[b, p // page_size]``.

The kernel writes each new K/V row in place at its position and reads
positions [0, pos) for attention.

``QuantizedPagedKVCache`` keeps e4m3 codes and a power-of-two scale byte for
each (position, kv head) instead, 65 bytes a row where bf16 takes 128; the
operators of ``speculative.py`` read and write both.
"""
from __future__ import annotations

import torch

from .config import LlamaDecodeConfig


class PagedKVCache:
    def __init__(self, cfg: LlamaDecodeConfig, max_batch: int, max_seq_len: int,
                 page_size: int = 64, num_pages: int | None = None, device="cuda"):
        if page_size % 8:
            raise ValueError("page_size must be a multiple of 8")
        self.cfg = cfg
        self.page_size = page_size
        self.max_batch = max_batch
        self.max_seq_len = max_seq_len
        self.max_blocks = (max_seq_len + page_size - 1) // page_size
        if num_pages is None:
            num_pages = max_batch * self.max_blocks
        self.num_pages = num_pages
        self.device = torch.device(device)
        self._allocate((cfg.num_layers, num_pages, cfg.num_kv_heads, page_size, cfg.head_dim))
        self.block_tables = torch.full((max_batch, self.max_blocks), -1, dtype=torch.int32,
                                       device=self.device)
        self._host_tables = [[] for _ in range(max_batch)]
        self._free = list(range(num_pages - 1, -1, -1))
        self.seq_lens = [0] * max_batch

    # ------------------------------------------------------------ allocation
    def _allocate(self, shape) -> None:
        self.k_pages = torch.zeros(shape, dtype=torch.bfloat16, device=self.device)
        self.v_pages = torch.zeros(shape, dtype=torch.bfloat16, device=self.device)

    def layer(self, index: int):
        """Layer ``index`` as the operators of ``speculative.py`` take it (the pools
        never move, so it stays valid)."""
        from .speculative import KVLayer

        return KVLayer(self.k_pages[index], self.v_pages[index], self.block_tables)

    def reserve(self, seq: int, length: int) -> None:
        """Make positions [0, length) of sequence ``seq`` addressable."""
        if length > self.max_blocks * self.page_size:
            raise ValueError(f"length {length} exceeds max_seq_len {self.max_seq_len}")
        need = (length + self.page_size - 1) // self.page_size
        table = self._host_tables[seq]
        more = need - len(table)
        if more > len(self._free):
            raise RuntimeError("KV page pool exhausted")
        if more > 0:
            table += [self._free.pop() for _ in range(more)]
            row = torch.tensor(table + [-1] * (self.max_blocks - len(table)), dtype=torch.int32)
            self.block_tables[seq].copy_(row.to(self.device))

    def reserve_all(self, lengths) -> None:
        """``reserve`` for sequences 0, 1, ... together: where one does not fit, none is."""
        if max(lengths) > self.max_blocks * self.page_size:
            raise ValueError(f"length {max(lengths)} exceeds max_seq_len {self.max_seq_len}")
        more = sum(max(0, -(-n // self.page_size) - len(table)) for n, table in zip(lengths, self._host_tables))
        if more > len(self._free):
            raise RuntimeError(f"KV page pool exhausted: {more} pages wanted, {len(self._free)} free")
        for seq, n in enumerate(lengths):
            self.reserve(seq, n)

    def room(self, seq: int) -> int:
        """Positions that sequence ``seq`` has pages for, the free ones counted."""
        return min(self.max_blocks, len(self._host_tables[seq]) + len(self._free)) * self.page_size

    def shuffle_free_pages(self, seed: int) -> None:
        """Hand out free pages in a seeded random order (exercises the page indirection)."""
        g = torch.Generator().manual_seed(seed)
        order = torch.randperm(len(self._free), generator=g).tolist()
        self._free = [self._free[i] for i in order]

    def release(self, seq: int) -> None:
        self._free.extend(reversed(self._host_tables[seq]))
        self._host_tables[seq] = []
        self.seq_lens[seq] = 0
        self.block_tables[seq].fill_(-1)

    def reset(self) -> None:
        for b in range(self.max_batch):
            self.release(b)

    def pages_of(self, seq: int) -> list[int]:
        return list(self._host_tables[seq])

    # ------------------------------------------------------------ contents
    def fill(self, seq: int, k_rows: torch.Tensor, v_rows: torch.Tensor) -> None:
        """Write positions [0, n) of ``seq`` from [num_layers, nkv, n, head_dim] tensors."""
        n = k_rows.shape[2]
        self.reserve(seq, n)
        ps = self.page_size
        table = self._host_tables[seq]
        for blk in range((n + ps - 1) // ps):
            p0, p1 = blk * ps, min(n, (blk + 1) * ps)
            page = table[blk]
            self.k_pages[:, page, :, : p1 - p0] = k_rows[:, :, p0:p1].to(self.device)
            self.v_pages[:, page, :, : p1 - p0] = v_rows[:, :, p0:p1].to(self.device)
        self.seq_lens[seq] = max(self.seq_lens[seq], n)

    def gather(self, seq: int, n: int) -> tuple[torch.Tensor, torch.Tensor]:
        """Rows [0, n) of ``seq`` as [num_layers, nkv, n, head_dim] (contiguous copy)."""
        ps = self.page_size
        nb = (n + ps - 1) // ps
        pages = torch.tensor(self._host_tables[seq][:nb], dtype=torch.long, device=self.device)
        L, _, nkv, _, hd = self.k_pages.shape
        k = self.k_pages[:, pages].permute(0, 2, 1, 3, 4).reshape(L, nkv, nb * ps, hd)[:, :, :n]
        v = self.v_pages[:, pages].permute(0, 2, 1, 3, 4).reshape(L, nkv, nb * ps, hd)[:, :, :n]
        return k.contiguous(), v.contiguous()

    def nbytes(self) -> int:
        return 2 * self.k_pages.numel() * 2


def encode_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows [..., head_dim] as ``mk_kv_write`` stores them in an 8-bit cache: e4m3 codes
    and the scale bytes [...] (exponent + 127 of the smallest power of two, at
    least 2^-110, with max|x| <= 448 times it; 255 for a row that is not finite)."""
    x = x.float()
    amax = x.abs().amax(-1)
    finite = torch.isfinite(x).all(-1)
    amax = torch.where(finite, amax, torch.ones_like(amax))
    frac, e2 = torch.frexp(amax)
    e = torch.where(amax > 0, e2 - 9 + (frac > 0.875).to(e2.dtype), torch.full_like(e2, -110)).clamp(min=-110)
    inv = ((127 - e.to(torch.int32)) << 23).view(torch.float32)  # 2^-e from its bits
    y = torch.where(finite[..., None], x * inv[..., None], torch.zeros_like(x))
    byte = torch.where(finite, e.to(torch.int32) + 127, torch.full_like(e, 255, dtype=torch.int32))
    return y.to(torch.float8_e4m3fn), byte.to(torch.uint8)


def decode_rows(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """What codes and scale bytes stand for, in bf16 (exact)."""
    byte = scales.to(torch.int32)
    f = (byte << 23).view(torch.float32)
    f = torch.where(byte == 0, torch.full_like(f, 2.0 ** -127), f)
    f = torch.where(byte == 255, torch.full_like(f, float("nan")), f)
    return (codes.float() * f[..., None]).to(torch.bfloat16)


class QuantizedPagedKVCache(PagedKVCache):
    """A paged cache of 8-bit rows: ``k_pages`` / ``v_pages`` hold e4m3 codes and
    ``k_scales`` / ``v_scales`` [num_layers, num_pages, num_kv_heads, page_size] one
    E8M0 byte per row. No counterpart in the reference, whose cache is bf16
    (llama_with_megakernel.py:134-139). Read and written by the operators of
    ``speculative.py``; the persistent kernel and the batched step take the bf16
    cache."""

    def _allocate(self, shape) -> None:
        self.k_pages = torch.zeros(shape, dtype=torch.float8_e4m3fn, device=self.device)
        self.v_pages = torch.zeros(shape, dtype=torch.float8_e4m3fn, device=self.device)
        self.k_scales = torch.full(shape[:-1], 17, dtype=torch.uint8, device=self.device)
        self.v_scales = torch.full(shape[:-1], 17, dtype=torch.uint8, device=self.device)

    def layer(self, index: int):
        from .speculative import KVLayer

        return KVLayer(self.k_pages[index], self.v_pages[index], self.block_tables, self.k_scales[index],
                       self.v_scales[index])

    def fill(self, seq: int, k_rows: torch.Tensor, v_rows: torch.Tensor) -> None:
        n = k_rows.shape[2]
        self.reserve(seq, n)
        ps, table = self.page_size, self._host_tables[seq]
        for pool, scales, rows in ((self.k_pages, self.k_scales, k_rows), (self.v_pages, self.v_scales, v_rows)):
            codes, byte = encode_rows(rows.to(self.device))
            for blk in range((n + ps - 1) // ps):
                p0, p1 = blk * ps, min(n, (blk + 1) * ps)
                pool.view(torch.uint8)[:, table[blk], :, : p1 - p0] = codes.view(torch.uint8)[:, :, p0:p1]
                scales[:, table[blk], :, : p1 - p0] = byte[:, :, p0:p1]
        self.seq_lens[seq] = max(self.seq_lens[seq], n)

    def gather(self, seq: int, n: int) -> tuple[torch.Tensor, torch.Tensor]:
        ps = self.page_size
        nb = (n + ps - 1) // ps
        pages = torch.tensor(self._host_tables[seq][:nb], dtype=torch.long, device=self.device)
        L, _, nkv, _, hd = self.k_pages.shape
        out = []
        for pool, scales in ((self.k_pages, self.k_scales), (self.v_pages, self.v_scales)):
            codes = pool.view(torch.uint8)[:, pages].view(torch.float8_e4m3fn)
            x = decode_rows(codes, scales[:, pages])
            out.append(x.permute(0, 2, 1, 3, 4).reshape(L, nkv, nb * ps, hd)[:, :, :n].contiguous())
        return out[0], out[1]

    def nbytes(self) -> int:
        return 2 * (self.k_pages.numel() + self.k_scales.numel())
