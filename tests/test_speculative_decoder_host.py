"""SpeculativeDecoder's host side on the CPU: a decoder whose passes are played by a stand-in, over a
cache in host memory."""
from __future__ import annotations

import types

import pytest
import torch

from llama1b_megakernel_b200.config import TINY
from llama1b_megakernel_b200.kv_cache import QuantizedPagedKVCache
from llama1b_megakernel_b200.speculative import DraftTree, SpeculativeDecoder


class Recorder:
    """Stands in for the library: notes the rows that each call is told to write."""

    def __init__(self):
        self.rows = []

    def mk_rmsnorm_rows(self, x, gamma, eps, rows, hidden, out, stream):
        self.rows.append(("norm", x, rows, out))
        return 0

    def mk_gemm_bf16(self, w, n, k, x, rows, pad, residual, out, out_f32, ws, nbytes, err, stream):
        self.rows.append(("gemm", out_f32, rows, pad))
        return 0


def _decoder(monkeypatch, max_batch=2, max_seq_len=512, num_pages=None, forward=True):
    dec = object.__new__(SpeculativeDecoder)
    dec.cfg, dec.dev, dec.lib = TINY, torch.device("cpu"), Recorder()
    dec.max_batch, dec.max_seq_len, dec.max_nodes, dec.top = max_batch, max_seq_len, 64, 4
    dec.kv = QuantizedPagedKVCache(TINY, max_batch, max_seq_len, 8, num_pages, device="cpu")
    dec._pending = [None] * max_batch
    dec.err = torch.zeros(1, dtype=torch.int32)
    dec._h = torch.zeros(dec.MAX_ROWS, TINY.hidden, dtype=torch.bfloat16)
    embed = torch.zeros(TINY.vocab, TINY.hidden, dtype=torch.bfloat16)
    dec.m = types.SimpleNamespace(packed=types.SimpleNamespace(embed=embed, norm_final=torch.zeros(TINY.hidden)))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda dev=None: types.SimpleNamespace(cuda_stream=0))
    dec.passes = []
    if forward:  # a pass that reserves what it is to write, as the real one does
        def play(trees):
            dec.passes.append([list(t.tokens) for t in trees])
            for b, t in enumerate(trees):
                assert dec.kv.seq_lens[b] + len(t) <= dec.max_seq_len
                dec.kv.reserve(b, dec.kv.seq_lens[b] + len(t))
            return torch.zeros(sum(map(len, trees)), TINY.hidden, dtype=torch.bfloat16)
        dec._forward = play
    return dec


@pytest.mark.parametrize("batch", [1, 127, 128, 129, 300])
def test_logits_of_more_prompts_than_a_gemm_takes(monkeypatch, batch):
    """No call writes more rows than its buffer has, and every prompt's row is computed once."""
    dec = _decoder(monkeypatch, max_batch=batch)
    logits = dec.prefill([[1]] * batch)
    assert logits.shape == (batch, TINY.vocab) and dec.kv.seq_lens == [1] * batch
    norms = [r for r in dec.lib.rows if r[0] == "norm"]
    gemms = [r for r in dec.lib.rows if r[0] == "gemm"]
    assert sum(r[2] for r in norms) == sum(r[2] for r in gemms) == batch
    at = 0
    for n, g in zip(norms, gemms):
        assert 1 <= n[2] == g[2] <= g[3] <= dec.MAX_ROWS == dec._h.shape[0]
        assert n[3] == dec._h.data_ptr()
        assert n[1] == norms[0][1] + at * TINY.hidden * 2 and g[1] == logits.data_ptr() + at * TINY.vocab * 4
        at += n[2]


def test_every_scale_byte_is_its_power_of_two():
    from llama1b_megakernel_b200.kv_cache import decode_rows

    codes = torch.full((256, 64), 1.5).to(torch.float8_e4m3fn)
    got = decode_rows(codes, torch.arange(256, dtype=torch.uint8)).double()
    assert torch.equal(got[:255, 0], 1.5 * torch.exp2(torch.arange(255, dtype=torch.float64) - 127))
    assert got[255].isnan().all()


# ------------------------------------------------------------------ refusals leave things as they were
def _state(dec):
    kv = dec.kv
    return list(kv.seq_lens), [kv.pages_of(b) for b in range(kv.max_batch)], sorted(kv._free), kv.block_tables.clone()


def _same(a, b):
    return a[:3] == b[:3] and torch.equal(a[3], b[3])


@pytest.mark.parametrize("prompts,error", [
    ([[1] * 300, [2] * 513], ValueError),               # the second is too long, after three passes of the first
    ([[1] * 300 + [TINY.vocab]], ValueError),           # a bad token in the third pass
    ([[1] * 10, [2] * 140 + [-1]], ValueError),
    ([[1] * 200, [2] * 200], RuntimeError),             # more pages than there are
])
def test_refused_prefill_changes_nothing(monkeypatch, prompts, error):
    dec = _decoder(monkeypatch, num_pages=64 if error is ValueError else 40)
    dec.prefill([[3] * 5, [4]])  # something committed before
    was, passes = _state(dec), len(dec.passes)
    with pytest.raises(error):
        dec.prefill(prompts)
    assert _same(was, _state(dec)) and len(dec.passes) == passes
    dec.prefill([[1, 2, 3]])
    assert dec.kv.seq_lens == [8, 1]


def test_prefill_in_passes(monkeypatch):
    """What is right still goes through: every token once, in order."""
    dec = _decoder(monkeypatch)
    a, b = list(range(1, 301)), list(range(400, 500))
    dec.prefill([a, b])
    assert dec.kv.seq_lens == [300, 100]
    assert [t for p in dec.passes for t in p[0]] == a and [t for p in dec.passes for t in p[1]] == b
    assert all(sum(map(len, p)) <= 128 for p in dec.passes)


@pytest.mark.parametrize("bad,error", [(DraftTree.chain([2] * 60), ValueError), (DraftTree.chain([2, TINY.vocab]), ValueError),
                                       (DraftTree.chain([2] * 30), RuntimeError)])
def test_refused_score_changes_nothing(monkeypatch, bad, error):
    dec = _decoder(monkeypatch, max_seq_len=64, num_pages=4 if error is RuntimeError else None)
    dec.prefill([[3] * 5, [4] * 8])
    was, passes = _state(dec), len(dec.passes)
    with pytest.raises(error):
        dec.score([DraftTree.chain([1] * 9), bad])
    assert _same(was, _state(dec)) and len(dec.passes) == passes and not any(dec._pending)


@pytest.mark.parametrize("prompt,new,pages,error", [([1] * 500, 14, None, ValueError), ([1] * 20, 46, 8, RuntimeError)])
def test_generate_that_does_not_fit_is_refused_first(monkeypatch, prompt, new, pages, error):
    """Not after most of its tokens, which would be lost."""
    dec = _decoder(monkeypatch, num_pages=pages)
    was = _state(dec)
    with pytest.raises(error):
        dec.generate(prompt, new)
    assert _same(was, _state(dec)) and not dec.passes


def test_generate_cuts_drafts_to_the_pool(monkeypatch):
    """Tokens that fit come out although the drafts on the way would not have."""
    from llama1b_megakernel_b200 import speculative as sp

    dec = _decoder(monkeypatch, num_pages=4)
    monkeypatch.setattr(dec, "check", lambda: None, raising=False)

    def zeros(logits, targets, top, error):
        n = logits.shape[0]
        return torch.zeros(targets.shape), torch.zeros(n), torch.zeros(n, top, dtype=torch.int32), torch.zeros(n, top)
    monkeypatch.setattr(sp, "token_logprobs", zeros)
    dec._logits = lambda x: torch.zeros(x.shape[0], TINY.vocab)
    tokens, passes = dec.generate([5] * 20, 13, lambda tokens: DraftTree.chain([0, 7, 7, 7, 7, 7]))
    assert tokens == [0] * 13 and dec.kv.seq_lens[0] <= 32
    assert max(len(p[0]) for p in dec.passes[1:]) == 7  # whole drafts while there is room
