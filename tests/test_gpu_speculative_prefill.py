"""SpeculativeDecoder.prefill beyond one pass of the GEMM: more prompts than it has rows.

The bar is that of the small configurations: cosine >= 0.999, max-abs <= 3e-2."""
from __future__ import annotations

import pytest
import torch

from llama1b_megakernel_b200 import synthetic as syn
from llama1b_megakernel_b200.config import SMALL
from llama1b_megakernel_b200.model import MegakernelLlamaForCausalLM
from llama1b_megakernel_b200.speculative import SpeculativeDecoder

pytestmark = pytest.mark.gpu


def test_prefill_of_more_prompts_than_rows():
    m = MegakernelLlamaForCausalLM(SMALL, syn.make_weights(SMALL, seed=23), max_batch=1, max_seq_len=64, page_size=16)
    batch = 300
    prompts = [syn.random_tokens(1 + b % 3, SMALL.vocab, seed=b).tolist() for b in range(batch)]
    dec = SpeculativeDecoder(m, batch, 16, page_size=16, cache="bf16")
    logits = dec.prefill(prompts)
    dec.check()
    assert dec.kv.seq_lens == [len(p) for p in prompts] and logits.isfinite().all()
    for b in (0, 1, 2, 126, 127, 128, 129, 255, 256, 299):
        one = SpeculativeDecoder(m, 1, 16, page_size=16, cache="bf16")
        want = one.prefill([prompts[b]])[0].double()
        one.check()
        got = logits[b].double()
        cos = float(got @ want / (got.norm() * want.norm()))
        assert cos >= 0.999 and float((got - want).abs().max()) <= 3e-2, (b, cos)
