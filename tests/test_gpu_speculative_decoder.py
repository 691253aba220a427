"""SpeculativeDecoder on the GPU: trees of drafted tokens through a small model.

Over a bf16 cache every node's logits are compared with the oracle's decode steps
along its path (HF semantics, CPU), at the bar of the small configurations:
cosine >= 0.999, max-abs <= 3e-2. Over an 8-bit cache a tree is compared with the
same tokens scored one at a time: the passes round at other places (bf16 sums, and
a code that falls to its neighbour), each within that bar of exact arithmetic on
its cache, so twice the bar: cosine >= 0.998, max-abs <= 6e-2.
"""
from __future__ import annotations

import pytest
import torch

from llama1b_megakernel_b200 import synthetic as syn
from llama1b_megakernel_b200.config import SMALL
from llama1b_megakernel_b200.model import MegakernelLlamaForCausalLM
from llama1b_megakernel_b200.speculative import DraftTree, SpeculativeDecoder, lookup_draft
from oracle import llama_oracle as O

pytestmark = pytest.mark.gpu


def _cos(a, b):
    a, b = a.double().flatten().cpu(), b.double().flatten().cpu()
    return float(a @ b / (a.norm() * b.norm()))


@pytest.fixture(scope="module")
def setup():
    w = syn.make_weights(SMALL, seed=23)
    return w, MegakernelLlamaForCausalLM(SMALL, w, max_batch=1, max_seq_len=512, page_size=16)


def _decoder(m, cache, lengths, seed=5, **kw):
    dec = SpeculativeDecoder(m, max_batch=max(1, len(lengths)), max_seq_len=512, page_size=16, cache=cache, **kw)
    dec.kv.shuffle_free_pages(seed)
    rows = []
    for b, n in enumerate(lengths):
        k, v = syn.random_kv_rows(SMALL, max(n, 1), seed=seed, seq=b)
        rows.append((k, v))
        if n:
            dec.kv.fill(b, k, v)
    return dec, rows


def _paths(tree):
    out = []
    for i in range(len(tree)):
        path, j = [], i
        while j >= 0:
            path.append(j)
            j = tree.parents[j]
        out.append(path[::-1])
    return out


TREES = [
    DraftTree([11, 70, 901, 33, 4002, 5, 17], [-1, 0, 0, 1, 1, 2, 5]),
    DraftTree([3], [-1]),
    DraftTree([8, 9, 10, 700, 12, 999], [-1, -1, 0, 1, 2, 3]),
]


def test_tree_logits_match_the_oracle(setup):
    w, m = setup
    lengths = [100, 0, 37]
    dec, rows = _decoder(m, "bf16", lengths)
    scores = dec.score(TREES)
    dec.check()
    for b, tree in enumerate(TREES):
        for i, path in enumerate(_paths(tree)):
            kv = O.OracleKV(torch.zeros_like(dec.kv.k_pages, device="cpu"), torch.zeros_like(dec.kv.v_pages, device="cpu"),
                            dec.kv.block_tables[b:b + 1].cpu().clone())
            if lengths[b]:
                kv.fill(0, *rows[b])
            for step, j in enumerate(path):
                ref = O.decode_step(SMALL, w, kv, torch.tensor([tree.tokens[j]]), [lengths[b] + step])
            got, want = scores.logits[scores.first[b] + i].cpu(), ref["logits"][0].float()
            err = float((got - want).abs().max())
            assert _cos(got, want) >= 0.999 and err <= 3e-2, (b, i, err)
            lp = torch.log_softmax(got.double(), 0)
            kids = tree.children()[i]
            for c, j in enumerate(kids):
                assert abs(float(scores.child_logprobs[scores.first[b] + i, c]) - float(lp[tree.tokens[j]])) <= 1e-4
            assert int(scores.top_ids[scores.first[b] + i, 0]) == int(got.argmax())


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
def test_tree_agrees_with_one_token_at_a_time(setup, cache):
    _, m = setup
    lengths = [100, 0, 37]
    dec, _ = _decoder(m, cache, lengths)
    scores = dec.score(TREES)
    for b, tree in enumerate(TREES):
        for i, path in enumerate(_paths(tree)):
            one, _ = _decoder(m, cache, lengths)
            for j in path:
                trees = [DraftTree([tree.tokens[j]], [-1]) if x == b else DraftTree([1], [-1]) for x in range(3)]
                s = one.score(trees)
                for x in range(3):
                    one.commit(x, [0] if x == b else [])
            one.check()
            got, want = scores.logits[scores.first[b] + i], s.logits[b]
            err = float((got - want).abs().max())
            assert _cos(got, want) >= 0.998 and err <= 6e-2, (b, i, err)
    dec.check()


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
def test_commit_keeps_exactly_the_path(setup, cache):
    _, m = setup
    dec, _ = _decoder(m, cache, [30, 14])
    tree = TREES[0]
    dec.score([tree, TREES[1]])
    before = [t.clone() for t in dec.kv.gather(0, 30 + len(tree))]
    other = [t.clone() for t in dec.kv.gather(1, 15)]
    path = [0, 2, 5, 6]
    dec.commit(0, path)
    dec.commit(1, [])
    assert dec.kv.seq_lens[:2] == [34, 14]
    after = dec.kv.gather(0, 34)
    for was, now in zip(before, after):
        assert torch.equal(now[:, :, :30], was[:, :, :30])
        assert torch.equal(now[:, :, 30:], was[:, :, [30 + j for j in path]])
    assert all(torch.equal(a, b) for a, b in zip(other, dec.kv.gather(1, 15)))
    with pytest.raises(ValueError):
        dec.commit(0, [0])  # nothing is pending any more
    dec.score([tree, TREES[1]])
    for bad in ([1], [0, 3], [0, 0], [0, 7]):
        with pytest.raises(ValueError):
            dec.commit(0, bad)
    dec.check()


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
def test_generate_with_and_without_drafts(setup, cache):
    """The drafted run takes the undrafted run's tokens up to a near tie, in fewer passes."""
    _, m = setup
    prompt = syn.random_tokens(150, SMALL.vocab, seed=9).tolist()  # two prefill passes
    dec, _ = _decoder(m, cache, [])
    plain, passes = dec.generate(prompt, 24)
    assert len(plain) == 24 and passes == 24
    dec.release(0)

    def draft(tokens):  # the right continuation beside a wrong one
        at = len(tokens) - len(prompt)
        right = plain[at:at + 5] if tokens[len(prompt):] == plain[:at] else []
        if not right:
            return None
        return DraftTree([(right[0] + 1) % SMALL.vocab, *right], [-1, *range(-1, 0), *range(1, len(right))])

    drafted, fewer = dec.generate(prompt, 24, draft)
    if drafted == plain:
        assert fewer <= 8
        return
    first = next(i for i, (a, b) in enumerate(zip(plain, drafted)) if a != b)
    dec.release(0)
    logits = dec.prefill([prompt + plain[:first]])[0]
    assert float(logits[plain[first]] - logits[drafted[first]]) <= 6e-2, first


def test_lookup_draft_and_refusals(setup):
    _, m = setup
    dec, _ = _decoder(m, "e4m3", [])
    tokens, passes = dec.generate([5, 6, 7, 8] * 6, 12, lookup_draft)
    assert len(tokens) == 12 and passes <= 12
    for bad in ([], [TREES[0], TREES[1]], [DraftTree([], [])], [DraftTree.chain(range(70))], [DraftTree([SMALL.vocab], [-1])]):
        with pytest.raises(ValueError):
            dec.score(bad)
    with pytest.raises(ValueError):
        dec.prefill([[]])
    with pytest.raises(ValueError):
        SpeculativeDecoder(m, 1, 512, cache="fp4")
    with pytest.raises(ValueError):
        SpeculativeDecoder(m, 1, 1 << 20)


def test_other_paths_refuse_the_8_bit_cache(setup):
    _, m = setup
    dec, _ = _decoder(m, "e4m3", [])
    with pytest.raises(ValueError):
        m.prefill(torch.tensor([[1, 2]]), past_key_values=dec.kv)
    dec = SpeculativeDecoder(m, 1, 512, page_size=16)
    with pytest.raises(ValueError):
        m.forward(torch.tensor([[1]]), torch.tensor([[0]]), past_key_values=dec.kv)
