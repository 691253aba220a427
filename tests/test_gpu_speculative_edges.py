"""The speculative-decoding operators where their arithmetic is easiest to break."""
from __future__ import annotations

import math

import pytest
import torch

from llama1b_megakernel_b200 import speculative as sp
from tests import test_gpu_speculative as base

pytestmark = pytest.mark.gpu
DEV, U = base.DEV, base.U


# ------------------------------------------------------------------ log probabilities
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(1, 128256), (2, 20000), (300, 4099), (700, 9000), (3, 700)])
@pytest.mark.parametrize("where", ["tail", "head", "middle", "most", "odd"])
def test_logprobs_of_tokens_at_the_lowest_value(dtype, rows, vocab, where):
    """Tokens forbidden by the type's lowest number instead of -inf have no probability, and the
    row keeps its entropy."""
    low = torch.finfo(dtype).min
    x = (torch.randn(rows, vocab, generator=base._gen(vocab), device=DEV) * 3).to(dtype)
    j = torch.arange(vocab, device=DEV)
    off = {"tail": j >= vocab // 2, "head": j < vocab // 2, "middle": (j > vocab // 4) & (j < vocab - vocab // 4),
           "most": j != vocab - 3, "odd": j % 2 == 1}[where]
    x[:, off] = low
    open_ = j[~off]
    targets = torch.stack([open_[torch.randint(len(open_), (rows,), generator=base._gen(1), device=DEV)],
                           j[off][torch.randint(int(off.sum()), (rows,), generator=base._gen(2), device=DEV)]], 1).to(torch.int32)
    top = min(4, len(open_))
    lp, ent, ids, tlp = sp.token_logprobs(x, targets, top)
    rlp, rent, rids, rtlp = base._logprobs_ref(x, targets, top)
    assert torch.equal(ids.long(), rids)
    size = float(x[:, ~off].abs().max())
    for got, ref in ((lp, rlp), (tlp, rtlp)):
        assert ((got.double() - ref).abs() <= 2.0 ** -14 + 2.0 ** -22 * (size + ref.abs())).all()
    xd = x[:, ~off].double()
    mean = ((xd - xd.amax(-1, keepdim=True)) * torch.softmax(xd, -1)).sum(-1).abs()
    assert ((ent.double() - rent).abs() <= (2.0 ** -14 + 2.0 ** -22 * size) * (1 + mean)).all()
