"""The speculative-decoding operators where their arithmetic is easiest to break: rows of an
8-bit cache whose scales lie far apart, logits at their type's lowest value, cache formats
that other code may write, places that are refused.

Tolerances follow from the roundings, beside those of tests/test_gpu_speculative.py:
* scores here are sums of one product that is exact, so what is left of a score's error is its
  rounding in powers of two, 2^-23 |x| for |x| <= 64, and that of exp2: e = 2^-16 in all;
* P in 8 significant bits (bf16) or more has u = 2^-8 of every p_j |v_j|, the output u once
  more; where P is f16, what its smallest numbers lose is kept below 2^-16 of
  sum_j p_j max_d |v_jd|:
    |err_d| <= (u + e) sum_j p_j |v_jd| + 2^-16 sum_j p_j max_d |v_jd| + u |o_d|.
"""
from __future__ import annotations

import math

import pytest
import torch

from llama1b_megakernel_b200 import speculative as sp
from tests import test_gpu_speculative as base

pytestmark = pytest.mark.gpu
DEV, U = base.DEV, base.U


def _put(s, x, b, pos, rows):
    """Rows `rows` [n, nkv, 64] (fp64) at places `pos` of sequence b in the pool x ("k" or "v")."""
    page, off = s["tables"][b].long()[pos // s["ps"]], pos % s["ps"]
    if s[x + "s"] is None:
        s[x][page, :, off] = rows.bfloat16()
        s[x + "64"][page, :, off] = rows.bfloat16().double()
        return
    y, byte, _ = base._quantise(rows)
    s[x].view(torch.uint8)[page, :, off] = y.float().to(torch.float8_e4m3fn).view(torch.uint8)
    s[x + "s"][page, :, off] = byte
    s[x + "64"][page, :, off] = y * base._pow2(byte.to(torch.int64) - 127)[..., None]


def _compare(s, out, lse, skip=()):
    """Against the definition in 64 bits, the scores taken as exact."""
    nq, nkv, ps = s["q"].shape[1], s["k"].shape[1], s["ps"]
    group, at = nq // nkv, 0
    for b, (p, n) in enumerate(zip(s["prefixes"], s["nodes"])):
        j = torch.arange(p + n, device=DEV)
        pg = s["right_tables"][b].long()[j // ps]
        kk, vv = (s[x][pg, :, j % ps].transpose(0, 1).repeat_interleave(group, 0) for x in ("k64", "v64"))
        q = s["q"][at:at + n].double().transpose(0, 1)
        seen = torch.cat([torch.ones(n, p, dtype=torch.bool), s["masks"][b]], 1).to(DEV)
        vv = torch.where(seen.any(0)[None, :, None], vv, 0.0)
        x = torch.where(seen, (q @ kk.transpose(1, 2)) * 0.125, -math.inf)
        w = torch.softmax(x, -1)
        want = torch.logsumexp(x, -1)
        for i in range(n):
            if (b, i) in skip:
                continue
            vi = torch.where(seen[i][None, :, None], vv, 0.0)
            wi = w[:, i:i + 1]
            ref, size, most = (wi @ vi)[:, 0], (wi @ vi.abs())[:, 0], wi @ vi.abs().amax(-1, keepdim=True)
            tol = (U + 2.0 ** -16) * size + 2.0 ** -16 * most[:, 0] + U * ref.abs()
            off = (out[at + i].double() - ref).abs()
            assert (off <= tol).all(), (b, i, float((off / tol).max()))
            assert ((lse[at + i].double() - want[:, i]).abs() <= 2.0 ** -16 + 2.0 ** -22 * want[:, i].abs()).all(), (b, i)
        at += n


def _scored(prefix, nodes, score, fmt="e4m3", nq=8, nkv=1, ps=64, seed=0):
    """One sequence whose scores are score[j] (multiples that an 8-bit row holds exactly), of
    every node alike: q is 8 in dim 0, and a key's dim 0 its score."""
    s = base._setup([prefix], [nodes], nq, nkv, ps, fmt, "chain", seed=seed)
    s["q"].zero_()
    s["q"][..., 0] = 8
    n = prefix + nodes
    k = torch.randn(n, nkv, 64, generator=base._gen(seed + 1), device=DEV).double()
    k[..., 0] = score[:n, None]
    _put(s, "k", 0, torch.arange(n, device=DEV), k)
    return s


def _many(s, batch=600):
    """The one sequence of s as many that share its pages, so that none is cut into ranges; the
    comparison is of the first, and every one has to give its bits."""
    nodes = s["nodes"][0]
    return dict(s, tables=s["tables"].repeat(batch, 1), q=s["q"].repeat(batch, 1, 1), mask=s["mask"].repeat(batch, 1),
                prefix=s["prefix"].repeat(batch), cu=torch.arange(batch + 1, dtype=torch.int32, device=DEV) * nodes)


def _attend_many(s):
    nodes = s["nodes"][0]
    out, lse, err = base._attend(_many(s))
    assert int(err) == 0
    for x in (out, lse):
        assert torch.equal(x.view(-1, nodes, *x.shape[1:]), x[:nodes].expand(x.shape[0] // nodes, *x[:nodes].shape))
    return out[:nodes], lse[:nodes]


# ------------------------------------------------------------------ scales far apart
@pytest.mark.parametrize("nodes", [1, 2, 20])
@pytest.mark.parametrize("spread", [0, 2, 4, 7, 10, 14, 24])
@pytest.mark.parametrize("peak,sink", [(10, False), (10, True), (14, True), (20, False), (20, True)])
def test_flat_tail_beside_a_peak(nodes, spread, peak, sink):
    """Thousands of keys of one small probability behind some with e^peak times theirs (with
    `sink`, of no value), where rows of 2^spread times the size came by that nobody looks at:
    the small probabilities together are the result, or a part of it that shows."""
    n = 4096 + nodes
    j = torch.arange(n, device=DEV)
    score = torch.zeros(n, dtype=torch.float64, device=DEV)
    outlier = j % 64 == 5
    score[outlier] = -208.0
    score[10:400:64] = peak  # one for each warp, wherever a block of positions goes
    s = _scored(4096, nodes, score, seed=peak + spread)
    v = torch.randn(n, 1, 64, generator=base._gen(7), device=DEV).double()
    v[outlier] *= 2.0 ** spread
    if sink:
        v[10:400:64] = 0
    _put(s, "v", 0, j, v)
    _compare(s, *_attend_many(s))


@pytest.mark.parametrize("nodes", [1, 2, 20])
@pytest.mark.parametrize("prefix", [100, 3000])
@pytest.mark.parametrize("late", [True, False])
def test_small_probabilities_of_large_values(nodes, prefix, late):
    """Half of the rows are 2^20 times as large and e^-14 times as probable: both halves count
    alike, whichever comes first."""
    n = prefix + nodes
    j = torch.arange(n, device=DEV)
    large = (j >= prefix // 2) == late
    s = _scored(prefix, nodes, torch.where(large, -14.0, 0.0).double(), seed=prefix)
    v = torch.randn(n, 1, 64, generator=base._gen(prefix), device=DEV).double()
    _put(s, "v", 0, j, torch.where(large[:, None, None], v * 2.0 ** 20, v))
    _compare(s, *_attend_many(s))


@pytest.mark.parametrize("nodes,nq,nkv", [(1, 8, 1), (4, 8, 2), (30, 8, 2)])
@pytest.mark.parametrize("lowest", [-4, -14, -40])
@pytest.mark.parametrize("size", [0, 20])
def test_rows_of_every_size(nodes, nq, nkv, lowest, size):
    """K and V rows of sizes spread over powers of two, and all of them large (scale bytes that
    take two factors to become bf16), with queries as much smaller."""
    s = base._setup([700, 0, 65], [nodes] * 3, nq, nkv, 16, "e4m3", "tree", seed=nodes - lowest)
    g = base._gen(size)
    for b, p in enumerate(s["prefixes"]):
        n = p + nodes
        j = torch.arange(n, device=DEV)
        for x, low in (("k", max(lowest, -6)), ("v", lowest)):
            e = torch.rand(n, nkv, 1, generator=g, device=DEV) * low + size
            _put(s, x, b, j, torch.randn(n, nkv, 64, generator=g, device=DEV).double() * torch.exp2(e.double()))
    s["q"] *= 2.0 ** -size
    out, lse, err = base._attend(s)
    assert int(err) == 0
    base._check(s, out, lse)


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("nodes", [2, 4, 30])
@pytest.mark.parametrize("prefix", [0, 40, 700])
@pytest.mark.parametrize("small", [0, 20, 60])
def test_huge_values_in_masked_places(fmt, nodes, prefix, small):
    """A node of 3e38 that only itself sees does not take a bit from the other rows, of size
    1 or 2^-small."""
    s = base._setup([prefix, 64], [nodes] * 2, 8, 2, 16, fmt, "tree", seed=prefix + nodes, qscale=6.0)
    j = torch.arange(prefix + nodes, device=DEV)
    v = torch.randn(prefix + nodes, 2, 64, generator=base._gen(small), device=DEV).double()
    _put(s, "v", 0, j, v * 2.0 ** -small)
    leaf = nodes - 1
    s["masks"][0][leaf, :leaf] = False  # a root of its own
    s["mask"] = base._words(s["masks"], s["T"])
    huge = torch.full((1, 2, 64), 3.0e38, dtype=torch.float64, device=DEV)
    huge[..., ::2] *= -1
    at = torch.tensor([prefix + leaf], device=DEV)
    _put(s, "k", 0, at, huge)
    _put(s, "v", 0, at, huge)
    out, lse, err = base._attend(s)
    assert int(err) == 0
    finite = dict(s, k64=torch.where(s["k64"].abs() > 1e38, 0.0, s["k64"]))  # the tolerance is of what rows see
    base._check(finite, out, lse, skip={(0, leaf)})


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("nodes", [1, 2, 20])
def test_huge_values_of_no_probability(fmt, nodes):
    """Committed rows of 3e38 with a probability of e^-208 of the others' add nothing (6e-53)."""
    prefix = 700
    n = prefix + nodes
    j = torch.arange(n, device=DEV)
    huge = (j % 32 == 6) & (j < 200)
    s = _scored(prefix, nodes, torch.where(huge, -208.0, 0.0).double(), fmt=fmt, seed=nodes)
    v = torch.randn(n, 1, 64, generator=base._gen(nodes), device=DEV).double()
    v[huge] = torch.where(v[huge] < 0, -3.0e38, 3.0e38).double()
    _put(s, "v", 0, j, v)
    out, lse, err = base._attend(s)
    assert int(err) == 0
    _compare(s, out, lse)


# ------------------------------------------------------------------ exponentials
@pytest.mark.parametrize("shift", [0, 1])
def test_exponentials_of_either_pipe(shift):
    """Of 32 committed positions the large tiles take columns 6, 7, 16, 17, 26 and 27 with a
    polynomial. Where only those (or only others) count, lse is a sum of such exponentials: right to
    the polynomial's 2^-22, the score's rounding (2^-24 of up to 2^4.5), the sum's and the
    logarithm's, 2^-18 in all."""
    prefix, nodes = 2048, 20
    n = prefix + nodes
    j = torch.arange(n, device=DEV)
    counts = (((j % 32)[:, None] - shift * 3 == torch.tensor([6, 7, 16, 17, 26, 27], device=DEV)).any(1)) & (j < prefix)
    x = torch.randint(-4096, 1, (n,), generator=base._gen(5), device=DEV).double() / 256  # -16 .. 0
    x = x.bfloat16().double()
    score = torch.where(counts, x, -60.0)
    s = _scored(prefix, nodes, score, fmt="bf16")
    out, lse = _attend_many(s)
    _compare(s, out, lse)
    seen = score.clone()
    want = torch.logsumexp(seen, 0)
    assert ((lse.double() - want).abs() <= 2.0 ** -18).all()


# ------------------------------------------------------------------ scale bytes that other code may write
@pytest.mark.parametrize("nodes", [1, 2, 20])
@pytest.mark.parametrize("x,byte", [("k", 0), ("v", 0), ("v", 1), ("v", 254)])
def test_extreme_scale_bytes(nodes, x, byte):
    """Byte 0 stands for 2^-127 and 254 for 2^127, as every other byte for its power."""
    prefix = 40
    s = base._setup([prefix], [nodes], 8, 1, 8, "e4m3", "chain", seed=byte)
    g, n = base._gen(byte + 1), prefix + nodes
    lo, hi = (64, 448) if byte < 254 else (2.0 ** -9, 2.0 ** -6)
    mag = torch.rand(n, 1, 64, generator=g, device=DEV) * (hi - lo) + lo
    code = (mag * torch.where(torch.rand(n, 1, 64, generator=g, device=DEV) < 0.5, -1.0, 1.0)).to(torch.float8_e4m3fn)
    j = torch.arange(n, device=DEV)
    page, off = s["tables"][0].long()[j // 8], j % 8
    s[x].view(torch.uint8)[page, :, off] = code.view(torch.uint8)
    s[x + "s"][page, :, off] = byte
    s[x + "64"][page, :, off] = code.double() * 2.0 ** (byte - 127)
    if x == "k":
        s["q"] *= 2.0 ** 118
    else:
        s["q"].zero_()
    out, lse, err = base._attend(s)
    assert int(err) == 0
    if x == "k":
        base._check(s, out, lse)
    else:
        _compare(s, out, lse)


def test_rows_of_scale_byte_0_read_back():
    from llama1b_megakernel_b200.kv_cache import decode_rows

    codes = torch.linspace(-448, 448, 64, device=DEV).to(torch.float8_e4m3fn).view(1, 1, 1, 64).expand(1, 1, 8, 64).contiguous()
    scales = torch.tensor([0, 1, 17, 127, 128, 200, 246, 255], dtype=torch.uint8, device=DEV).view(1, 1, 8)
    layer = sp.KVLayer(codes, codes, torch.zeros(1, 1, dtype=torch.int32, device=DEV), scales, scales)
    k, _ = sp.kv_read(layer, torch.tensor([8], dtype=torch.int32, device=DEV), 8)
    want = (codes.double() * torch.exp2(scales.double() - 127)[..., None]).bfloat16()[0]
    host = decode_rows(codes.cpu(), scales.cpu())[0]
    assert torch.equal(k[0, :, :7], want[:, :7]) and torch.equal(host[:, :7], want[:, :7].cpu())
    assert k[0, :, 7].isnan().all() and host[:, 7].isnan().all()


# ------------------------------------------------------------------ refusals
@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("nq,nkv", [(1, 1), (4, 2), (8, 8)])
@pytest.mark.parametrize("pos", [-1, 4, 1 << 30])
def test_row_of_a_bad_position_is_not_stored(fmt, nq, nkv, pos):
    """Neither K nor V: the place keeps the row that it has."""
    k, v, ks, vs, _, _ = base._pool(2, nkv, 8, fmt, base._gen(3))
    pools = [t if t.dtype == torch.uint8 else t.view(torch.uint8) for t in (k, v, ks, vs) if t is not None]
    was = [t.clone() for t in pools]
    layer = sp.KVLayer(k, v, torch.tensor([[1, 0]], dtype=torch.int32, device=DEV), ks, vs)
    cos = torch.ones(4, 64, device=DEV).bfloat16()
    qkv = torch.randn(2, (nq + 2 * nkv) * 64, generator=base._gen(4), device=DEV).bfloat16()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    q, err = torch.zeros(2, nq, 64, dtype=torch.bfloat16, device=DEV), base._err()
    sp.kv_write(layer, qkv, cos, cos, i32(0, 0), i32(3, 9), i32(pos, 2), q, error=err)
    assert int(err) == 1
    for t, w in zip(pools, was):
        assert torch.equal(t[1], w[1])      # the bad row's page
        assert not torch.equal(t[0], w[0]) or t.dim() == 3  # the other row is there (a scale may stay the same)
    err = base._err()
    sp.kv_write(layer, qkv, cos, cos, i32(0, 0), i32(3, 9), i32(1, 2), q, error=err)
    assert int(err) == 0


# ------------------------------------------------------------------ caches and calls that are right
def test_cache_whose_scales_start_on_8_bytes():
    """One K/V head, pages of 8 and an odd number of them: the second layer's scales lie on 8 bytes, not 16."""
    g = base._gen(2)
    pages, ps, nq, n, T = 5, 8, 4, 21, 3
    k, v = (torch.randn(2, pages, 1, ps, 64, generator=g, device=DEV).to(torch.float8_e4m3fn) for _ in range(2))
    ks, vs = (torch.randint(120, 130, (2, pages, 1, ps), generator=g, device=DEV).to(torch.uint8) for _ in range(2))
    table = torch.tensor([[3, 0, 4, 1]], dtype=torch.int32, device=DEV)
    qkv = torch.randn(T, (nq + 2) * 64, generator=g, device=DEV).bfloat16()
    ang = torch.rand(64, 32, generator=g, device=DEV)
    cos, sin = (torch.cat([f(ang), f(ang)], 1).bfloat16() for f in (torch.cos, torch.sin))
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    got = []
    assert ks[1].data_ptr() % 16 == 8
    for x in ((k[1], v[1], ks[1], vs[1]), tuple(t[1].clone() for t in (k, v, ks, vs))):
        layer, err = sp.KVLayer(*x[:2], table, *x[2:]), base._err()
        q = torch.empty(T, nq, 64, dtype=torch.bfloat16, device=DEV)
        sp.kv_write(layer, qkv, cos, sin, i32(0, 0, 0), i32(n, n + 1, n + 2), i32(n, n + 1, n + 2), q, error=err)
        mask = i32(1, 3, 7).long()[:, None].contiguous()
        o, lse = sp.tree_attention(q, layer, i32(0, T), mask, i32(n), T, n + T, error=err)
        got.append((q, o, lse, *sp.kv_read(layer, i32(n + T), n + T, error=err)))
        assert int(err) == 0
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_calls_without_rows():
    """No rows, no positions, no tokens: empty results, not a refusal."""
    s = base._setup([20, 3], [2, 1], 8, 2, 16, "e4m3", "chain", seed=1)
    layer, err = sp.KVLayer(s["k"], s["v"], s["tables"], s["ks"], s["vs"]), base._err()
    i0 = torch.zeros(0, dtype=torch.int32, device=DEV)
    one = torch.ones(4, 64, device=DEV).bfloat16()
    q = torch.empty(0, 8, 64, dtype=torch.bfloat16, device=DEV)
    sp.kv_write(layer, torch.empty(0, 12 * 64, dtype=torch.bfloat16, device=DEV), one, one, i0, i0, i0, q, error=err)
    k, v = sp.kv_read(layer, s["prefix"], 0, error=err)
    assert k.shape == v.shape == (2, 2, 0, 64)
    cu = torch.zeros(3, dtype=torch.int32, device=DEV)
    out, lse = sp.tree_attention(q, layer, cu, torch.empty(0, 1, dtype=torch.int64, device=DEV), s["prefix"], 2, 22, error=err)
    assert out.shape == (0, 8, 64) and lse.shape == (0, 8)
    for n, top in ((0, 0), (2, 3)):
        t = torch.empty(0, n, dtype=torch.int32, device=DEV)
        lp, ent, ids, tlp = sp.token_logprobs(torch.empty(0, 50, device=DEV), t, top, error=err)
        assert lp.shape == (0, n) and ent.shape == (0,) and ids.shape == tlp.shape == (0, top)
    assert int(err) == 0


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


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(1, 128256), (300, 4099)])
@pytest.mark.parametrize("level", ["lowest", 0.0, 96.0, -30000.0])
def test_logprobs_of_equal_logits_at_any_level(dtype, rows, vocab, level):
    """log p_t = (x_t - m) - log s: what the logits are has no part in it, so of equal ones it is
    -log V to a few units of log's last place (|log V| < 16, an ulp is 2^-20 of 1)."""
    level = torch.finfo(dtype).min if level == "lowest" else level
    x = torch.full((rows, vocab), level, dtype=dtype, device=DEV)
    t = torch.full((rows, 1), vocab // 2, dtype=torch.int32, device=DEV)
    lp, ent, ids, tlp = sp.token_logprobs(x, t, 3)
    want = math.log(vocab)
    for got, ref in ((lp, -want), (tlp, -want), (ent, want)):
        assert ((got.double() - ref).abs() <= 2.0 ** -19).all()
    assert (ids == torch.arange(3, device=DEV)).all()


def test_arguments_of_other_shapes():
    """Vectors where matrices belong and the other way round are a ValueError, as other shapes are."""
    s = base._setup([20], [3], 8, 2, 16, "e4m3", "chain", seed=1)
    layer = sp.KVLayer(s["k"], s["v"], s["tables"], s["ks"], s["vs"])
    i32 = lambda *shape: torch.zeros(*shape, dtype=torch.int32, device=DEV)  # noqa: E731
    x = torch.zeros(2, 50, device=DEV)
    for bad in (lambda: sp.token_logprobs(x, i32(2)), lambda: sp.token_logprobs(x, i32(2, 1, 1)),
                lambda: sp.kv_read(layer, torch.tensor(3, dtype=torch.int32, device=DEV), 4),
                lambda: sp.kv_read(layer, i32(1, 1), 4),
                lambda: sp.tree_attention(s["q"], layer, s["cu"], s["mask"], s["prefix"][0], 3, 23),
                lambda: sp.tree_attention(s["q"], layer, s["cu"], s["mask"], s["prefix"][:, None], 3, 23),
                lambda: sp.tree_attention(s["q"][0], layer, s["cu"], s["mask"], s["prefix"], 3, 23)):
        with pytest.raises(ValueError):
            bad()
