"""The speculative-decoding operators (csrc/mk_kv8.cuh, mk_tree.cuh, mk_logprobs.cuh)
against plain evaluations of their definitions in 64 bits.

Tolerances follow from the roundings each operator makes:
* bf16 has 8 significant bits, so a stored value is within u = 2^-8 of its size of
  the number it rounds; an e4m3 code is within half a step; rotations add one
  fp32 rounding;
* attention: scores are fp32 sums of 64 exact products (an error of at most
  64 * 2^-23 * sum|q k| * scale, called d), probabilities are rounded to bf16
  before P V (u each), the output once more:
    |err| <= (u + 4 d + 2^-18) sum_j p_j |v_j| + u |o|;
  lse, from unrounded fp32 probabilities: 2 d + 2^-18 + 2^-22 |lse|;
* log probabilities: fp32 sums of at most 1024 terms per thread, each exp within
  2^-20: 2^-14 + 2^-22 max|x|, times (1 + the mean |x - max|) for the entropy.
"""
from __future__ import annotations

import math

import pytest
import torch

from llama1b_megakernel_b200 import _lib
from llama1b_megakernel_b200 import speculative as sp

pytestmark = pytest.mark.gpu
DEV = "cuda"
NAN_BYTE = 255
U = 2.0 ** -8  # unit roundoff of bf16


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _err():
    return torch.zeros(1, dtype=torch.int32, device=DEV)


def _pow2(e):
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _quantise(x):
    """fp64 rows -> (their 8-bit values without the scale, scale bytes), from the definition."""
    amax = x.abs().amax(-1)
    e = torch.full_like(amax, -110)
    for k in range(-110, 121):
        e = torch.where(amax > 448 * 2.0 ** (k - 1), torch.full_like(e, float(k)), e) if k > -110 else e
    y = x / _pow2(e)[..., None]
    f = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
    step = _pow2(f - 3)
    return torch.round(y / step) * step, (e + 127).to(torch.uint8), step * _pow2(e)[..., None]


def _pool(pages, nkv, ps, fmt, g, scale=1.0, fill=None):
    """(k, v, ks, vs, their fp64 values)."""
    out = []
    for _ in range(2):
        x = torch.randn(pages, nkv, ps, 64, generator=g, device=DEV) * scale
        if fmt == "bf16":
            p = x.bfloat16()
            out.append((p, None, p.double()))
        else:
            y, byte, _ = _quantise(x.double())
            c = y.float().to(torch.float8_e4m3fn)
            assert torch.equal(c.double(), y)
            out.append((c, byte, y * _pow2(byte.to(torch.int64) - 127)[..., None]))
    (k, ks, k64), (v, vs, v64) = out
    return k, v, ks, vs, k64, v64


def _tables(batch, blocks, pages, g):
    return torch.randperm(pages, generator=g, device=DEV)[:batch * blocks].view(batch, blocks).to(torch.int32)


# ------------------------------------------------------------------ cache rows
@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("rows,nq,nkv,ps", [(1, 32, 8, 64), (7, 4, 1, 8), (33, 8, 8, 24), (130, 16, 2, 16)])
def test_write(fmt, rows, nq, nkv, ps):
    g = _gen(rows)
    batch, blocks = 3, 5
    pages = batch * blocks + 2
    qkv = (torch.randn(rows, (nq + 2 * nkv) * 64, generator=g, device=DEV)
           * torch.exp(torch.randn(rows, 1, generator=g, device=DEV) * 4)).bfloat16()
    qkv[0, nq * 64:(nq + 1) * 64] = 0  # a row of zeros
    ang = torch.rand(64, 32, generator=g, device=DEV) * 6
    cos, sin = (torch.cat([f(ang), f(ang)], 1).bfloat16() for f in (torch.cos, torch.sin))
    place = torch.randperm(batch * blocks * ps, generator=g, device=DEV)[:rows]
    seqs, slots = (place // (blocks * ps)).to(torch.int32), (place % (blocks * ps)).to(torch.int32)
    positions = torch.randint(64, (rows,), generator=g, device=DEV).to(torch.int32)
    if rows > 3:
        slots[3] = -1  # a padding row
    tables = _tables(batch, blocks, pages, g)
    k, v, ks, vs, _, _ = _pool(pages, nkv, ps, fmt, g)
    before = [t.clone() for t in (k, v)]
    layer = sp.KVLayer(k, v, tables, ks, vs)
    q, err = torch.zeros(rows, nq, 64, dtype=torch.bfloat16, device=DEV), _err()
    sp.kv_write(layer, qkv, cos, sin, seqs, slots, positions, q, error=err)
    assert int(err) == 0
    x = qkv.double().view(rows, nq + 2 * nkv, 32, 2).transpose(-1, -2).reshape(rows, nq + 2 * nkv, 64)
    turned = torch.cat([-x[..., 32:], x[..., :32]], -1)
    c, s = (t[positions.long()].double()[:, None] for t in (cos, sin))
    rot, size = x * c + turned * s, (x * c).abs() + (turned * s).abs()
    assert ((q.double() - rot[:, :nq]).abs() <= U * rot[:, :nq].abs() + 2.0 ** -23 * size[:, :nq]).all()
    touched = torch.zeros(pages, ps, dtype=torch.bool, device=DEV)
    for r in range(rows):
        if int(slots[r]) < 0:
            continue
        page, at = int(tables[int(seqs[r]), int(slots[r]) // ps]), int(slots[r]) % ps
        touched[page, at] = True
        for pool, scales, ref, sz in ((k, ks, rot[r, nq:nq + nkv], size[r, nq:nq + nkv]),
                                      (v, vs, x[r, nq + nkv:], 0 * x[r, nq + nkv:])):
            got = pool[page, :, at].float().double()
            if fmt == "bf16":
                assert ((got - ref).abs() <= U * ref.abs() + 2.0 ** -23 * sz).all()
                continue
            _, byte, step = _quantise(ref)
            assert torch.equal(scales[page, :, at], byte)  # no threshold is within fp32 rounding here
            got = got * _pow2(byte.to(torch.int64) - 127)[:, None]
            assert ((got - ref).abs() <= step / 2 + 2.0 ** -23 * sz).all()
    rest = ~touched[:, None, :, None].expand(k.shape)
    for pool, was in zip((k, v), before):
        assert torch.equal(pool.view(torch.uint8).view(*k.shape, -1)[rest], was.view(torch.uint8).view(*k.shape, -1)[rest])


def test_write_of_non_finite_and_extreme_rows():
    """NaN and infinity make the row NaN; the largest and smallest numbers keep theirs."""
    nq, nkv, ps = 1, 1, 8
    qkv = torch.zeros(6, 3 * 64, dtype=torch.bfloat16, device=DEV)
    vals = [float("nan"), float("inf"), -float("inf"), 3.0e38, 1e-30, 1e-40]
    for r, x in enumerate(vals):
        qkv[r, 2 * 64:] = x / 4 if math.isfinite(x) else 1.0
        qkv[r, 2 * 64 + 7] = x
    cos, sin = torch.ones(1, 64, device=DEV).bfloat16(), torch.zeros(1, 64, device=DEV).bfloat16()
    k = torch.zeros(1, nkv, ps, 64, dtype=torch.float8_e4m3fn, device=DEV)
    v, ks = k.clone(), torch.zeros(1, nkv, ps, dtype=torch.uint8, device=DEV)
    vs = ks.clone()
    layer = sp.KVLayer(k, v, torch.zeros(1, 1, dtype=torch.int32, device=DEV), ks, vs)
    i = torch.arange(6, dtype=torch.int32, device=DEV)
    z = torch.zeros_like(i)
    err = _err()
    sp.kv_write(layer, qkv, cos, sin, z, i, z, torch.empty(6, nq, 64, dtype=torch.bfloat16, device=DEV), error=err)
    kk, vv = sp.kv_read(layer, torch.tensor([6], dtype=torch.int32, device=DEV), 8, error=err)
    assert int(err) == 0
    assert (vs[0, 0, :3] == NAN_BYTE).all() and vv[0, 0, :3].isnan().all()
    ref = qkv[3:, 128:].double().view(3, 32, 2).transpose(1, 2).reshape(3, 64)
    y, byte, _ = _quantise(ref)
    assert torch.equal(vs[0, 0, 3:6], byte)
    assert torch.equal(vv[0, 0, 3:6].double(), (y * _pow2(byte.to(torch.int64) - 127)[:, None]).bfloat16().double())
    assert not kk[0, 0].float().any() and not vv[0, 0, 6:].float().any()


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("lengths,nkv,ps", [([1], 8, 64), ([0, 5, 129, 40], 2, 24), ([77, 300, 1], 1, 8)])
def test_read(fmt, lengths, nkv, ps):
    g = _gen(len(lengths))
    batch, n = len(lengths), max(lengths)
    blocks = -(-n // ps)
    pages = batch * blocks + 1
    tables = _tables(batch, blocks, pages, g)
    k, v, ks, vs, k64, v64 = _pool(pages, nkv, ps, fmt, g, scale=30.0)
    err = _err()
    lens = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    outs = sp.kv_read(sp.KVLayer(k, v, tables, ks, vs), lens, n, error=err)
    assert int(err) == 0
    for got, ref in zip(outs, (k64, v64)):
        for b, m in enumerate(lengths):
            p = torch.arange(m, device=DEV)
            want = ref[tables[b].long()[p // ps], :, p % ps].transpose(0, 1)
            assert torch.equal(got[b, :, :m].double(), want)
            assert not got[b, :, m:].float().any()


# ------------------------------------------------------------------ tree attention
def _tree_masks(nodes, kind, g):
    """Per sequence a bool [n, n]; trees from random parents, chains causal, "empty" has rows of nothing."""
    out = []
    for n in nodes:
        a = torch.zeros(n, n, dtype=torch.bool)
        for i in range(n):
            if kind == "chain":
                a[i, :i + 1] = True
                continue
            p = int(torch.randint(-1, max(i, 1), (1,), generator=g)) if i else -1
            if p >= 0:
                a[i] = a[p]
            a[i, i] = True
        if kind == "empty" and n:
            a[::3] = False
        out.append(a)
    return out


def _words(masks, width):
    rows = sum(len(a) for a in masks)
    w = -(-width // 64)
    full = torch.zeros(rows, w * 64, dtype=torch.bool)
    at = 0
    for a in masks:
        full[at:at + len(a), :len(a)] = a
        full[at:at + len(a), len(a):] = True  # bits past the nodes mean nothing
        at += len(a)
    bit = torch.ones(64, dtype=torch.int64) << torch.arange(64)
    return (full.view(rows, w, 64).long() * bit).sum(-1).to(DEV)


def _setup(prefixes, nodes, nq, nkv, ps, fmt, kind, seed, qscale=1.5):
    g = _gen(seed)
    batch, max_len = len(nodes), max(p + n for p, n in zip(prefixes, nodes))
    blocks = max(1, -(-max_len // ps))
    pages = batch * blocks + 2
    k, v, ks, vs, k64, v64 = _pool(pages, nkv, ps, fmt, g)
    masks = _tree_masks(nodes, kind, torch.Generator().manual_seed(seed))
    T = max(nodes)
    rows = sum(nodes)
    return dict(prefixes=prefixes, nodes=nodes, masks=masks, T=T, max_len=max_len, k=k, v=v, ks=ks, vs=vs,
                k64=k64, v64=v64, tables=(tables := _tables(batch, blocks, pages, g)), right_tables=tables.clone(), ps=ps,
                q=(torch.randn(rows, nq, 64, generator=g, device=DEV) * qscale).bfloat16(),
                mask=_words(masks, T), prefix=torch.tensor(prefixes, dtype=torch.int32, device=DEV),
                cu=torch.tensor([sum(nodes[:b]) for b in range(batch + 1)], dtype=torch.int32, device=DEV))


def _attend(s, err=None, **kw):
    err = _err() if err is None else err
    out = sp.tree_attention(s["q"], sp.KVLayer(s["k"], s["v"], s["tables"], s["ks"], s["vs"]), s["cu"], s["mask"],
                            s["prefix"], s["T"], s["max_len"], error=err, **kw)
    return (*out, err)


def _check(s, out, lse, skip=()):
    nq, nkv, ps = s["q"].shape[1], s["k"].shape[1], s["ps"]
    group, at = nq // nkv, 0
    for b, (p, n) in enumerate(zip(s["prefixes"], s["nodes"])):
        j = torch.arange(p + n, device=DEV)
        pg = s["right_tables"][b].long()[j // ps]
        kk, vv = (s[x][pg, :, j % ps].transpose(0, 1).repeat_interleave(group, 0) for x in ("k64", "v64"))
        q = s["q"][at:at + n].double().transpose(0, 1)
        seen = torch.cat([torch.ones(n, p, dtype=torch.bool), s["masks"][b]], 1).to(DEV)
        x = torch.where(seen, (q @ kk.transpose(1, 2)) * 0.125, -math.inf)
        d = 64 * 2.0 ** -23 * float((q.abs() @ kk.abs().transpose(1, 2)).max()) * 0.125 if n and p + n else 0.0
        w = torch.where(seen.any(1, keepdim=True), torch.softmax(x, -1), 0.0)
        ref, size = w @ vv, w @ vv.abs()
        got, ls = out[at:at + n].double().transpose(0, 1), lse[at:at + n].double().T
        want = torch.logsumexp(x, -1)
        for i in range(n):
            if (b, i) in skip:
                continue
            if not seen[i].any():
                assert not got[:, i].any() and (ls[:, i] == -math.inf).all(), (b, i)
                continue
            tol = (U + 4 * d + 2.0 ** -18) * size[:, i] + U * ref[:, i].abs()
            off = (got[:, i] - ref[:, i]).abs()
            assert (off <= tol).all(), (b, i, float((off / tol).max()))
            assert ((ls[:, i] - want[:, i]).abs() <= 2 * d + 2.0 ** -18 + 2.0 ** -22 * want[:, i].abs()).all(), (b, i)
        at += n


SHAPES = [
    # prefixes, nodes, nq, nkv, page size
    ([0], [1], 32, 8, 64),
    ([1024], [1], 32, 8, 64),
    ([0, 1, 31, 32, 33, 63, 64, 65, 300], [1] * 9, 4, 1, 8),
    ([5, 0, 700, 129], [2, 4, 1, 3], 8, 2, 24),
    ([100, 0, 511, 64], [5, 0, 8, 7], 32, 8, 16),
    ([260, 17, 0], [16, 9, 13], 16, 8, 32),
    ([1000, 3], [25, 31], 32, 8, 64),
    ([127, 0, 128, 129], [64, 63, 33, 1], 8, 2, 128),
    ([400, 90], [65, 130], 4, 1, 40),
    ([1025, 0], [256, 200], 8, 4, 64),
    ([513], [32], 8, 8, 64),
    ([77, 1200], [3, 40], 16, 2, 8),
    ([5000], [1], 8, 1, 64),
    ([6001], [20], 4, 1, 16),
]


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_tree_attention(fmt, i):
    prefixes, nodes, nq, nkv, ps = SHAPES[i]
    s = _setup(prefixes, nodes, nq, nkv, ps, fmt, ("tree", "chain", "empty")[i % 3], seed=i)
    out, lse, err = _attend(s)
    assert int(err) == 0
    _check(s, out, lse)
    again, lse2, _ = _attend(s)  # no order of additions depends on the run
    assert torch.equal(out, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("nodes", [1, 4, 8])
def test_full_gpu_of_long_sequences(fmt, nodes):
    """Every ring goes round many times while copies finish in any order: each call gives
    the same bits, the right ones."""
    s = _setup([4096 - 61 * i for i in range(32)], [nodes] * 32, 32, 8, 64, fmt, "tree", seed=nodes)
    out, lse, err = _attend(s)
    for _ in range(30):
        again, lse2, _ = _attend(s, err=err)
        assert torch.equal(out, again) and torch.equal(lse, lse2)
    assert int(err) == 0
    for b in range(0, 32, 5):  # the comparison in 64 bits, of some
        rows = slice(b * nodes, (b + 1) * nodes)
        one = dict(s, prefixes=s["prefixes"][b:b + 1], nodes=[nodes], masks=s["masks"][b:b + 1], q=s["q"][rows],
                   right_tables=s["right_tables"][b:b + 1])
        _check(one, out[rows], lse[rows])


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("nodes", [1, 7, 40])
def test_large_scores(fmt, nodes):
    """Scores of hundreds: the running maximum has to carry the sums."""
    s = _setup([300, 90], [nodes, nodes], 8, 2, 16, fmt, "chain", seed=nodes, qscale=60.0)
    out, lse, err = _attend(s)
    assert int(err) == 0
    _check(s, out, lse)


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("nodes", [2, 9, 50, 140])
def test_masked_places_have_no_effect(fmt, nodes):
    """NaN and infinities behind the last node, in nodes that a row does not see and
    in pages of nobody change nothing; a row that sees one is not finite."""
    s = _setup([45, 0, 130], [nodes, nodes, 1], 8, 2, 24, fmt, "tree", seed=nodes)
    used = torch.zeros(s["k"].shape[0], s["ps"], dtype=torch.bool, device=DEV)
    for b, (p, n) in enumerate(zip(s["prefixes"], s["nodes"])):
        j = torch.arange(p + n, device=DEV)
        used[s["tables"][b].long()[j // s["ps"]], j % s["ps"]] = True
    bad_node = nodes - 1  # of sequences 0 and 1: a leaf, seen by itself only
    where = ~used[:, None, :].expand(s["k"].shape[:3]).clone()
    for b in (0, 1):
        at = s["prefixes"][b] + bad_node
        where[int(s["tables"][b, at // s["ps"]]), :, at % s["ps"]] = True
    if fmt == "bf16":
        s["k"][where] = math.nan
        s["v"][where] = math.inf
        s["v"][..., ::2][where] = math.nan
    else:
        s["k"].view(torch.uint8)[where] = 0x7F
        s["v"].view(torch.uint8)[where] = 0xFF
        s["ks"][where] = NAN_BYTE
        s["vs"][where] = NAN_BYTE
    out, lse, err = _attend(s)
    assert int(err) == 0
    _check(s, out, lse, skip={(0, bad_node), (1, bad_node)})
    for row in (bad_node, nodes + bad_node):
        assert not out[row].isfinite().any() and lse[row].isnan().all()


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("prefix", [300, 640, 1500, 2047])
def test_masked_places_behind_long_prefixes(fmt, prefix):
    """The blocks with drafted nodes come after many without: what lies behind the last
    node, and in a node that only itself sees, still has no effect, on a busy GPU."""
    batch, nodes = 24, 20
    s = _setup([prefix - i for i in range(batch)], [nodes] * batch, 32, 8, 64, fmt, "tree", seed=prefix)
    where = torch.zeros(s["k"].shape[:3], dtype=torch.bool, device=DEV)
    for b, p in enumerate(s["prefixes"]):
        at = torch.arange(p + nodes - 1, s["tables"].shape[1] * 64, device=DEV)  # a leaf, and all behind it
        where[s["tables"][b].long()[at // 64], :, at % 64] = True
    if fmt == "bf16":
        s["v"][where] = math.nan
    else:
        s["v"].view(torch.uint8)[where] = 0xFF
        s["vs"][where] = NAN_BYTE
    err = _err()
    out, lse, _ = _attend(s, err=err)
    for _ in range(20):
        again, lse2, _ = _attend(s, err=err)
        assert torch.equal(out.view(torch.int16), again.view(torch.int16))
        assert torch.equal(lse.view(torch.int32), lse2.view(torch.int32))
    assert int(err) == 0
    leaves = torch.arange(nodes - 1, batch * nodes, nodes, device=DEV)
    assert out[leaves].isnan().all() and lse[leaves].isnan().all()
    for b in range(0, batch, 7):
        rows = slice(b * nodes, (b + 1) * nodes)
        one = dict(s, prefixes=s["prefixes"][b:b + 1], nodes=[nodes], masks=s["masks"][b:b + 1], q=s["q"][rows],
                   right_tables=s["right_tables"][b:b + 1])
        _check(one, out[rows], lse[rows], skip={(0, nodes - 1)})


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
def test_value_of_a_seen_node_is_not_finite(fmt):
    """Only V holds the NaN: rows that see the node are not finite, the others are untouched."""
    s = _setup([70], [30], 8, 2, 16, fmt, "chain", seed=3)
    at = 70 + 20
    page = int(s["tables"][0, at // 16])
    if fmt == "bf16":
        s["v"][page, :, at % 16, 5] = math.nan
    else:
        s["vs"][page, :, at % 16] = NAN_BYTE
    out, lse, err = _attend(s)
    assert int(err) == 0
    _check(s, out, lse, skip={(0, i) for i in range(20, 30)})
    assert not out[20:, :, 5].isfinite().any()


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("nodes", [1, 4, 20])
@pytest.mark.parametrize("which", ["k", "v"])
def test_committed_row_is_not_finite(fmt, nodes, which):
    """A NaN row at any place of a block of committed positions makes its K/V head's
    results NaN, and no others."""
    batch, nq, nkv = 64, 8, 2
    s = _setup([300] * batch, [nodes] * batch, nq, nkv, 16, fmt, "chain", seed=nodes)
    b = torch.arange(batch, device=DEV)
    page, off = s["tables"][b, (64 + b) // 16].long(), (64 + b) % 16  # position 64 + b of sequence b
    if fmt == "bf16":
        s[which][page, 0, off] = math.nan
    else:
        s[which + "s"][page, 0, off] = NAN_BYTE
    out, lse, err = _attend(s)
    assert int(err) == 0
    assert out[:, :nq // nkv].isnan().all() and out[:, nq // nkv:].isfinite().all()
    assert lse[:, nq // nkv:].isfinite().all()
    if which == "k":
        assert lse[:, :nq // nkv].isnan().all()


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("nodes", [1, 20])
def test_more_ranges_than_a_cluster(fmt, nodes):
    """Few long sequences are split further than a cluster joins: partials in the workspace."""
    s = _setup([17000, 40, 9000], [nodes] * 3, 4, 1, 64, fmt, "tree", seed=nodes)
    nbytes = _lib.load().mk_tree_attention_workspace(3, 4, 1, nodes, s["max_len"])
    assert nbytes > 0
    ws = torch.empty(nbytes + 8, dtype=torch.uint8, device=DEV)
    out, lse, err = _attend(s, workspace=ws[:nbytes])
    assert int(err) == 0
    _check(s, out, lse)
    with pytest.raises(_lib.MkError, match="16-byte"):
        _attend(s, workspace=ws[8:])
    with pytest.raises(_lib.MkError, match="workspace"):
        _attend(s, workspace=ws[:nbytes - 16])


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("batch,nodes,nq,nkv", [(70, 20, 8, 4), (100, 1, 8, 8), (33, 40, 16, 8)])
def test_many_ragged_sequences(fmt, batch, nodes, nq, nkv):
    """More CTAs than SMs or slots: the longer sequences go first, each exactly once."""
    lengths = [(37 * i * i) % 700 if i % 5 else 300 for i in range(batch)]
    lengths[3] = 0
    s = _setup(lengths, [nodes - (i % 2 if nodes > 1 else 0) for i in range(batch)], nq, nkv, 16, fmt, "tree", seed=batch)
    out, lse, err = _attend(s)
    assert int(err) == 0
    _check(s, out, lse)


def test_strided_sequences_of_a_larger_table_and_other_stream():
    """Fewer sequences than the table has rows, on a stream of its own."""
    s = _setup([90, 33, 200], [6, 2, 11], 8, 2, 16, "e4m3", "tree", seed=8)
    wide = torch.full((5, s["tables"].shape[1] + 3), -1, dtype=torch.int32, device=DEV)
    wide[:3, :s["tables"].shape[1]] = s["tables"]
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        err = _err()
        out, lse = sp.tree_attention(s["q"], sp.KVLayer(s["k"], s["v"], wide, s["ks"], s["vs"]), s["cu"], s["mask"],
                                     s["prefix"], s["T"], s["max_len"] + 40, error=err)
    st.synchronize()
    assert int(err) == 0
    _check(s, out, lse)


@pytest.mark.parametrize("nodes", [1, 3, 40])
def test_captured_in_a_graph(nodes):
    s = _setup([90, 400], [nodes, nodes], 8, 2, 16, "e4m3", "chain", seed=nodes)
    layer, err = sp.KVLayer(s["k"], s["v"], s["tables"], s["ks"], s["vs"]), _err()
    args = (s["q"], layer, s["cu"], s["mask"], s["prefix"], s["T"], s["max_len"])
    out, lse, _ = _attend(s)
    o2, l2 = torch.empty_like(out), torch.empty_like(lse)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sp.tree_attention(*args, out=o2, lse=l2, error=err)
    for _ in range(3):
        o2.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, o2) and torch.equal(lse, l2)
    assert int(err) == 0


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("nodes", [1, 20])
def test_pool_beyond_32_bits(fmt, nodes):
    """Pages whose byte offsets pass 2^32: the write, the attention and the read agree
    with the same pages in a small pool."""
    ps, nkv, nq = 64, 2, 8
    pages = (2 ** 32 // (128 if fmt == "bf16" else 64)) // (nkv * ps) + 40
    s = _setup([200], [nodes], nq, nkv, ps, fmt, "chain", seed=9)
    big = {}
    for x in ("k", "v"):
        big[x] = torch.empty(pages, nkv, ps, 64, dtype=s[x].dtype, device=DEV)
        big[x].view(torch.uint8)[-s[x].shape[0]:] = s[x].view(torch.uint8)
    for x in ("ks", "vs"):
        big[x] = None
        if fmt == "e4m3":
            big[x] = torch.empty(pages, nkv, ps, dtype=torch.uint8, device=DEV)
            big[x][-s[x].shape[0]:] = s[x]
    tables = (s["tables"] + (pages - s["k"].shape[0])).contiguous()
    out, lse, err = _attend(s)
    layer = sp.KVLayer(big["k"], big["v"], tables, big["ks"], big["vs"])
    o2, l2 = sp.tree_attention(s["q"], layer, s["cu"], s["mask"], s["prefix"], s["T"], s["max_len"], error=err)
    assert torch.equal(out, o2) and torch.equal(lse, l2)
    n = torch.tensor([200], dtype=torch.int32, device=DEV)
    small = sp.KVLayer(s["k"], s["v"], s["tables"], s["ks"], s["vs"])
    assert all(torch.equal(a, b) for a, b in zip(sp.kv_read(layer, n, 200), sp.kv_read(small, n, 200)))
    qkv = torch.randn(1, (nq + 2 * nkv) * 64, generator=_gen(1), device=DEV).bfloat16()
    one = torch.ones(1, 64, device=DEV).bfloat16()
    z = torch.zeros(1, dtype=torch.int32, device=DEV)
    qo = torch.empty(1, nq, 64, dtype=torch.bfloat16, device=DEV)
    for lay in (layer, small):
        sp.kv_write(lay, qkv, one, one, z, z + 3, z, qo, error=err)
    assert all(torch.equal(a, b) for a, b in zip(sp.kv_read(layer, n, 200), sp.kv_read(small, n, 200)))
    assert int(err) == 0


@pytest.mark.parametrize("nodes", [1, 12, 70])
def test_device_side_refusals(nodes):
    """Bad pages, lengths and node ranges are reported, and the other sequences still right."""
    for what in ("page", "prefix", "nodes"):
        s = _setup([150, 60, 90], [nodes] * 3, 8, 2, 16, "bf16", "chain", seed=4)
        if what == "page":
            s["tables"][1, 2] = s["k"].shape[0]
        elif what == "prefix":
            s["prefix"][1] = s["max_len"] + 5
        else:
            s["cu"][2] = s["cu"][1] - 1  # sequence 1 has -1 nodes, sequence 2 one too many or its own
            s["prefixes"] = s["prefixes"][:1]
            s["nodes"] = s["nodes"][:1]
        out, lse, err = _attend(s)
        assert int(err) == 1
        if what != "nodes":
            skip = {(1, i) for i in range(nodes)}
            _check(s, out, lse, skip=skip)
        else:
            _check(s, out, lse)


def test_write_and_read_device_side_refusals():
    g = _gen(0)
    k, v, ks, vs, _, _ = _pool(4, 1, 8, "e4m3", g)
    tables = torch.tensor([[0, 1], [2, 9]], dtype=torch.int32, device=DEV)
    layer = sp.KVLayer(k, v, tables, ks, vs)
    one = torch.ones(4, 64, device=DEV).bfloat16()
    was = [t.clone() for t in (k.view(torch.uint8), v.view(torch.uint8), ks, vs)]
    for seq, slot, pos in ((2, 0, 0), (-1, 0, 0), (0, 16, 0), (0, -2, 0), (1, 8, 0), (0, 0, 4), (0, 0, -1)):
        args = [torch.tensor([x], dtype=torch.int32, device=DEV) for x in (seq, slot, pos)]
        err = _err()
        qkv = torch.randn(1, 3 * 64, generator=g, device=DEV).bfloat16()
        sp.kv_write(layer, qkv, one, one, *args, torch.empty(1, 1, 64, dtype=torch.bfloat16, device=DEV), error=err)
        assert int(err) == 1, (seq, slot, pos)
        now = (k.view(torch.uint8), v.view(torch.uint8), ks, vs)
        if pos == 0:
            assert all(torch.equal(a, b) for a, b in zip(was, now))
        else:  # only V, which is not rotated
            assert torch.equal(was[0], now[0]) and torch.equal(was[2], now[2])
    err = _err()
    sp.kv_read(layer, torch.tensor([3, 9], dtype=torch.int32, device=DEV), 9, error=err)
    assert int(err) == 1


def test_argument_refusals():
    s = _setup([20], [3], 8, 2, 16, "e4m3", "chain", seed=1)
    layer = sp.KVLayer(s["k"], s["v"], s["tables"], s["ks"], s["vs"])
    args = dict(q=s["q"], layer=layer, cu_nodes=s["cu"], mask=s["mask"], prefix_lens=s["prefix"], max_nodes=3,
                max_len=23)

    def refused(**kw):
        with pytest.raises((ValueError, sp._lib.MkError)):
            sp.tree_attention(**{**args, **kw})

    refused(q=s["q"].float())
    refused(q=s["q"].transpose(0, 1))
    refused(q=s["q"][:, :7].contiguous())  # 7 query heads on 2
    refused(cu_nodes=s["cu"][:1])
    refused(cu_nodes=s["cu"].long())
    refused(mask=torch.cat([s["mask"], s["mask"]], 1))
    refused(max_nodes=257)
    refused(max_nodes=0)
    refused(max_len=s["tables"].shape[1] * 16 + 1)
    refused(prefix_lens=s["prefix"].cpu())
    refused(workspace=torch.empty(1, dtype=torch.uint8, device=DEV), max_nodes=3, max_len=0)
    with pytest.raises(ValueError):
        sp.KVLayer(s["k"], s["v"], s["tables"])  # codes without scales
    with pytest.raises(ValueError):
        sp.KVLayer(s["k"], s["v"], s["tables"], s["ks"])
    with pytest.raises(ValueError):
        sp.kv_read(layer, torch.zeros(9, dtype=torch.int32, device=DEV), 4)
    x = torch.zeros(2, 50, device=DEV)
    for bad in (dict(top=33), dict(top=-1), dict(targets=torch.zeros(2, 1, device=DEV)),
                dict(targets=torch.zeros(3, 1, dtype=torch.int32, device=DEV))):
        with pytest.raises((ValueError, RuntimeError)):
            sp.token_logprobs(x, **bad)
    for t in (x.half(), x.T, x.cpu()):
        with pytest.raises(ValueError):
            sp.token_logprobs(t)


# ------------------------------------------------------------------ log probabilities
def _logprobs_ref(x, targets, top):
    x = x.double()
    lse = torch.logsumexp(x, -1, keepdim=True)
    lp = torch.where(x == -math.inf, -math.inf, x - lse)
    ent = -torch.where(lp == -math.inf, 0.0, lp * lp.exp()).sum(-1)
    t = targets.long()
    got = torch.where(t >= 0, torch.gather(lp, 1, t.clamp(min=0)), 0.0)
    ids = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top]
    return got, ent, ids, torch.gather(lp, 1, ids)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,n,top,kind", [
    (1, 128256, 1, 20, "normal"), (3, 128256, 4, 32, "ties"), (70, 5003, 2, 5, "banned"), (5, 1, 1, 1, "normal"),
    (2, 33, 3, 32, "ties"), (4, 1000, 1, 0, "normal"), (300, 4099, 1, 8, "sorted"), (9, 32064, 0, 7, "equal"),
    (2, 64128, 1, 32, "few"), (17, 8200, 1, 31, "steep")])
def test_logprobs(dtype, rows, vocab, n, top, kind):
    g = _gen(vocab + top)
    x = torch.randn(rows, vocab, generator=g, device=DEV) * 3
    if kind == "ties":
        x = (x * 2).round() / 2
        x[:, 0] = 0.0
        x[:, vocab // 2] = -0.0
    elif kind == "banned":
        x[:, torch.rand(vocab, generator=g, device=DEV) < 0.6] = -math.inf
    elif kind == "few":
        x.fill_(-math.inf)
        x[:, 7::9001] = 1.5
    elif kind == "sorted":
        x = x.sort(dim=-1).values
    elif kind == "equal":
        x.fill_(-2.25)
    elif kind == "steep":
        x[:, vocab // 3] = 300.0
    x = x.to(dtype)
    targets = torch.randint(-1, vocab, (rows, n), generator=g, device=DEV).to(torch.int32)
    err = _err()
    lp, ent, ids, tlp = sp.token_logprobs(x, targets if n else None, top, error=err)
    assert int(err) == 0
    rlp, rent, rids, rtlp = _logprobs_ref(x, targets, top)
    assert torch.equal(ids.long(), rids)
    fin = x.double()
    fin = torch.where(fin == -math.inf, 0.0, fin)
    tol = 2.0 ** -14 + 2.0 ** -22 * float(fin.abs().max())
    for got, ref in ((lp, rlp), (tlp, rtlp)):
        inf = ref == -math.inf
        assert torch.equal(got == -math.inf, inf)
        assert ((got.double() - ref).abs() <= tol)[~inf].all()
    mean = ((fin - fin.amax(-1, keepdim=True)) * torch.softmax(x.double(), -1)).sum(-1).abs()
    assert ((ent.double() - rent).abs() <= tol * (1 + mean)).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_logprobs_of_strided_rows_and_odd_rows(dtype):
    g = _gen(5)
    wide = (torch.randn(6, 3001, generator=g, device=DEV) * 2).to(dtype)
    for x in (wide[:, 1:2000], wide[:, 3:3000], wide[::2, :1003], wide[:1, 2:]):
        ids = torch.randint(x.shape[1], (x.shape[0], 2), generator=g, device=DEV).to(torch.int32)
        lp, ent, top, tlp = sp.token_logprobs(x, ids, 9)
        rlp, rent, rids, rtlp = _logprobs_ref(x, ids, 9)
        assert torch.equal(top.long(), rids)
        assert ((lp - rlp).abs() <= 2.0 ** -13).all() and ((tlp - rtlp).abs() <= 2.0 ** -13).all()
        assert ((ent - rent).abs() <= 10 * 2.0 ** -13).all()


@pytest.mark.parametrize("vocab", [50, 20000])
def test_logprobs_of_rows_without_a_distribution(vocab):
    x = torch.randn(4, vocab, generator=_gen(2), device=DEV)
    x[0] = -math.inf
    x[1, 3] = math.nan
    x[2, 4] = math.inf
    t = torch.full((4, 1), 5, dtype=torch.int32, device=DEV)
    lp, ent, ids, tlp = sp.token_logprobs(x, t, 4)
    assert lp[0, 0] == -math.inf and ent[0] == 0 and (tlp[0] == -math.inf).all()
    assert ids[0].tolist() == [0, 1, 2, 3]
    for r in (1, 2):
        assert lp[r].isnan().all() and ent[r].isnan() and tlp[r].isnan().all()
        assert ((ids[r] >= 0) & (ids[r] < vocab)).all()
    assert lp[3].isfinite().all() and ent[3].isfinite()
    err = _err()
    t[3] = vocab
    lp, *_ = sp.token_logprobs(x, t, 0, error=err)
    assert int(err) == 1 and lp[3].isnan().all()
