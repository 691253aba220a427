"""What the speculative-decoding operators are timed on: writing drafted rows into a paged 8-bit
K/V cache and reading it back, attention of a tree of drafted tokens over a paged cache, and the
log probabilities of given tokens.

Each case is one call of one operator. With ``own`` false ``run`` evaluates its formula with
elementary tensor operations in 32 bits, rounded once at the end; with ``own`` true it makes the
call of ``llama1b_megakernel_b200.speculative`` on the same inputs. ``exact`` evaluates the
definition in 64 bits.

Head layouts are those of the decoder configurations: 32 query heads on 8 K/V heads of 64
(Llama-3.2-1B), and its tensor-parallel shards and small variants.
"""
import math

import torch

own = False

D = 64  # head dimension
ROPE_LEN = 32768

# The vocabulary of the full-size configuration.
VOCAB = 128256


def listed():
    return [
        # One sequence decodes one token: its q/k/v row is rotated and enters the 8-bit cache.
        {"name": "write 1 row", "op": "write", "rows": 1, "batch": 1, "nq": 32, "nkv": 8, "page": 64, "ctx": 1024},
        # A long prompt's rows enter the cache in one pass (4093: not a multiple of anything).
        {"name": "write 4093 rows", "op": "write", "rows": 4093, "batch": 7, "nq": 32, "nkv": 8, "page": 16, "ctx": 2048},
        # One sequence's 8-bit rows of a layer leave the cache as bf16.
        {"name": "read 1 x 129", "op": "read", "batch": 1, "nkv": 8, "page": 64, "ctx": 129, "spread": 0},
        # A batch of ragged sequences handed over to code that wants contiguous bf16 rows.
        {"name": "read 32 x 8191", "op": "read", "batch": 32, "nkv": 8, "page": 64, "ctx": 8191, "spread": 4000},
        # The single-token form: plain decode of one sequence at the headline context.
        {"name": "decode 1 x 1025 bf16", "op": "attention", "batch": 1, "nodes": 1, "jitter": 0, "nq": 32, "nkv": 8, "page": 64, "ctx": 1024, "spread": 0, "cache": "bf16", "kind": "chain"},
        # Decode of a full batch over the 8-bit cache, ragged lengths.
        {"name": "decode 64 x 4097 e4m3", "op": "attention", "batch": 64, "nodes": 1, "jitter": 0, "nq": 32, "nkv": 8, "page": 64, "ctx": 4096, "spread": 1500, "cache": "e4m3", "kind": "chain"},
        # A draft tree of about 25 nodes for eight sequences, small pages, some rows without any key.
        {"name": "tree 8 x 25 bf16", "op": "attention", "batch": 8, "nodes": 25, "jitter": 9, "nq": 32, "nkv": 8, "page": 16, "ctx": 1111, "spread": 1111, "cache": "bf16", "kind": "tree"},
        # The largest draft trees over long 8-bit contexts.
        {"name": "tree 32 x 64 e4m3", "op": "attention", "batch": 32, "nodes": 64, "jitter": 0, "nq": 32, "nkv": 8, "page": 64, "ctx": 8192, "spread": 3000, "cache": "e4m3", "kind": "tree"},
        # A chunk of a prompt against its long cached beginning: causal rows.
        {"name": "chunk 4 x 256 bf16", "op": "attention", "batch": 4, "nodes": 256, "jitter": 31, "nq": 32, "nkv": 8, "page": 64, "ctx": 16000, "spread": 5000, "cache": "bf16", "kind": "chain"},
        # Log probabilities of one decoded token with twenty alternatives.
        {"name": "logprobs 1", "op": "logprobs", "rows": 1, "vocab": VOCAB, "targets": 1, "top": 20, "dtype": "float32", "banned": 0.0},
        # The nodes of draft trees, each scored for its children, part of the vocabulary forbidden.
        {"name": "logprobs 200", "op": "logprobs", "rows": 200, "vocab": VOCAB, "targets": 4, "top": 5, "dtype": "bfloat16", "banned": 0.3},
        # A prompt scored token by token.
        {"name": "logprobs 2047", "op": "logprobs", "rows": 2047, "vocab": VOCAB, "targets": 1, "top": 8, "dtype": "float32", "banned": 0.0},
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["write", "read", "attention", "attention", "attention", "logprobs"])
    heads = rng.choice([(32, 8), (32, 8), (16, 4), (8, 2), (4, 1), (8, 8), (16, 2), (8, 4)])
    page = rng.choice([8, 16, 24, 32, 64, 128])
    if op == "write":
        return {"op": op, "rows": _log_uniform(rng, 1, 4093), "batch": rng.randint(1, 32), "nq": heads[0], "nkv": heads[1], "page": page, "ctx": _log_uniform(rng, 200, 4096)}
    if op == "read":
        batch, ctx = _log_uniform(rng, 1, 29), _log_uniform(rng, 1, 8191)
        return {"op": op, "batch": batch, "nkv": heads[1], "page": page, "ctx": ctx, "spread": rng.randint(0, ctx)}
    if op == "logprobs":
        rows = _log_uniform(rng, 1, 1800)
        vocab = rng.choice([VOCAB, VOCAB // 2, VOCAB // 4, 5003, 4099, 1000])
        return {"op": op, "rows": rows, "vocab": vocab, "targets": rng.randint(1, 6), "top": rng.randint(0, 20), "dtype": rng.choice(["float32", "float32", "bfloat16"]), "banned": rng.choice([0.0, 0.0, 0.5])}
    while True:
        kind = rng.choice(["tree", "tree", "chain"])
        nodes = _log_uniform(rng, 1, 64 if kind == "tree" else 256)
        batch, ctx = _log_uniform(rng, 1, 64), _log_uniform(rng, 1, 16000)
        case = {"op": op, "batch": batch, "nodes": nodes, "jitter": rng.randint(0, nodes - 1), "nq": heads[0], "nkv": heads[1], "page": page, "ctx": ctx, "spread": rng.randint(0, ctx), "cache": rng.choice(["bf16", "e4m3"]), "kind": kind}
        w = work(case)
        if w["flops"] <= 110e9 and w["bytes"] <= 220e6:
            return case


# ------------------------------------------------------------------ sizes that follow from a case


def _prefixes(case):
    """Cached positions of each sequence before the drafted ones (or all of them, for a read);
    where they spread over half the range, every fourth sequence has none yet."""
    wide = 2 * case["spread"] >= case["ctx"]
    return [0 if wide and b % 4 == 3 else case["ctx"] - (b * 977) % (case["spread"] + 1) for b in range(case["batch"])]


def _nodes(case):
    return [case["nodes"] - (b * 5) % (case["jitter"] + 1) for b in range(case["batch"])]


def work(case):
    if case["op"] == "write":
        nh = case["nq"] + 2 * case["nkv"]
        per_row = nh * D * 2 + case["nq"] * D * 2 + 2 * case["nkv"] * (D + 1) + 12
        return {"bytes": case["rows"] * (per_row + 2 * D * 2), "flops": case["rows"] * nh * D * 3}
    if case["op"] == "read":
        n = sum(_prefixes(case)) * case["nkv"]
        written = case["batch"] * case["ctx"] * case["nkv"] * 2 * D * 2
        return {"bytes": n * 2 * (D + 1) + written, "flops": n * 2 * D}
    if case["op"] == "logprobs":
        size = 4 if case["dtype"] == "float32" else 2
        return {"bytes": case["rows"] * (case["vocab"] * size + 8 * case["targets"] + 4 + 8 * case["top"]), "flops": case["rows"] * case["vocab"] * 5}
    per_key = 2 * D * 2 if case["cache"] == "bf16" else 2 * (D + 1)
    pairs = keys = rows = 0
    for p, n in zip(_prefixes(case), _nodes(case)):
        keys += p + n
        rows += n
        pairs += n * p + (n * (n + 1) // 2 if case["kind"] == "chain" else n)
    words = -(-case["nodes"] // 64)
    return {"bytes": keys * case["nkv"] * per_key + rows * case["nq"] * (D * 4 + 4) + rows * 8 * words, "flops": pairs * case["nq"] * 4 * D}


# ------------------------------------------------------------------ inputs


def _rope(device):
    """bf16 cos / sin rows of every position (theta 500000, halves repeated)."""
    inv = 500000.0 ** (-torch.arange(0, D, 2, device=device, dtype=torch.float64) / D)
    ang = torch.arange(ROPE_LEN, device=device, dtype=torch.float64)[:, None] * inv[None, :]
    ang = torch.cat([ang, ang], dim=1)
    return ang.cos().bfloat16(), ang.sin().bfloat16()


def _tables(batch, blocks, g, device):
    """Every sequence's pages, in a random order, out of a pool with a few more."""
    pages = batch * blocks + 3
    perm = torch.randperm(pages, generator=g, device=device)[: batch * blocks]
    return perm.view(batch, blocks).to(torch.int32), pages


def _cached(shape, g, device):
    """Cached K or V rows as they come: unit size, a few channels several times larger."""
    gain = torch.ones(D, device=device)
    gain[5], gain[17], gain[40] = 6.0, 3.0, 4.0
    return torch.randn(shape, generator=g, device=device) * gain


def _power(e):
    """2**e in fp32 for integers e in [-126, 127], from its bits."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _encode(x):
    """float rows [..., 64] -> (e4m3 codes, one power-of-two scale byte a row): the smallest
    exponent e, at least -110, with amax <= 448 * 2**e; the byte is e + 127."""
    frac, e2 = torch.frexp(x.abs().amax(-1))
    e = (e2 - 9 + (frac > 0.875).to(e2.dtype)).clamp(min=-110)
    e = torch.where(frac == 0, torch.full_like(e, -110), e)
    codes = (x * _power(-e)[..., None]).to(torch.float8_e4m3fn)
    return codes, (e + 127).to(torch.uint8)


def _decode(codes, scales):
    return codes.float() * _power(scales.to(torch.int32) - 127)[..., None]


def prepare(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device=device).manual_seed(seed)
    s = {"case": case, "error": torch.zeros(1, dtype=torch.int32, device=device)}
    if case["op"] == "logprobs":
        dt = torch.float32 if case["dtype"] == "float32" else torch.bfloat16
        rows, V = case["rows"], case["vocab"]
        x = torch.randn(rows, V, generator=g, device=device).mul_(2.5)
        t = torch.randint(V, (rows, case["targets"]), generator=g, device=device)
        x.scatter_add_(1, t[:, :1], torch.rand(rows, 1, generator=g, device=device) * 20)
        if case["banned"]:
            x.masked_fill_(torch.rand(1, V, generator=g, device=device) < case["banned"], -math.inf)
        s["logits"] = x.to(dt)
        t[:, 1:].masked_fill_(torch.rand(t[:, 1:].shape, generator=g, device=device) < 0.2, -1)
        s["targets"] = t.to(torch.int32)
        return s
    nkv, page, batch = case["nkv"], case["page"], case["batch"]
    if case["op"] == "write":
        rows, nq = case["rows"], case["nq"]
        per = -(-rows // batch)
        blocks = -(-(case["ctx"] + per) // page)
        s["tables"], pages = _tables(batch, blocks, g, device)
        s["qkv"] = (torch.randn(rows, (nq + 2 * nkv) * D, generator=g, device=device) * 1.5).bfloat16()
        s["cos"], s["sin"] = _rope(device)
        r = torch.arange(rows, device=device)
        s["seqs"] = (r // per).to(torch.int32)
        s["slots"] = (case["ctx"] - s["seqs"] % 5 + r % per).to(torch.int32)  # unequal starts
        depth = torch.div(r % per, 2, rounding_mode="floor")  # siblings share a position
        s["positions"] = (case["ctx"] - s["seqs"] % 5 + depth).to(torch.int32)
        s["k"] = torch.zeros(pages, nkv, page, D, dtype=torch.float8_e4m3fn, device=device)
        s["v"] = torch.zeros_like(s["k"])
        s["ks"] = torch.zeros(pages, nkv, page, dtype=torch.uint8, device=device)
        s["vs"] = torch.zeros_like(s["ks"])
        s["q"] = torch.zeros(rows, nq, D, dtype=torch.bfloat16, device=device)
        return s
    prefixes = _prefixes(case)
    nodes = _nodes(case) if case["op"] == "attention" else [0] * batch
    blocks = -(-max(p + n for p, n in zip(prefixes, nodes)) // page)
    s["tables"], pages = _tables(batch, blocks, g, device)
    k, v = (_cached((pages, nkv, page, D), g, device) for _ in range(2))
    if case["op"] == "read" or case["cache"] == "e4m3":
        (s["k"], s["ks"]), (s["v"], s["vs"]) = _encode(k), _encode(v)
    else:
        s["k"], s["v"], s["ks"], s["vs"] = k.bfloat16(), v.bfloat16(), None, None
    s["prefix"] = torch.tensor(prefixes, dtype=torch.int32, device=device)
    if case["op"] == "read":
        return s
    total, T = sum(nodes), max(nodes)
    words = -(-T // 64)
    s["cu"] = torch.tensor([sum(nodes[:b]) for b in range(batch + 1)], dtype=torch.int32, device=device)
    if case["kind"] == "chain":
        index = torch.cat([torch.arange(n) for n in nodes])
        allowed = torch.arange(words * 64)[None, :] <= index[:, None]
    else:
        parents = torch.rand(total, generator=torch.Generator().manual_seed(seed)).tolist()
        allowed = torch.zeros(total, words * 64, dtype=torch.bool)
        at = 0
        for b, n in enumerate(nodes):
            for i in range(n):
                # a parent among the five nodes before it, now and then a second root
                p = i - 1 - int(parents[at] * 5)
                if p >= 0:
                    allowed[at] = allowed[at - i + p]
                allowed[at, i] = True
                at += 1
            if b % 4 == 3:
                allowed[at - 1] = False  # a padding node: nothing of the draft
    bit = torch.ones(64, dtype=torch.int64) << torch.arange(64)
    s["mask"] = (allowed.view(total, words, 64).long() * bit).sum(-1).to(device)
    s["q"] = (torch.randn(total, case["nq"], D, generator=g, device=device) * 1.2).bfloat16()
    s["T"], s["max_len"] = T, max(p + n for p, n in zip(prefixes, nodes))
    return s


# ------------------------------------------------------------------ the operators, plain


def _write_plain(s):
    case = s["case"]
    nq, nkv, page = case["nq"], case["nkv"], case["page"]
    x = s["qkv"].float().view(case["rows"], nq + 2 * nkv, D // 2, 2)
    x0, x1 = x[..., 0], x[..., 1]
    cos, sin = (t[s["positions"].long()].float()[:, None, :] for t in (s["cos"], s["sin"]))
    h = D // 2
    rot = torch.cat([x0 * cos[..., :h] - x1 * sin[..., :h], x1 * cos[..., h:] + x0 * sin[..., h:]], -1)
    s["q"].copy_(rot[:, :nq])
    seqs, slots = s["seqs"].long(), s["slots"].long()
    pages = s["tables"][seqs, torch.div(slots, page, rounding_mode="floor")].long()
    k, ks = _encode(rot[:, nq : nq + nkv])
    v, vs = _encode(torch.cat([x0, x1], -1)[:, nq + nkv :])
    s["k"].view(torch.uint8)[pages, :, slots % page] = k.view(torch.uint8)
    s["v"].view(torch.uint8)[pages, :, slots % page] = v.view(torch.uint8)
    s["ks"][pages, :, slots % page] = ks
    s["vs"][pages, :, slots % page] = vs
    return {"q": s["q"], "k": s["k"], "v": s["v"], "ks": s["ks"], "vs": s["vs"]}


def _gather(pool, scales, tables, length):
    """Positions [0, length) of every sequence, fp32 [batch, nkv, length, 64]."""
    blocks = -(-length // pool.shape[2])
    t = tables[:, :blocks].long()
    x = pool[t] if scales is not None else pool[t].float()
    x = _decode(x, scales[t]) if scales is not None else x
    b, _, nkv, page, d = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(b, nkv, blocks * page, d)[:, :, :length]


def _read_plain(s):
    n = s["case"]["ctx"]
    keep = (torch.arange(n, device=s["prefix"].device)[None, :] < s["prefix"][:, None])[:, None, :, None]
    zero = torch.zeros((), device=keep.device)
    return {x: torch.where(keep, _gather(s[x], s[x + "s"], s["tables"], n), zero).bfloat16() for x in ("k", "v")}


def _seen(s, batch, T, length):
    """Whether node i of sequence b sees position j: [batch, T, length]."""
    dev = s["q"].device
    n = (s["cu"][1:] - s["cu"][:-1]).long()
    i = torch.arange(T, device=dev)
    row = (s["cu"][:-1, None].long() + i).clamp(max=s["q"].shape[0] - 1)
    real = i[None, :] < n[:, None]
    j = torch.arange(length, device=dev)[None, :] - s["prefix"][:, None].long()  # draft index
    inside = (j >= 0) & (j < n[:, None])
    jj = j.clamp(0, T - 1)
    words = torch.gather(s["mask"][row], 2, torch.div(jj, 64, rounding_mode="floor")[:, None, :].expand(batch, T, length))
    bit = ((words >> (jj % 64)[:, None, :]) & 1).bool()
    return row, real, ((j < 0)[:, None, :] | (inside[:, None, :] & bit)) & real[:, :, None]


def _attention_plain(s):
    case, T, length = s["case"], s["T"], s["max_len"]
    batch, nq, nkv = case["batch"], case["nq"], case["nkv"]
    group = nq // nkv
    row, real, seen = _seen(s, batch, T, length)
    k, v = (_gather(s[x], s[x + "s"], s["tables"], length) for x in ("k", "v"))
    # what lies past a sequence's end is no value
    v = v * (torch.arange(length, device=v.device)[None, :] < (s["prefix"] + s["cu"][1:] - s["cu"][:-1])[:, None])[:, None, :, None]
    q = s["q"][row].float().view(batch, T, nkv, group, D).permute(0, 2, 1, 3, 4).reshape(batch, nkv, T * group, D)
    x = torch.matmul(q, k.transpose(-1, -2)).mul_(D**-0.5).view(batch, nkv, T, group, length)
    x.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p = x.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(batch, nkv, T * group, length), v).view(batch, nkv, T, group, D)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    lse = (m + total.log()).squeeze(-1)
    out = o.permute(0, 2, 1, 3, 4).reshape(batch, T, nq, D)[real]
    return {"out": out.bfloat16(), "lse": lse.permute(0, 2, 1, 3).reshape(batch, T, nq)[real]}


def _logprobs_plain(s):
    x, t = s["logits"].float(), s["targets"].long()
    m = x.amax(-1, keepdim=True)
    e = (x - m).exp()
    total = e.sum(-1, keepdim=True)
    lse = m + total.log()
    # 0 * -inf is 0 here: a forbidden token adds nothing
    mean = (e * torch.where(e > 0, x - m, torch.zeros_like(x))).sum(-1) / total[:, 0]
    lp = torch.where(t >= 0, torch.gather(x, 1, t.clamp(min=0)) - lse, torch.zeros_like(lse))
    top = s["case"]["top"]
    values, ids = torch.sort(x, dim=-1, descending=True, stable=True)
    return {"logprobs": lp, "entropy": total[:, 0].log() - mean, "top_ids": ids[:, :top].to(torch.int32), "top_logprobs": values[:, :top] - lse}


# ------------------------------------------------------------------ the operators, by the framework


def _run_own(s):
    from llama1b_megakernel_b200 import speculative as sp

    op, err = s["case"]["op"], s["error"]
    if op == "logprobs":
        lp, ent, ids, top = sp.token_logprobs(s["logits"], s["targets"], s["case"]["top"], error=err)
        return {"logprobs": lp, "entropy": ent, "top_ids": ids, "top_logprobs": top}
    layer = sp.KVLayer(s["k"], s["v"], s["tables"], s["ks"], s["vs"])
    if op == "write":
        sp.kv_write(layer, s["qkv"], s["cos"], s["sin"], s["seqs"], s["slots"], s["positions"], s["q"], error=err)
        return {"q": s["q"], "k": s["k"], "v": s["v"], "ks": s["ks"], "vs": s["vs"]}
    if op == "read":
        k, v = sp.kv_read(layer, s["prefix"], s["case"]["ctx"], error=err)
        return {"k": k, "v": v}
    out, lse = sp.tree_attention(s["q"], layer, s["cu"], s["mask"], s["prefix"], s["T"], s["max_len"], error=err)
    return {"out": out, "lse": lse}


def run(state):
    if own:
        return _run_own(state)
    return {"write": _write_plain, "read": _read_plain, "attention": _attention_plain, "logprobs": _logprobs_plain}[state["case"]["op"]](state)


# ------------------------------------------------------------------ the definition in 64 bits


def _power64(e):
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _value64(codes, scales):
    return codes.float().double() * _power64(scales.to(torch.int64) - 127)[..., None]


def _round64(x):
    """float64 rows -> what their e4m3 codes stand for before the row's scale is applied."""
    amax = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(amax / 448.0))
    e = torch.where(amax > 448.0 * _power64(e), e + 1, e)  # log2 may land beside an integer
    e = torch.where(amax <= 448.0 * _power64(e - 1), e - 1, e)
    y = x / _power64(e.clamp(min=-110.0))
    step = _power64(torch.floor(torch.log2(y.abs().clamp(min=2.0**-6))) - 3)
    return torch.round(y / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logprobs":
        out = {"logprobs": [], "entropy": [], "top_logprobs": []}
        for r in range(0, case["rows"], 64):
            x, t = s["logits"][r : r + 64].double(), s["targets"][r : r + 64].long()
            lse = torch.logsumexp(x, -1, keepdim=True)
            lp = x - lse
            out["logprobs"].append(torch.where(t < 0, 0.0, torch.gather(lp, 1, t.clamp(min=0))))
            out["entropy"].append(-torch.where(lp == -math.inf, 0.0, lp * lp.exp()).sum(-1))
            out["top_logprobs"].append(torch.topk(lp, case["top"], dim=-1).values)
        return {k: torch.cat(v) for k, v in out.items()} | {"top_ids": None}
    if case["op"] == "write":
        nq, nkv, page = case["nq"], case["nkv"], case["page"]
        head = s["qkv"].double().view(case["rows"], nq + 2 * nkv, D // 2, 2)
        pos = s["positions"].long()
        c, sn = s["cos"][pos].double(), s["sin"][pos].double()
        full = torch.cat([head[..., 0], head[..., 1]], -1)
        half = torch.cat([-head[..., 1], head[..., 0]], -1)
        rot = full * c[:, None] + half * sn[:, None]
        slots = s["slots"].long()
        pages = s["tables"].long()[s["seqs"].long(), slots // page]
        k, v = (torch.zeros(s["k"].shape, dtype=torch.float64, device="cuda") for _ in range(2))
        k[pages, :, slots % page] = _round64(rot[:, nq : nq + nkv])
        v[pages, :, slots % page] = _round64(full[:, nq + nkv :])
        return {"q": rot[:, :nq], "k": k, "v": v, "ks": None, "vs": None}
    nkv, page, batch = case["nkv"], case["page"], case["batch"]
    if case["op"] == "read":
        out = {}
        for name in ("k", "v"):
            full = torch.zeros(batch, nkv, case["ctx"], D, dtype=torch.float64, device="cuda")
            for b, n in enumerate(_prefixes(case)):
                p = torch.arange(n, device="cuda")
                pg = s["tables"][b].long()[p // page]
                full[b, :, :n] = _value64(s[name][pg, :, p % page], s[name + "s"][pg, :, p % page]).transpose(0, 1)
            out[name] = full
        return out
    group = case["nq"] // nkv
    outs, lses = [], []
    at = 0
    for b, (n, t) in enumerate(zip(_prefixes(case), _nodes(case))):
        p = torch.arange(n + t, device="cuda")
        pg = s["tables"][b].long()[p // page]
        kk, vv = (s[x][pg, :, p % page].float().double() if s[x + "s"] is None else _value64(s[x][pg, :, p % page], s[x + "s"][pg, :, p % page]) for x in ("k", "v"))
        bits = (s["mask"][at : at + t, :, None] >> torch.arange(64, device="cuda")) & 1
        draft = bits.reshape(t, -1)[:, :t].bool()
        seen = torch.cat([torch.ones(t, n, dtype=torch.bool, device="cuda"), draft], 1)
        o = torch.zeros(t, case["nq"], D, dtype=torch.float64, device="cuda")
        ls = torch.zeros(t, case["nq"], dtype=torch.float64, device="cuda")
        for h in range(case["nq"]):
            x = s["q"][at : at + t, h].double() @ kk[:, h // group].T * D**-0.5
            x = torch.where(seen, x, -math.inf)
            ls[:, h] = torch.logsumexp(x, -1)
            w = torch.where(seen.any(-1, keepdim=True), torch.softmax(x, -1), 0.0)
            o[:, h] = w @ vv[:, h // group]
        outs.append(o)
        lses.append(ls)
        at += t
    return {"out": torch.cat(outs), "lse": torch.cat(lses)}
