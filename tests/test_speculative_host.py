"""The speculative-decoding entry points refuse bad arguments before they touch CUDA."""
import ctypes

import pytest

from llama1b_megakernel_b200 import _lib


@pytest.fixture(scope="module")
def lib():
    from llama1b_megakernel_b200 import build

    build.build()
    return _lib.load()


PTR = 1 << 20  # an aligned address that nothing reads


def _layer(**kw):
    base = dict(k_pages=PTR, v_pages=PTR, k_scales=PTR, v_scales=PTR, block_tables=PTR, format=_lib.MK_KV_E4M3,
                num_pages=10, page_size=16, num_kv_heads=2, max_blocks=5)
    base.update(kw)
    return _lib.MkKVLayer(**base)


BAD_LAYERS = [dict(k_pages=None), dict(v_pages=None), dict(block_tables=None), dict(k_scales=None),
              dict(v_scales=None), dict(format=2), dict(num_pages=0), dict(page_size=12), dict(page_size=0),
              dict(num_kv_heads=0), dict(max_blocks=0), dict(k_pages=PTR + 8), dict(max_blocks=1 << 30)]


def _write(lib, layer, batch=2, qkv=PTR, rope_len=64, rows=3, nq=8, q_out=PTR, error=PTR, slots=PTR):
    return lib.mk_kv_write(ctypes.byref(layer), batch, qkv, PTR, PTR, rope_len, PTR, slots, PTR, rows, nq, q_out,
                           error, None)


def _read(lib, layer, lengths=PTR, batch=2, max_len=80, k=PTR, v=PTR, error=PTR):
    return lib.mk_kv_read(ctypes.byref(layer), lengths, batch, max_len, k, v, error, None)


def _attend(lib, layer, q=PTR, cu=PTR, mask=PTR, prefix=PTR, batch=2, rows=6, max_nodes=3, max_len=80, nq=8,
            ws=PTR, ws_bytes=1 << 40, out=PTR, error=PTR):
    return lib.mk_tree_attention(q, ctypes.byref(layer), cu, mask, prefix, batch, rows, max_nodes, max_len, nq,
                                 ctypes.c_float(0.125), ws, ws_bytes, out, None, error, None)


def _logprobs(lib, logits=PTR, dtype=_lib.MK_F32, rows=2, vocab=100, ld=100, targets=PTR, n=1, top=4, lp=PTR, ent=PTR,
              ids=PTR, tlp=PTR, error=PTR, ws=PTR, ws_bytes=1 << 40):
    return lib.mk_token_logprobs(logits, dtype, rows, vocab, ld, targets, n, top, ws, ws_bytes, lp, ent, ids, tlp,
                                 error, None)


@pytest.mark.parametrize("bad", BAD_LAYERS)
def test_bad_layers(lib, bad):
    layer = _layer(**bad)
    for call in (_write, _read, _attend):
        assert call(lib, layer) == _lib.MK_EINVAL
        assert lib.mk_last_error().decode()


@pytest.mark.parametrize("bad", [dict(batch=0), dict(qkv=None), dict(rope_len=0), dict(rows=-1), dict(nq=0),
                                 dict(q_out=None), dict(error=None), dict(slots=None), dict(qkv=PTR + 2)])
def test_write_refusals(lib, bad):
    assert _write(lib, _layer(), **bad) == _lib.MK_EINVAL


@pytest.mark.parametrize("bad", [dict(batch=0), dict(batch=70000), dict(lengths=None), dict(max_len=81),
                                 dict(max_len=-1), dict(k=None), dict(v=PTR + 4), dict(error=None)])
def test_read_refusals(lib, bad):
    assert _read(lib, _layer(), **bad) == _lib.MK_EINVAL


@pytest.mark.parametrize("bad", [dict(q=None), dict(cu=None), dict(mask=None), dict(prefix=None), dict(batch=0),
                                 dict(rows=-1), dict(max_nodes=0), dict(max_nodes=257), dict(max_len=0),
                                 dict(max_len=81), dict(nq=0), dict(nq=7), dict(nq=6), dict(nq=32), dict(out=None),
                                 dict(error=None), dict(q=PTR + 8), dict(out=PTR + 2)])
def test_attention_refusals(lib, bad):
    assert _attend(lib, _layer(), **bad) == _lib.MK_EINVAL


@pytest.mark.parametrize("bad", [dict(logits=None), dict(dtype=2), dict(rows=-1), dict(vocab=0), dict(ld=99),
                                 dict(targets=None), dict(n=-1), dict(top=33), dict(top=-1), dict(lp=None),
                                 dict(ent=None), dict(ids=None), dict(tlp=None), dict(error=None),
                                 dict(vocab=3, ld=3, top=4)])
def test_logprobs_refusals(lib, bad):
    assert _logprobs(lib, **bad) == _lib.MK_EINVAL


def test_calls_without_rows_do_nothing(lib):
    assert _write(lib, _layer(), rows=0) == _lib.MK_OK
    assert _read(lib, _layer(), max_len=0) == _lib.MK_OK
    assert _attend(lib, _layer(), rows=0) == _lib.MK_OK
    assert _logprobs(lib, rows=0) == _lib.MK_OK


def test_workspaces_cover_the_call(lib):
    for args in ((1, 32, 8, 1, 8192), (64, 32, 8, 1, 4096), (4, 8, 2, 256, 16384), (3, 4, 4, 7, 33)):
        need = lib.mk_tree_attention_workspace(*args)
        assert need >= 0
        if need:
            layer = _layer(num_kv_heads=args[2], max_blocks=1100)
            rc = _attend(lib, layer, batch=args[0], nq=args[1], max_nodes=args[3], max_len=args[4], ws_bytes=need - 1)
            assert rc == _lib.MK_EINVAL and "workspace" in lib.mk_last_error().decode()
    for args in ((1, 128256, 20), (64, 5003, 0), (2000, 128256, 32)):
        need = lib.mk_token_logprobs_workspace(*args)
        assert need >= 0
        if need:
            assert _logprobs(lib, rows=args[0], vocab=args[1], ld=args[1], top=args[2],
                             ws_bytes=need - 1) == _lib.MK_EINVAL


# ------------------------------------------------------------------ host-side parts
def test_draft_tree():
    from llama1b_megakernel_b200.speculative import DraftTree, lookup_draft, mask_words

    t = DraftTree([5, 6, 7, 8], [-1, 0, 0, 2])
    assert t.depths() == [0, 1, 1, 2]
    assert t.masks() == [1, 0b11, 0b101, 0b1101]
    assert t.children() == [[1, 2], [], [3], [], [0]]
    assert DraftTree.chain([4, 4, 4]).parents == [-1, 0, 1] and len(DraftTree.chain([])) == 0
    for tokens, parents in (([1], [0]), ([1, 2], [-1, 1]), ([1, 2], [-1]), ([1], [-2])):
        with pytest.raises(ValueError):
            DraftTree(tokens, parents)
    w = mask_words([1 << 63, 1 << 64 | 1], 70)
    assert w.tolist() == [[-(1 << 63), 0], [1, 1]]
    assert lookup_draft([1, 2, 3, 9, 1, 2, 3]).tokens == [9, 1, 2, 3]
    assert lookup_draft([1, 2, 3]) is None


def test_quantised_cache_rows():
    """What the 8-bit cache holds of rows: half a code step from them, exact on the way back."""
    import torch

    from llama1b_megakernel_b200.config import TINY
    from llama1b_megakernel_b200.kv_cache import QuantizedPagedKVCache, decode_rows, encode_rows

    g = torch.Generator().manual_seed(0)
    x = torch.randn(50, 64, generator=g) * torch.exp(3 * torch.randn(50, 1, generator=g))
    x[0] = 0
    x[1, 3] = float("nan")
    x[2, 5] = float("inf")
    x[3] = 448.0
    codes, byte = encode_rows(x)
    y = decode_rows(codes, byte).double()
    assert (byte[1:3] == 255).all() and y[1:3].isnan().all() and not y[0].any() and (y[3] == 448).all()
    amax = x[3:].abs().amax(1).double()
    scale = 2.0 ** (byte[3:].double() - 127)
    assert (amax <= 448 * scale).all() and (amax > 224 * scale).all()
    step = torch.maximum(2.0 ** torch.floor(torch.log2(x[3:].abs().double() / scale[:, None])), torch.tensor(2.0 ** -6)) / 8
    assert ((y[3:] - x[3:].double()).abs() <= step * scale[:, None] / 2).all()
    kv = QuantizedPagedKVCache(TINY, max_batch=2, max_seq_len=64, page_size=8, device="cpu")
    kv.shuffle_free_pages(1)
    rows = torch.randn(TINY.num_layers, TINY.num_kv_heads, 21, 64, generator=g)
    kv.fill(1, rows, 2 * rows)
    k, v = kv.gather(1, 21)
    assert torch.equal(k, decode_rows(*encode_rows(rows))) and torch.equal(v, decode_rows(*encode_rows(2 * rows)))
    assert kv.nbytes() == 2 * TINY.num_layers * kv.num_pages * TINY.num_kv_heads * 8 * 65
