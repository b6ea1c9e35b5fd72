"""CPU checks of the rotated append, the gather, the attention of several tokens,
4-bit pages and the drafts' verification: bad arguments come back as status
codes, or as RuntimeError from the Python functions, before any device is touched."""
import ctypes
import math

import pytest
import torch

from naylis_amd import _lib


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


P = ctypes.c_void_p(1 << 20)  # aligned, never read
ODD = ctypes.c_void_p((1 << 20) + 2)


def _i64(*v):
    return (ctypes.c_int64 * len(v))(*v)


def _refused(lib, rc, text):
    assert rc == _lib.NAYLIS_ERR_ARG
    assert text in lib.naylis_mom_last_error().decode(), lib.naylis_mom_last_error()


def _rope(lib, dtype=1, q=P, k=P, strides=(256, 64, 128, 64, 128, 64), freq=P, scaling=1.0, table=P, pos=P, rows=None, out=P, T=4, H=4,
          half=32, pages=8, Hkv=2, page=16, hd=64, B=4, W=3, scale=P):
    return lib.naylis_mom_paged_append_rope(P, P, scale, scale, dtype, q, k, P, _i64(*strides), freq, scaling, table, pos, rows, out, T,
                                            H, half, pages, Hkv, page, hd, B, W, None)


@pytest.mark.parametrize("bad,text", [
    (dict(dtype=0), "dtype"), (dict(dtype=4), "dtype"), (dict(dtype=2, scale=None), "e4m3"), (dict(dtype=3, scale=None), "e2m1"),
    (dict(dtype=3, scale=ODD), "aligned"), (dict(page=8), "page_size"), (dict(hd=32), "head_dim"), (dict(pages=0), "bad shape"),
    (dict(T=5), "without rows"), (dict(T=-1), "token count"), (dict(T=1 << 24, rows=P), "token count"), (dict(H=-1), "bad shape"),
    (dict(H=1 << 20), "bad shape"), (dict(half=0), "frequencies"), (dict(half=12), "frequencies"), (dict(half=40), "frequencies"),
    (dict(scaling=math.inf), "scaling"), (dict(scaling=math.nan), "scaling"), (dict(freq=None), "null"), (dict(table=None), "null"),
    (dict(pos=None), "null"), (dict(k=None), "null"), (dict(k=ODD), "aligned"), (dict(q=ODD), "aligned"), (dict(out=None), "null"),
    (dict(strides=(4, 64, 128, 64, 128, 64)), "strides"), (dict(strides=(256, 64, 128, 4, 128, 64)), "strides"),
    (dict(strides=(256, 64, 128, 64, 1 << 23, 64)), "strides")])
def test_append_rope_refusals(lib, bad, text):
    _refused(lib, _rope(lib, **bad), text)


def test_append_rope_nothing_to_do(lib):
    assert _rope(lib, T=0) == _lib.NAYLIS_OK


def _gather(lib, dtype=1, pages=8, Hkv=2, page=16, hd=64, B=4, W=3, T=9, table=P, cu=P, out=P, scale=P):
    return lib.naylis_mom_paged_gather(P, P, scale, scale, dtype, table, cu, out, P, T, pages, Hkv, page, hd, B, W, None)


@pytest.mark.parametrize("bad,text", [
    (dict(dtype=9), "dtype"), (dict(dtype=3, scale=None), "e2m1"), (dict(page=24), "page_size"), (dict(hd=96), "head_dim"),
    (dict(B=0), "bad shape"), (dict(B=1 << 17), "bad shape"), (dict(T=-1), "token count"), (dict(T=(1 << 28) - 15), "token count"),
    (dict(table=None), "null"), (dict(cu=None), "null"), (dict(out=None), "null"), (dict(out=ODD), "aligned")])
def test_gather_refusals(lib, bad, text):
    _refused(lib, _gather(lib, **bad), text)


def test_gather_nothing_to_do(lib):
    assert _gather(lib, T=0) == _lib.NAYLIS_OK


def _tokens(lib, dtype=3, B=2, N=3, H=4, pages=8, Hkv=2, page=16, hd=64, W=3, scale=0.1, ws_bytes=1 << 40, q=P, ws=P, lens=P, s=P,
            strides=(768, 256, 64)):
    return lib.naylis_mom_paged_attn_tokens(q, P, P, s, s, dtype, P, lens, P, P, ws, ws_bytes, _i64(*strides), scale, B, N, H, pages, Hkv,
                                            page, hd, W, None)


@pytest.mark.parametrize("bad,text", [
    (dict(N=0), "too many"), (dict(N=2049), "too many"), (dict(N=1 << 40), "too many"), (dict(H=5), "query heads"),
    (dict(H=4096, Hkv=4096, N=4096), "too many"), (dict(dtype=4), "dtype"), (dict(s=None), "e2m1"), (dict(s=ODD), "aligned"),
    (dict(q=None), "null"), (dict(q=ODD), "aligned"), (dict(lens=None), "null"), (dict(W=100, ws=None), "null"),
    (dict(strides=(768, 4, 64)), "strides"), (dict(strides=(768, 1 << 23, 64)), "strides"), (dict(strides=(-8, 256, 64)), "strides"),
    (dict(scale=math.nan), "scale"), (dict(B=1 << 17), "bad shape")])
def test_attention_of_tokens_refusals(lib, bad, text):
    _refused(lib, _tokens(lib, **bad), text)


def test_attention_of_tokens_workspace(lib):
    need = lambda n, dtype=3, W=100: lib.naylis_mom_paged_attn_tokens_workspace_bytes(dtype, 2, n, 4, 2, 16, 64, W)  # noqa: E731
    assert need(1) > 0 and need(9) > need(1) and need(3, W=3) == 0 and need(0) == 0 and need(1, dtype=5) == 0
    assert need(1, dtype=1) == lib.naylis_mom_paged_attn_workspace_bytes(1, 2, 4, 2, 16, 64, 100)
    assert _tokens(lib, W=100, ws_bytes=need(3) - 1) == _lib.NAYLIS_ERR_WORKSPACE
    assert _tokens(lib, B=0) == _lib.NAYLIS_OK


def test_attention_of_tokens_batch_strides(lib):
    """From sequence to sequence q may step as far as memory goes."""
    for far in (1 << 23, (1 << 40) - 8):
        assert _tokens(lib, W=100, ws_bytes=0, strides=(far, 256, 64)) == _lib.NAYLIS_ERR_WORKSPACE
    for bad in (1 << 40, (1 << 23) + 4):
        _refused(lib, _tokens(lib, W=100, ws_bytes=0, strides=(bad, 256, 64)), "strides")


def _verify(lib, dtype=1, strides=(300, 100), logits=P, drafts=P, uniforms=P, probs=P, probs_dtype=0, probs_strides=(200, 100), temps=P,
            temperature=1.0, tokens=P, ws=P, ws_bytes=1 << 40, B=3, N=2, V=100):
    return lib.naylis_mom_verify_drafts(logits, dtype, strides and _i64(*strides), drafts, uniforms, probs, probs_dtype,
                                        probs_strides and _i64(*probs_strides), P, temps, temperature, tokens, P, ws, ws_bytes, B, N, V,
                                        None)


@pytest.mark.parametrize("bad,text", [
    (dict(dtype=2), "dtype"), (dict(probs_dtype=3), "dtype"), (dict(B=-1), "bad shape"), (dict(B=1 << 16), "bad shape"),
    (dict(N=-1), "bad shape"), (dict(N=1024), "bad shape"), (dict(V=0), "bad shape"), (dict(V=(1 << 28) + 1), "bad shape"),
    (dict(logits=None), "null"), (dict(strides=None), "null"), (dict(drafts=None), "null"), (dict(uniforms=None), "null"),
    (dict(probs_strides=None), "null"), (dict(tokens=None), "null"), (dict(V=100000, ws=None), "null"), (dict(V=100000, ws=ODD), "aligned"),
    (dict(strides=(-1, 100)), "strides"), (dict(probs_strides=(200, 1 << 40)), "strides"), (dict(logits=ctypes.c_void_p(4097)), "aligned"),
    (dict(probs=ODD), "aligned"), (dict(temps=None, temperature=-0.5), "temperature"),
    (dict(temps=None, temperature=math.nan), "temperature"), (dict(temps=None, temperature=math.inf), "temperature")])
def test_verify_refusals(lib, bad, text):
    _refused(lib, _verify(lib, **bad), text)


def test_verify_workspace(lib):
    need = lambda B, N, V, q: lib.naylis_mom_verify_drafts_workspace_bytes(B, N, V, q)  # noqa: E731
    assert need(3, 2, 100000, 1) > need(3, 2, 100000, 0) > 0 and need(3, 2, 0, 0) == 0
    assert need(3, 2, 500, 1) == need(0, 0, 1, 0) == 0  # one launch
    assert _verify(lib, V=100000, ws_bytes=need(3, 2, 100000, 1) - 1) == _lib.NAYLIS_ERR_WORKSPACE
    assert _verify(lib, B=0) == _lib.NAYLIS_OK


def test_cpu_tensors_are_refused():
    from naylis_amd import mom_kernels as mk
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    table = torch.zeros(4, 1, dtype=torch.int32)
    for fp4 in (False, True):
        cache = mk.new_paged_cache(2, 2, 16, 64, "cpu", fp4=fp4)
        for call in (lambda: mk.paged_append_rope(cache, x, x, x, torch.ones(32), table, table[:, 0]),
                     lambda: mk.paged_gather(cache, table, torch.arange(5, dtype=torch.int32), 4),
                     lambda: mk.paged_attention(x[:, None], cache, table, table[:, 0]),
                     lambda: mk.verify_drafts(torch.zeros(2, 2, 9), torch.zeros(2, 1, dtype=torch.long), torch.zeros(2, 2))):
            with pytest.raises(RuntimeError, match="ROCm device"):
                call()


def test_dequantize_of_4_bits():
    from naylis_amd.mom_kernels import new_paged_cache
    c = new_paged_cache(2, 1, 16, 64, "cpu", fp4=True)
    c.k[0, 0, 3] = 0x7a  # -1 and 6
    c.k_scale[0, 0, 3] = torch.tensor([128, 255], dtype=torch.uint8)
    k, v = c.dequantize()
    assert k.shape == (2, 1, 16, 64) and k[0, 0, 3, :4].tolist() == [-2.0, 12.0, -2.0, 12.0]
    assert bool(k[0, 0, 3, 32:].isnan().all()) and float(k[0, 0, :3].abs().sum()) == 0 and float(v.abs().sum()) == 0
