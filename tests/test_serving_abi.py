"""CPU checks of the packed attention, paged cache and log-probability entry
points: bad arguments come back as status codes, or as RuntimeError from the
Python functions, before any device is touched."""
import ctypes

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


def _packed(lib, n=1, T=10, Tk=10, H=4, Hkv=2, hd=64, scale=0.1, q=P, cu=P, strides=(256, 64, 128, 64, 128, 64, 256, 64), ws_bytes=1 << 40):
    fwd = lib.naylis_mom_packed_attn_fwd(q, P, P, cu, cu, P, P, P, _i64(*strides), scale, n, T, Tk, H, Hkv, hd, None)
    msg = lib.naylis_mom_last_error()
    bwd = lib.naylis_mom_packed_attn_bwd(q, P, P, cu, cu, P, P, P, P, P, P, P, P, ws_bytes, _i64(*strides), scale, n, T, Tk, H, Hkv,
                                         hd, None)
    assert fwd == bwd and msg.split(b":")[1] == lib.naylis_mom_last_error().split(b":")[1]
    return fwd


@pytest.mark.parametrize("bad,text", [
    (dict(n=0), "bad shape"), (dict(T=-1), "bad shape"), (dict(H=3), "bad shape"), (dict(Hkv=0), "bad shape"),
    (dict(hd=32), "head_dim"), (dict(hd=96), "head_dim"), (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(T=1 << 30), "too large"), (dict(n=1 << 20), "too large"), (dict(q=None), "null"), (dict(cu=None), "null"),
    (dict(q=ODD), "aligned"), (dict(strides=(260, 64, 128, 64, 128, 64, 256, 64)), "strides"),
    (dict(strides=(256, 64, 128, 64, -128, 64, 256, 64)), "strides"),
    (dict(strides=(1 << 23, 64, 128, 64, 128, 64, 256, 64)), "strides"),
    # rows of the output over 2^23 features; more tiles than a launch has workgroups
    (dict(H=1 << 18, Hkv=1 << 10), "too large"), (dict(T=1 << 29, H=4, Hkv=4), "too large")])
def test_packed_refusals(lib, bad, text):
    _refused(lib, _packed(lib, **bad), text)


def test_packed_workspace(lib):
    need = lib.naylis_mom_packed_attn_bwd_workspace_bytes(1, 10, 10, 4, 2, 64)
    args = (P, P, P, P, P, P, P, P, P, P, P, P, P, need - 1, _i64(256, 64, 128, 64, 128, 64, 256, 64), 0.1, 1, 10, 10, 4, 2, 64)
    assert lib.naylis_mom_packed_attn_bwd(*args, None) == _lib.NAYLIS_ERR_WORKSPACE
    # the group's heads in parts where few key tiles stand for many heads, not where they fill the chip
    few, many = (lib.naylis_mom_packed_attn_bwd_workspace_bytes(1, n, n, 8, 2, 128) for n in (1000, 1000000))
    assert few > 2 * 8 * 1000 * 4 + 2 * 2 * 1000 * 2 * 128 * 4 and many == 2 * 8 * 1000000 * 4
    assert lib.naylis_mom_packed_attn_bwd_workspace_bytes(1, 10, 10, 3, 2, 64) == 0


def test_packed_nothing_to_do(lib):
    assert _packed(lib, T=0, Tk=0) == _lib.NAYLIS_OK


def _append(lib, dtype=1, T=4, pages=8, Hkv=2, page=16, hd=64, B=4, W=3, scale=P, k=P, rows=None, table=P,
            strides=(128, 64, 128, 64)):
    return lib.naylis_mom_paged_append(P, P, scale, scale, dtype, k, P, _i64(*strides), table, P, rows, T, pages, Hkv,
                                       page, hd, B, W, None)


@pytest.mark.parametrize("bad,text", [
    (dict(dtype=0), "dtype"), (dict(dtype=2, scale=None), "scales"), (dict(page=8), "page_size"),
    (dict(page=48), "page_size"), (dict(page=512), "page_size"), (dict(hd=32), "head_dim"), (dict(pages=0), "bad shape"),
    (dict(Hkv=0), "bad shape"), (dict(W=0), "bad shape"), (dict(B=70000), "bad shape"), (dict(W=1 << 28), "bad shape"),
    (dict(T=5), "without rows"), (dict(T=-1), "token count"), (dict(k=None), "null"), (dict(table=None), "null"),
    (dict(k=ODD), "aligned"), (dict(strides=(4, 64, 128, 64)), "strides"),
    (dict(T=1 << 28, rows=P), "token count")])
def test_append_refusals(lib, bad, text):
    _refused(lib, _append(lib, **bad), text)


def test_append_nothing_to_do(lib):
    assert _append(lib, T=0) == _lib.NAYLIS_OK


def _attn(lib, dtype=1, B=2, H=4, pages=8, Hkv=2, page=16, hd=64, W=3, scale=0.1, ws_bytes=1 << 40, q=P, ws=P, lens=P):
    return lib.naylis_mom_paged_attn(q, P, P, P, P, dtype, P, lens, P, ws, ws_bytes, _i64(256, 64), scale, B, H, pages,
                                     Hkv, page, hd, W, None)


@pytest.mark.parametrize("bad,text", [
    (dict(H=5), "query heads"), (dict(Hkv=0), "query heads"), (dict(H=0), "query heads"), (dict(page=24), "page_size"),
    (dict(hd=256), "head_dim"), (dict(scale=-1.0), "scale"), (dict(dtype=7), "dtype"), (dict(q=None), "null"),
    (dict(W=100, ws=None), "null"), (dict(lens=None), "null"), (dict(q=ODD), "aligned"), (dict(B=1 << 20), "bad shape"),
    (dict(H=4096 * 257, Hkv=4096), "too many")])
def test_paged_attention_refusals(lib, bad, text):
    _refused(lib, _attn(lib, **bad), text)


def test_paged_attention_workspace(lib):
    need = lib.naylis_mom_paged_attn_workspace_bytes(1, 2, 4, 2, 16, 64, 100)
    assert need > 0 and lib.naylis_mom_paged_attn_workspace_bytes(1, 2, 4, 2, 16, 64, 3) == 0
    assert _attn(lib, W=100, ws_bytes=need - 1) == _lib.NAYLIS_ERR_WORKSPACE
    assert lib.naylis_mom_paged_attn_workspace_bytes(1, 2, 5, 2, 16, 64, 3) == 0
    assert "query heads" in lib.naylis_mom_last_error().decode()
    assert _attn(lib, B=0) == _lib.NAYLIS_OK


@pytest.mark.parametrize("which", [0, 1])
def test_scales_out_of_line_are_refused(lib, which):
    """The kernels read an e4m3 cache's scales four at a time."""
    for off in (4, 8, 12):
        s = [P, P]
        s[which] = ctypes.c_void_p(P.value + off)
        _refused(lib, lib.naylis_mom_paged_attn(P, P, P, *s, 2, P, P, P, P, 1 << 40, _i64(256, 64), 0.1, 2, 4, 8, 2, 16, 64, 3,
                                                None), "aligned")
        _refused(lib, lib.naylis_mom_paged_append(P, P, *s, 2, P, P, _i64(128, 64, 128, 64), P, P, None, 4, 8, 2, 16, 64, 4, 3,
                                                  None), "aligned")


@pytest.mark.parametrize("page", [16, 256])
def test_paged_tables_of_2_to_the_31_tokens(lib, page):
    """A table row may hold 2^31 - 2048 tokens and no more: behind a longer sequence's
    end the kernels' 32-bit token numbers would wrap, and their table reads with them."""
    last = (2 ** 31 - 2048) // page
    for W in (last + 1, last + 2, 2 ** 31 // page - 1, 2 ** 31 // page, 2 ** 60):
        assert lib.naylis_mom_paged_attn_workspace_bytes(1, 1, 4, 2, page, 64, W) == 0
        _refused(lib, _attn(lib, B=1, page=page, W=W), "bad shape")
        _refused(lib, _append(lib, T=1, B=1, page=page, W=W), "bad shape")
    assert lib.naylis_mom_paged_attn_workspace_bytes(1, 1, 4, 2, page, 64, last) > 0


def _logprobs(lib, dtype=1, ld=100, N=3, V=100, top=0, x=P, tok=P, ids=P, ws=P, ws_bytes=1 << 40):
    return lib.naylis_mom_logprobs_fwd(x, dtype, ld, tok, P, P, P, ids, ids, ws, ws_bytes, N, V, top, -100, None)


@pytest.mark.parametrize("bad,text", [
    (dict(dtype=2), "dtype"), (dict(N=-1), "bad shape"), (dict(N=1 << 24), "bad shape"), (dict(V=0), "bad shape"), (dict(ld=-1), "row stride"),
    (dict(top=-1), "top"), (dict(top=65), "top"), (dict(V=10, top=11), "top"), (dict(x=None), "null"),
    (dict(tok=None), "null"), (dict(top=1, ids=None), "null"), (dict(x=ctypes.c_void_p(4097)), "aligned"),
    (dict(dtype=0, x=ODD), "aligned"), (dict(V=70000, ld=70000, ws=None), "workspace"), (dict(V=70000, ws=ODD), "workspace")])
def test_logprobs_refusals(lib, bad, text):
    _refused(lib, _logprobs(lib, **bad), text)


def test_logprobs_workspace(lib):
    need = lib.naylis_mom_logprobs_workspace_bytes(3, 70000, 20)
    assert need > 0 and lib.naylis_mom_logprobs_workspace_bytes(3, 1000, 20) == 0
    assert lib.naylis_mom_logprobs_workspace_bytes(4096, 70000, 20) == 0
    assert _logprobs(lib, V=70000, top=20, ws_bytes=need - 1) == _lib.NAYLIS_ERR_WORKSPACE


def test_logprobs_backward_refusals(lib):
    def call(dtype=1, stat=P, dx=P, stride=1, N=3):
        return lib.naylis_mom_logprobs_bwd(P, dtype, 100, P, stat, P, stride, P, 1, dx, N, 100, -100, None)
    _refused(lib, call(dtype=5), "dtype")
    _refused(lib, call(stat=None), "null")
    _refused(lib, call(dx=None), "null")
    _refused(lib, call(dx=ctypes.c_void_p(4097)), "aligned")
    _refused(lib, call(stride=-1), "strides")
    assert call(N=0) == _lib.NAYLIS_OK and _logprobs(lib, N=0) == _lib.NAYLIS_OK


def test_cpu_tensors_are_refused():
    from naylis_amd import mom_kernels as mk
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    cache = mk.new_paged_cache(2, 2, 16, 64, "cpu")
    table = torch.zeros(4, 1, dtype=torch.int32)
    for call in (lambda: mk.packed_attention(x, x, x, cu), lambda: mk.paged_append(cache, x, x, table, table[:, 0]),
                 lambda: mk.paged_attention(x, cache, table, table[:, 0]),
                 lambda: mk.token_logprobs(torch.zeros(2, 9), torch.zeros(2, dtype=torch.long))):
        with pytest.raises(RuntimeError, match="ROCm device"):
            call()


def test_dequantize():
    from naylis_amd.mom_kernels import new_paged_cache
    c = new_paged_cache(2, 1, 16, 64, "cpu", fp8=True)
    c.k[0, 0, 3] = torch.tensor(2.5).to(torch.float8_e4m3fn).view(torch.uint8)
    c.k_scale[0, 0, 3] = 0.5
    k, v = c.dequantize()
    assert float(k[0, 0, 3, 5]) == 1.25 and float(v.abs().sum()) == 0
