"""Argument checks of the norm and 8-bit entry points that need no GPU: error codes, no launch."""
import pytest
import torch

FAKE = 0x10000            # never read: every call below is refused before a launch


@pytest.fixture(scope="module")
def lib():
    from ccfuser_amd import _lib
    if not _lib.LIB_PATH.exists():
        from ccfuser_amd import build
        build.build(verbose=False)
    return _lib.lib()


def _norm(lib, x=FAKE, residual=None, weight=FAKE, rows=2, d=64, eps=1e-5, dtype=0, wtype=0, y=FAKE, total=None, codes=None,
          scales=None, rstd=None):
    return lib.ccf_rms_norm(x, residual, weight, rows, d, eps, dtype, wtype, y, total, codes, scales, rstd, None)


@pytest.mark.parametrize("bad,code", [
    (dict(rows=-1), 1), (dict(d=0), 1), (dict(d=(1 << 24) + 1), 1), (dict(x=None), 1), (dict(weight=None), 1),
    (dict(y=None), 1), (dict(codes=FAKE), 1), (dict(scales=FAKE), 1), (dict(residual=FAKE), 1), (dict(total=FAKE), 1),
    (dict(eps=-1.0), 1), (dict(eps=float("nan")), 1), (dict(x=FAKE + 1), 1), (dict(dtype=1, wtype=1, weight=FAKE + 2), 1),
    (dict(dtype=0, wtype=2), 5), (dict(dtype=1, wtype=0), 5), (dict(dtype=7, wtype=7), 5)])
def test_norm_refuses(lib, bad, code):
    assert _norm(lib, **bad) == code
    assert lib.ccf_last_error()


@pytest.mark.parametrize("bad,code", [
    (dict(rows=-1), 1), (dict(d=0), 1), (dict(gx=None, gw=None), 1), (dict(gy=None), 1), (dict(rstd=None), 1), (dict(ws=None), 3),
    (dict(nbytes=0), 3), (dict(dtype=0, wtype=2), 5), (dict(gy=FAKE + 1), 1)])
def test_norm_backward_refuses(lib, bad, code):
    a = dict(gy=FAKE, total=FAKE, w=FAKE, rstd=FAKE, gt=None, rows=2, d=64, dtype=0, wtype=0, gx=FAKE, gw=FAKE, ws=FAKE, nbytes=1 << 20)
    a.update(bad)
    assert lib.ccf_rms_norm_backward(a["gy"], a["total"], a["w"], a["rstd"], a["gt"], a["rows"], a["d"], a["dtype"], a["wtype"],
                                     a["gx"], a["gw"], a["ws"], a["nbytes"], None) == code


def test_quantize_refuses(lib):
    assert lib.ccf_quantize_rows(FAKE, -1, 64, 0, FAKE, FAKE, None) == 1
    assert lib.ccf_quantize_rows(FAKE, 1, 0, 0, FAKE, FAKE, None) == 1
    assert lib.ccf_quantize_rows(None, 1, 64, 0, FAKE, FAKE, None) == 1
    assert lib.ccf_quantize_rows(FAKE + 1, 1, 64, 0, FAKE, FAKE, None) == 1
    assert lib.ccf_quantize_rows(FAKE, 1, 64, 9, FAKE, FAKE, None) == 5
    assert lib.ccf_quantize_weight(FAKE, 1, 0, 64, 0, FAKE, FAKE, None) == 1
    assert lib.ccf_quantize_weight(FAKE, 1, 64, 64, 0, None, FAKE, None) == 1
    assert lib.ccf_quantize_weight(FAKE, 1 << 24, 1 << 14, 1 << 14, 0, FAKE, FAKE, None) == 2


def test_no_cpu_path():
    from ccfuser_amd import ops
    from ccfuser_amd.mix_moe import RMSNorm
    x, w = torch.ones(2, 64), torch.ones(64)
    for call in (lambda: ops.rms_norm(x, w), lambda: ops.quantize_rows(x), lambda: ops.quantize_weight(x), lambda: RMSNorm(64)(x)):
        with pytest.raises(ValueError, match="GPU"):
            call()


def _linear(lib, x=FAKE, xs=FAKE, rows=2, k=64, w=FAKE, ws=FAKE, n=64, bias=None, dtype=0, y=FAKE):
    return lib.ccf_linear_fp8(x, xs, rows, k, w, ws, n, bias, dtype, y, None)


@pytest.mark.parametrize("bad,code", [
    (dict(rows=-1), 1), (dict(k=0), 1), (dict(n=0), 1), (dict(k=24), 2), (dict(n=12), 2), (dict(x=None), 1), (dict(xs=None), 1),
    (dict(w=None), 1), (dict(ws=None), 1), (dict(y=None), 1), (dict(x=FAKE + 1), 1), (dict(w=FAKE + 8), 1), (dict(y=FAKE + 2), 1),
    (dict(bias=FAKE + 2), 1), (dict(dtype=1), 5), (dict(dtype=9), 5), (dict(rows=1 << 30), 2), (dict(rows=1 << 24, k=1 << 16), 2),
    (dict(k=1 << 17, n=1 << 15), 2)])
def test_linear_refuses(lib, bad, code):
    assert _linear(lib, **bad) == code
    assert lib.ccf_last_error()


def test_no_rows_are_no_call(lib):
    assert _linear(lib, rows=0, x=None, xs=None, y=None) == 0


@pytest.mark.parametrize("bad,code", [
    (dict(rows=-1), 1), (dict(E=0), 1), (dict(E=1025), 2), (dict(d=24), 2), (dict(f=12), 2), (dict(x=None), 1), (dict(off=None), 1),
    (dict(w=None), 1), (dict(out=None), 1), (dict(b=FAKE + 2), 1)])
def test_grouped_products_refuse(lib, bad, code):
    a = dict(x=FAKE, xs=FAKE, src=None, off=FAKE, rows=4, E=2, d=64, f=64, w=FAKE, ws=FAKE, b=None, out=FAKE, out_s=FAKE)
    a.update(bad)
    assert lib.ccf_ffn1_fp8(a["x"], a["xs"], a["src"], a["off"], a["rows"], a["E"], a["d"], a["f"], a["w"], a["ws"], a["b"], a["out"],
                            a["out_s"], None) == code
    if "d" in bad or "f" in bad:                       # the other product contracts the other width
        a["d"], a["f"] = a["f"], a["d"]
    assert lib.ccf_ffn2_fp8(a["x"], a["xs"], a["src"], a["off"], a["rows"], a["E"], a["d"], a["f"], a["w"], a["ws"], a["b"], a["out"],
                            None) == code


LAYER = dict(T=4, d=64, f=64, E=4, k=2)


def _layer(lib, **bad):
    a = dict(x=FAKE, xc=None, xs=None, wg=FAKE, bg=None, w1=FAKE, s1=FAKE, b1=None, w2=FAKE, s2=FAKE, b2=None, cap=-1, out=FAKE, ws=FAKE,
             nbytes=1 << 30, **LAYER)
    a.update(bad)
    return lib.ccf_moe_forward_fp8(a["x"], a["xc"], a["xs"], a["wg"], a["bg"], a["w1"], a["s1"], a["b1"], a["w2"], a["s2"], a["b2"], a["T"],
                                   a["d"], a["f"], a["E"], a["k"], a["cap"], a["out"], None, None, a["ws"], a["nbytes"], None)


def _few(lib, **bad):
    a = dict(x=FAKE, wg=FAKE, bg=None, w1=FAKE, b1=FAKE, w2=FAKE, b2=FAKE, out=FAKE, ws=FAKE, nbytes=1 << 30, **LAYER)
    a.update(bad)
    return lib.ccf_moe_forward_few(a["x"], a["wg"], a["bg"], a["w1"], a["b1"], a["w2"], a["b2"], a["T"], a["d"], a["f"], a["E"], a["k"],
                                   a["out"], None, None, a["ws"], a["nbytes"], None)


@pytest.mark.parametrize("bad", [dict(T=-1), dict(d=72), dict(f=72), dict(E=0), dict(E=1025), dict(k=0), dict(k=5), dict(k=9, E=16),
                                 dict(x=None), dict(wg=None), dict(w1=None), dict(w2=None), dict(out=None), dict(ws=None), dict(nbytes=8),
                                 dict(x=FAKE + 2), dict(w1=FAKE + 8)], ids=str)
def test_layers_refuse(lib, bad):
    assert _layer(lib, **bad) not in (0, 4)
    assert _few(lib, **bad) not in (0, 4)
    assert lib.ccf_last_error()


def test_layers_refuse_what_is_their_own(lib):
    assert _few(lib, T=17) == 2
    assert _layer(lib, T=1 << 29, nbytes=1 << 62) == 2 and _layer(lib, T=1 << 24, f=1 << 16, nbytes=1 << 62) == 2
    assert _layer(lib, d=1 << 17, f=1 << 15, nbytes=1 << 62) == 2
    assert _layer(lib, s1=None) == 1 and _layer(lib, s2=None) == 1 and _layer(lib, xc=FAKE) == 1
    for f in (lib.ccf_moe_few_workspace_bytes, lib.ccf_moe_fp8_workspace_bytes):
        assert f(4, 64, 64, 4, 2) > 0


@pytest.mark.parametrize("bad,code", [
    (dict(rows=-1), 1), (dict(k=24), 2), (dict(n=12), 2), (dict(x=None), 1), (dict(x=FAKE + 1), 1), (dict(ws=None), 3), (dict(nbytes=64), 3),
    (dict(ws=FAKE + 4), 1), (dict(xt=9), 5), (dict(dtype=1), 5), (dict(w=None), 1), (dict(s=None), 1), (dict(y=None), 1)])
def test_linear_of_16_bit_rows_refuses(lib, bad, code):
    a = dict(x=FAKE, xt=0, rows=2, k=64, w=FAKE, s=FAKE, n=64, dtype=0, y=FAKE, ws=FAKE, nbytes=1 << 20)
    a.update(bad)
    assert lib.ccf_linear_fp8_rows(a["x"], a["xt"], a["rows"], a["k"], a["w"], a["s"], a["n"], None, a["dtype"], a["y"], a["ws"],
                                   a["nbytes"], None) == code
