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
