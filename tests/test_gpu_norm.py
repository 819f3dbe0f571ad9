"""The root-mean-square norm, its 8-bit output and its backward, and rows and weights in 8 bits, against float64.

Tolerances: a result rounded to type t is off by eps(t) / 2 of its value (and half the smallest subnormal); before that the
fp32 arithmetic is off by a few u = 2^-24 of the magnitudes that go into it.  A row's sum of squares has positive terms, at
most 8 * 2 * 3 of them one after the other in a thread (rows up to 49152) and then ten levels of a tree: under 64 u, which
the square root halves; four more roundings follow."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
SIZES = [(1, 1), (3, 7), (1, 128), (5, 129), (2, 511), (4, 512), (7, 1000), (3, 1023), (1, 4096), (6, 2047), (3, 4097), (2, 8191),
         (2, 16384), (2, 16385), (1, 20001), (1999, 768), (257, 4096)]


def _rows(seed, *shape, dtype=torch.float16, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(dtype).cuda()


def _half_step(ref, dtype):
    """Half a step of the type around ref: relative, or of the smallest subnormal."""
    f = torch.finfo(dtype)
    return ref.abs() * (f.eps / 2) + f.tiny * f.eps / 2


def _norm64(x, w, eps, residual=None):
    total = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    t = total.double()
    rstd = (t.square().mean(-1, keepdim=True) + eps).rsqrt()
    return total, t * rstd * w.double(), rstd


def codes_of(t):
    """e4m3 codes and power-of-two scales of rows [R, K], in float64 on the CPU: what a block's scale and codes are by
    definition, elements that are no numbers aside."""
    t = t.double().cpu()
    R, K = t.shape
    nb = -(-K // 128)
    full = torch.zeros(R, nb * 128, dtype=torch.float64)
    full[:, :K] = t
    full = full.view(R, nb, 128)
    top = full.abs().amax(-1)
    power = torch.ceil(torch.log2(top / 448.0).clamp_min(-126.0))
    for step in (-1.0, 1.0):                                     # log2 may be an ulp off next to a power of two
        trial = power + step
        fits = top <= 448.0 * torch.exp2(trial)
        power = torch.where(fits & (step < 0) & (trial >= -126), trial, power)
        power = torch.where((top > 448.0 * torch.exp2(power)) & (step > 0), trial, power)
    scale = torch.exp2(power)
    codes = (full / scale[..., None]).float().to(torch.float8_e4m3fn).view(R, -1)[:, :K]
    return codes, scale


@pytest.mark.parametrize("rows,d", SIZES)
@pytest.mark.parametrize("types", ["fp16", "bf16", "fp32", "fp16 fp32", "bf16 fp32"])
def test_norm_with_and_without_residual(rows, d, types):
    from ccfuser_amd import ops
    dt, wt = (TYPES[n] for n in (types.split() * 2)[:2])
    x, r = _rows(1, rows, d, dtype=dt), _rows(2, rows, d, dtype=dt, std=3.0)
    w = (1.0 + 0.1 * _rows(3, d, dtype=torch.float32)).to(wt)
    for residual in (None, r):
        total, ref, rstd = _norm64(x, w, 1e-5, residual)
        got = ops.rms_norm(x, w, 1e-5, residual=residual, want_fp8=True, want_rstd=True)
        assert torch.equal(got.total, total) and (residual is not None or got.total is x)
        assert ((got.rstd.double() - rstd[:, 0]).abs() <= 40 * U * rstd[:, 0]).all()
        slack = 40 * U * ref.abs()
        assert ((got.y.double() - ref).abs() <= _half_step(ref, dt) * (1 + 40 * U) + slack).all()
        # the 8-bit form: one rounding of the unrounded result, by half a step of e4m3 or of its smallest subnormal
        scale = got.scale.double().repeat_interleave(128, -1)[:, :d]
        values = got.codes.float().double() * scale
        assert ((values - ref).abs() <= ref.abs() * 2.0 ** -4 * (1 + 40 * U) + scale * 2.0 ** -10 + slack).all()
        mantissa, _ = torch.frexp(got.scale)
        assert (mantissa == 0.5).all()
        top = torch.nn.functional.pad(ref.abs(), (0, -d % 128)).view(rows, -1, 128).amax(-1) / got.scale.double()
        assert (top <= 448 * (1 + 40 * U)).all() and ((top > 224 * (1 - 40 * U)) | (got.scale == 2.0 ** -126)).all()


def test_norm_of_other_shapes_and_of_no_rows():
    from ccfuser_amd import ops
    x, w = _rows(4, 2, 3, 200), torch.ones(200, dtype=torch.float16, device="cuda")
    a, b = ops.rms_norm(x, w, want_fp8=True), ops.rms_norm(x.view(6, 200), w, want_fp8=True)
    assert a.y.shape == x.shape and a.scale.shape == (2, 3, 2) and torch.equal(a.y.view(6, 200), b.y)
    assert torch.equal(a.codes.view(torch.uint8).view(6, 200), b.codes.view(torch.uint8))
    empty = ops.rms_norm(x[:0], w, residual=x[:0], want_fp8=True, want_rstd=True)
    assert empty.y.shape == (0, 3, 200) and empty.total.shape == (0, 3, 200) and empty.scale.shape == (0, 3, 2)
    g_x, g_w = ops.rms_norm_backward(empty.y, empty.total, w, empty.rstd)
    assert g_x.shape == (0, 3, 200) and not g_w.any()
    only = ops.rms_norm(x, w, want_y=False, want_fp8=True)
    assert only.y is None and torch.equal(only.codes.view(torch.uint8), a.codes.view(torch.uint8))


@pytest.mark.parametrize("dt", ["fp16", "fp32"])
@pytest.mark.parametrize("d", [96, 515, 4096])
def test_rows_that_start_at_any_element(dt, d):
    """Views that begin one element into their storage give the bits of aligned copies, and write nothing beside."""
    from ccfuser_amd import ops
    buf = _rows(5, 3 * d + 1, dtype=TYPES[dt])
    x, w = buf[1:].view(3, d), _rows(6, d + 1, dtype=TYPES[dt])[1:]
    a = ops.rms_norm(x, w, residual=x, want_fp8=True)
    b = ops.rms_norm(x.clone(), w.clone(), residual=x.clone(), want_fp8=True)
    assert torch.equal(a.y, b.y) and torch.equal(a.total, b.total) and torch.equal(a.scale, b.scale)
    assert torch.equal(a.codes.view(torch.uint8), b.codes.view(torch.uint8))
    assert torch.equal(ops.quantize_rows(x)[0].view(torch.uint8), ops.quantize_rows(x.clone())[0].view(torch.uint8))


def test_zeros_infinities_and_nan():
    from ccfuser_amd import ops
    x = _rows(7, 4, 256)
    x[0] = 0
    x[1, 3] = float("inf")
    x[2, 200] = float("nan")
    w = torch.ones(256, dtype=torch.float16, device="cuda")
    n = ops.rms_norm(x, w, want_fp8=True)
    assert not n.y[0].any() and not n.codes[0].float().any() and (n.scale[0] == 2.0 ** -126).all()
    assert n.y[1, 3].isnan() and not n.y[1, :3].any()            # inf * 0
    assert n.y[2].isnan().all() and n.codes[2].float().isnan().all()
    assert n.y[3].isfinite().all() and n.codes[3].float().isfinite().all()
    codes, scale = ops.quantize_rows(x)
    v = codes.float()
    assert v[1, 3].isnan() and v[1, 4:].isfinite().all() and v[2, 200].isnan() and v[2, :200].isfinite().all()
    assert scale.isfinite().all()


@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 127), (2, 128), (5, 1000), (33, 4096), (4097, 64)])
def test_rows_in_8_bits_are_exact(dt, rows, k):
    from ccfuser_amd import ops
    x = _rows(8, rows, k, dtype=TYPES[dt], std=2.0)
    x[0, 0] = 448.0                                              # borders of the scales, ties of the codes
    if k > 3:
        x[0, 1:4] = torch.tensor([1.0625, 1.1875, 2.0 ** -14], dtype=TYPES[dt])
    if rows > 1:
        x[1] *= 2.0 ** -12
        x[1, 0] = 1.75 * 2.0 ** -9
    codes, scale = ops.quantize_rows(x)
    want, want_scale = codes_of(x)
    assert torch.equal(scale.cpu().double(), want_scale)
    assert torch.equal(codes.cpu().float(), want.float())
    if dt == "fp32":                                             # small and large blocks of the wide type
        x = x * 2.0 ** -120
        codes, scale = ops.quantize_rows(x)
        want, want_scale = codes_of(x)
        assert torch.equal(scale.cpu().double(), want_scale) and torch.equal(codes.cpu().float(), want.float())


@pytest.mark.parametrize("shape", [(1, 1), (128, 128), (129, 257), (64, 1000), (3, 200, 192), (2, 16, 16)])
def test_weights_in_8_bits_are_exact(shape):
    from ccfuser_amd import ops
    for dt in (torch.float16, torch.float32):
        w = _rows(9, *shape, dtype=dt, std=0.02)
        codes, scale = ops.quantize_weight(w)
        full = torch.zeros(*shape[:-2], -(-shape[-2] // 128) * 128, -(-shape[-1] // 128) * 128, dtype=torch.float64)
        full[..., :shape[-2], :shape[-1]] = w.double().cpu()
        tiles = full.unflatten(-2, (-1, 128)).unflatten(-1, (-1, 128))          # [..., nb, 128, kb, 128]
        flat = tiles.transpose(-3, -2).flatten(-2)                              # a block as one row
        top = flat.abs().amax(-1).reshape(-1, 1)
        _, want_scale = codes_of(top)
        want_scale = want_scale.view(scale.shape)
        want = (tiles / want_scale[..., :, None, :, None]).float().to(torch.float8_e4m3fn).float()
        want = want.flatten(-2).flatten(-3, -2)[..., :shape[-2], :shape[-1]]
        assert torch.equal(scale.cpu().double(), want_scale)
        assert torch.equal(codes.cpu().float(), want)


def _backward64(g, total, w, eps, grad_total):
    t, r = total.double(), None
    rstd = (t.square().mean(-1, keepdim=True) + eps).rsqrt()
    gw = g.double() * w.double()
    c = (gw * t).mean(-1, keepdim=True)
    gx = rstd * (gw - t * rstd.square() * c)
    size = rstd * (gw.abs() + t.abs() * rstd.square() * (gw * t).abs().mean(-1, keepdim=True))
    if grad_total is not None:
        gx, size = gx + grad_total.double(), size + grad_total.double().abs()
    terms = g.double() * t * rstd
    return gx, size, terms.sum(0), terms.abs().sum(0)


@pytest.mark.parametrize("rows,d", SIZES)
@pytest.mark.parametrize("types", ["fp16", "bf16", "fp32", "bf16 fp32"])
def test_backward_against_the_formula(rows, d, types):
    from ccfuser_amd import ops
    dt, wt = (TYPES[n] for n in (types.split() * 2)[:2])
    t, g, gt = _rows(11, rows, d, dtype=dt, std=2.0), _rows(12, rows, d, dtype=dt, std=0.1), _rows(13, rows, d, dtype=dt, std=0.1)
    w = (1.0 + 0.1 * _rows(14, d, dtype=torch.float32)).to(wt)
    rstd = ops.rms_norm(t, w, 1e-5, want_rstd=True).rstd
    for grad_total in (None, gt):
        gx, size, gw, terms = _backward64(g, t, w, 1e-5, grad_total)
        a, b = ops.rms_norm_backward(g, t, w, rstd, grad_total)
        assert ((a.double() - gx).abs() <= _half_step(gx, dt) * (1 + U) + 128 * U * size).all()
        # a column's terms: one after the other in a workgroup, then over workgroups, at most rows additions in all
        assert ((b.double() - gw).abs() <= _half_step(gw, wt) * (1 + U) + (40 + rows) * U * terms).all()
        again = ops.rms_norm_backward(g, t, w, rstd, grad_total)
        assert torch.equal(a, again[0]) and torch.equal(b, again[1])
    only_x, none = ops.rms_norm_backward(g, t, w, rstd, gt, want_weight=False)
    nothing, only_w = ops.rms_norm_backward(g, t, w, rstd, gt, want_x=False)
    assert none is None and nothing is None and torch.equal(only_x, a) and torch.equal(only_w, b)


def test_autograd_and_differences():
    """The module's gradients against the formula, and against central differences of its own fp32 forward: a step of 2^-7
    along a direction of unit elements leaves h^2 terms of relative 1e-4 and roundings of u / h, 1e-5."""
    from ccfuser_amd.mix_moe import RMSNorm
    norm = RMSNorm(300, eps=1e-3).cuda()
    with torch.no_grad():
        norm.weight.copy_(1.0 + 0.1 * _rows(20, 300, dtype=torch.float32))
    x, r = _rows(21, 4, 5, 300, dtype=torch.float32).requires_grad_(), _rows(22, 4, 5, 300, dtype=torch.float32).requires_grad_()
    gy, gt = _rows(23, 4, 5, 300, dtype=torch.float32), _rows(24, 4, 5, 300, dtype=torch.float32)
    y, total = norm(x, r)
    grads = torch.autograd.grad((y, total), (x, r, norm.weight), (gy, gt))
    assert torch.equal(grads[0], grads[1])

    def loss(a, b, w):
        from ccfuser_amd import ops
        n = ops.rms_norm(a, w, 1e-3, residual=b)
        return (n.y.double() * gy.double()).sum() + (n.total.double() * gt.double()).sum()

    args = [x.detach(), r.detach(), norm.weight.detach()]
    for i, g in enumerate(grads):
        v = _rows(30 + i, *args[i].shape, dtype=torch.float32)
        h = 2.0 ** -7
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + h * v, args[i] - h * v
        slope = (loss(*up) - loss(*down)) / (2 * h)
        want = (g.double() * v.double()).sum()
        assert (slope - want).abs() <= 2e-3 * (g.double() * v.double()).norm() * v.numel() ** 0.5 / 10 + 1e-3 * want.abs()


def test_autograd_of_parts():
    """Only what needs a gradient gets one; unused outputs count as zero."""
    from ccfuser_amd.mix_moe import rms_norm
    x, r = _rows(25, 6, 128), _rows(26, 6, 128)
    w = torch.ones(128, dtype=torch.float16, device="cuda")
    gy = _rows(27, 6, 128)
    xr = x.clone().requires_grad_()
    y, total = rms_norm(xr, w, 1e-5, r)
    g, = torch.autograd.grad(total, xr, gy, retain_graph=True)
    assert torch.equal(g, gy)
    g, = torch.autograd.grad(y, xr, gy)
    wr = w.clone().requires_grad_()
    y = rms_norm(x, wr)
    gw, = torch.autograd.grad(y, wr, gy)
    from ccfuser_amd import ops
    n = ops.rms_norm(x, w, residual=r, want_rstd=True)
    assert torch.equal(g, ops.rms_norm_backward(gy, n.total, w, n.rstd)[0])
    n = ops.rms_norm(x, w, want_rstd=True)
    assert torch.equal(gw, ops.rms_norm_backward(gy, x, w, n.rstd)[1])
    with torch.no_grad():
        assert not rms_norm(xr, w).requires_grad
    broadcast = gy[:1].expand(6, 128)                             # a gradient that is not contiguous
    y = rms_norm(xr, w)
    g, = torch.autograd.grad(y, xr, broadcast)
    assert torch.equal(g, ops.rms_norm_backward(broadcast.contiguous(), x, w, n.rstd)[0])


def test_in_a_graph_and_on_another_stream():
    from ccfuser_amd import ops
    x, r, w = _rows(31, 50, 1000), _rows(32, 50, 1000), _rows(33, 1000)
    g = _rows(34, 50, 1000)

    def both():
        n = ops.rms_norm(x, w, residual=r, want_fp8=True, want_rstd=True)
        return (*n[:2], n.codes.view(torch.uint8), n.scale, *ops.rms_norm_backward(g, n.total, w, n.rstd))

    eager = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        aside = both()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, aside))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for seed in (35, 36, 37):
        x.copy_(_rows(seed, 50, 1000))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(both(), out))


def test_refusals():
    from ccfuser_amd import _lib, ops
    x, w = _rows(40, 4, 64), _rows(41, 64)
    with pytest.raises(ValueError):
        ops.rms_norm(x.t(), _rows(41, 4))
    with pytest.raises(ValueError):
        ops.rms_norm(x, w[:32].contiguous())
    with pytest.raises(TypeError):
        ops.rms_norm(x, w.bfloat16())
    with pytest.raises(TypeError):
        ops.rms_norm(x.double(), w.double())
    with pytest.raises(TypeError):
        ops.rms_norm(x, w, residual=x.float())
    with pytest.raises(ValueError):
        ops.rms_norm(x, w, residual=x[:2])
    with pytest.raises(ValueError):
        ops.rms_norm(x, w.cpu())
    with pytest.raises(ValueError):
        ops.rms_norm(x, w, want_y=False)
    with pytest.raises(ValueError):
        ops.rms_norm(x[:, :0].contiguous(), w[:0].contiguous())
    with pytest.raises(_lib.CcfError):
        ops.rms_norm(x, w, eps=-1.0)
    n = ops.rms_norm(x, w, want_rstd=True)
    with pytest.raises(ValueError):
        ops.rms_norm_backward(x[:2].contiguous(), x, w, n.rstd)
    with pytest.raises(ValueError):
        ops.rms_norm_backward(x, x, w, n.rstd[:3].contiguous())
    with pytest.raises(TypeError):
        ops.rms_norm_backward(x.float(), x, w, n.rstd)
    with pytest.raises(TypeError):
        ops.quantize_rows(x.double())
    with pytest.raises(ValueError):
        ops.quantize_rows(x[:, ::2])
    with pytest.raises(ValueError):
        ops.quantize_weight(x[0])
