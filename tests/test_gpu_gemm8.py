"""Products in 8 bits, dense and grouped by expert, against float64.

Tolerances: products of codes are exact in fp32; a sum of K of them and its scaling are off by at most (K + 8) u of the sum
of magnitudes, u = 2^-24, however it is ordered and each addition rounded or truncated (2 u); the output is rounded once, by
half a step of its type.  The matrix instruction adds eight consecutive products at a time and cuts each of them off at
2^-13 of 2^(the largest sum of a product's two exponents) (measured: next to 448 * 448 = 3.06 * 2^16, of which one of each
sign cancel, 8 = 2^-13 * 2^16 counts and 4 does not, 12 counts as 8; behind the next multiple of eight everything counts).
The largest product of the eight is at least that power of two and is not cut itself beyond its own last bit, so they lose
at most 7 * 2^-13 of it: in all 7 * 2^-13 of the sum over groups of eight of max |a| max |w|.  Through the GELU (Lipschitz constant 1.13, itself within 4e-6 |v| + 1e-9) to 8 bits: half a step of
e4m3, 2^-4, or of its smallest subnormal, and a scale's border may fall either way, which costs the subnormals one bit."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(params=range(7), ids=["by_rule", "k_over_wavefronts", "tiles", "tiles_of_128", "tiles_of_64", "tiles_and_rest", "two_groups"],
                autouse=True)
def form(request):
    """Every test in the form that the library picks, and in each of them."""
    from ccfuser_amd import ops
    ops.set_option("fp8_form", request.param)
    yield request.param
    ops.set_option("fp8_form", 0)


def _randn(seed, *shape, std=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).cuda()


def _codes(seed, *shape):
    """Codes of every exponent and any scales: magnitudes over four powers of ten."""
    c = _randn(seed, *shape, std=30.0).clamp(-448, 448).to(torch.float8_e4m3fn)
    return c


def _row_scales(seed, rows, k):
    return torch.exp(_randn(seed, rows, -(-k // 128)) * 2.0 - 4.0)


def _block_scales(seed, *shape):
    *e, n, k = shape
    return torch.exp(_randn(seed, *e, -(-n // 128), -(-k // 128)) * 2.0 - 6.0)


def _row_values(c, s):
    return c.float().double() * s.double().repeat_interleave(128, -1)[..., :c.shape[-1]]


def _weight_values(c, s):
    n, k = c.shape[-2:]
    return c.float().double() * s.double().repeat_interleave(128, -2)[..., :n, :].repeat_interleave(128, -1)[..., :k]


def _largest_of_eight(v):
    return torch.nn.functional.pad(v.abs(), (0, -v.shape[-1] % 8)).unflatten(-1, (-1, 8)).amax(-1)


def _product(x, w, bias):
    """(exact result, bound of what the sums lose) of x [r, k] and w [n, k] in float64."""
    y, size = x @ w.t(), x.abs() @ w.abs().t()
    cut = _largest_of_eight(x) @ _largest_of_eight(w).t()
    if bias is not None:
        y, size = y + bias.double(), size + bias.double().abs()
    return y, 2 * (x.shape[1] + 8) * U * size + 7 * 2.0 ** -13 * cut


def _within(got, ref, slack, dtype):
    f = torch.finfo(dtype)
    err = (got.double() - ref).abs()
    big = ref.abs() + slack > f.max                              # beyond the type: infinities
    ok = err <= ref.abs() * f.eps / 2 + f.tiny * f.eps / 2 + slack * (1 + f.eps)
    assert (ok | big).all(), (err / (ref.abs() + 1e-30)).max()


@pytest.mark.parametrize("rows,k,n", [
    (1, 16, 8), (1, 128, 64), (3, 144, 72), (16, 256, 128), (17, 640, 200), (31, 1024, 64), (33, 400, 264), (64, 128, 1000),
    (65, 2048, 128), (129, 336, 520), (200, 64, 256), (333, 1024, 4096), (2049, 1040, 2056), (4096, 4096, 1024), (1, 4096, 14336)])
@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp16 of ones"])
def test_dense_product(rows, k, n, dt):
    from ccfuser_amd import ops
    dtype = torch.bfloat16 if dt == "bf16" else torch.float16
    x, xs = _codes(1, rows, k), _row_scales(2, rows, k) * 1e-2
    w, ws = _codes(3, n, k), _block_scales(4, n, k) * 1e-2
    if "ones" in dt:                                             # results about 1 in size, far from fp16's subnormals
        xs, ws = xs * 1e2, ws * (4.0 * 1e2 / k ** 0.5)
    bias = _randn(5, n, std=0.1).to(dtype)
    a, b = _row_values(x, xs), _weight_values(w, ws)
    for bi in (bias, None):
        y = ops.linear_fp8((x, xs), w, ws, bi, dtype=dtype)
        assert y.dtype == dtype and y.shape == (rows, n)
        _within(y, *_product(a, b, bi), dtype)
        assert torch.equal(y, ops.linear_fp8((x, xs), w, ws, bi, dtype=dtype))


@pytest.mark.parametrize("rows", [1, 40, 300])
def test_dense_product_of_16_bit_rows(rows):
    """The call quantises rows of 16 bits as quantize_rows does."""
    from ccfuser_amd import ops
    for dtype in (torch.float16, torch.bfloat16):
        x = _randn(6, rows, 512).to(dtype)
        w, ws = ops.quantize_weight(_randn(7, 320, 512, std=0.02).to(dtype))
        y = ops.linear_fp8(x, w, ws)
        assert y.dtype == dtype
        assert torch.equal(y, ops.linear_fp8(ops.quantize_rows(x), w, ws, dtype=dtype))
        _within(y, *_product(_row_values(*ops.quantize_rows(x)), _weight_values(w, ws), None), dtype)
        # and is near the product in 16 bits: two roundings of 2^-4 at most per product, of either sign
        near = x.double() @ _weight_values(w, ws).t()
        assert (y.double() - near).norm() <= 2.0 ** -4 * near.norm()


def _experts(seed, counts):
    E, n = len(counts), sum(counts)
    offsets = torch.tensor([0] + counts, dtype=torch.int32).cumsum(0).to(torch.int32).cuda()
    g = torch.Generator().manual_seed(seed)
    return E, n, offsets, torch.randperm(max(n, 1), generator=g)[:n].to(torch.int32).cuda()


COUNTS = [[1], [0, 3, 0, 0], [16, 0, 1, 17], [5] * 32, [0] * 70 + [9, 0, 31], [300, 1, 0, 129], [256, 257, 512], [1030, 1000, 0, 900, 1100],
          [40, 60, 80, 128], [2, 0, 700]]


@pytest.mark.parametrize("size", [1.0, 30.0])
@pytest.mark.parametrize("counts", COUNTS, ids=str)
@pytest.mark.parametrize("d,f", [(64, 192), (320, 1024), (1024, 4096)])
def test_grouped_products(counts, d, f, size):
    """Both expert products over every kind of load; rows behind the last expert's stay as they were."""
    from ccfuser_amd import ops
    if len(counts) > 16 and d > 320:
        d, f = 320, 512
    E, n, offsets, src = _experts(8, counts)
    spare = 5                                                    # rows that belong to nobody (max_rows bounds offsets[-1])
    tokens = n + spare
    x, xs = _codes(9, tokens, d), _row_scales(10, tokens, d) * 1e-2
    w1, s1 = _codes(11, E, f, d), _block_scales(12, E, f, d) * 1e-2 * size
    w2, s2 = _codes(13, E, d, f), _block_scales(14, E, d, f) * 1e-2 * size
    b1, b2 = _randn(15, E, f, std=0.2).half(), _randn(16, E, d, std=0.2).half()
    src = torch.cat([src, torch.zeros(spare, dtype=torch.int32, device="cuda")])
    h, hs = ops.ffn1_fp8((x, xs), src, offsets, n + spare, w1, s1, b1)
    y = torch.full((n + spare, d), 7.0, dtype=torch.float16, device="cuda")
    ops.ffn2_fp8((h, hs), src, offsets, n + spare, w2, s2, b2, y)
    written = torch.zeros(n + spare, dtype=torch.bool, device="cuda")
    at = 0
    for e, c in enumerate(counts):
        if c == 0:
            continue
        j = slice(at, at + c)
        at += c
        row = src[j].long()
        v, lost = _product(_row_values(x[row], xs[row]), _weight_values(w1[e], s1[e]), b1[e])
        ref = 0.5 * v * (1 + torch.erf(v * 0.5 ** 0.5))
        slack = 1.13 * lost + 5e-6 * v.abs() + 1e-8
        mine = _row_values(h[j], hs[j])
        scale = hs[j].double().repeat_interleave(128, -1)[:, :f]
        assert ((mine - ref).abs() <= ref.abs() * 2.0 ** -4 + scale * 2.0 ** -10 + slack * 1.1).all()
        assert (torch.frexp(hs[j])[0] == 0.5).all()
        top = torch.nn.functional.pad(ref.abs() + slack, (0, -f % 128)).view(c, -1, 128).amax(-1) / hs[j].double()
        assert (top > 224 * (1 - 1e-4)).logical_or(hs[j] == 2.0 ** -126).all()
        _within(y[row], *_product(mine, _weight_values(w2[e], s2[e]), b2[e]), torch.float16)
        written[row] = True
    assert (y[~written] == 7.0).all()


def test_without_row_lists_and_without_rows():
    from ccfuser_amd import ops
    counts = [7, 0, 50]
    E, n, offsets, _ = _experts(17, counts)
    x = _randn(18, n, 256).half()
    w1, s1 = ops.quantize_weight(_randn(19, E, 128, 256, std=0.05).half())
    w2, s2 = ops.quantize_weight(_randn(20, E, 256, 128, std=0.05).half())
    rows = torch.arange(n, dtype=torch.int32, device="cuda")
    a, b = ops.ffn1_fp8(x, None, offsets, n, w1, s1, None), ops.ffn1_fp8(x, rows, offsets, n, w1, s1, None)
    assert torch.equal(a[0].view(torch.uint8), b[0].view(torch.uint8)) and torch.equal(a[1], b[1])
    y, z = torch.empty_like(x), torch.empty_like(x)
    assert torch.equal(ops.ffn2_fp8(a, None, offsets, n, w2, s2, None, y), ops.ffn2_fp8(a, rows, offsets, n, w2, s2, None, z))
    nobody = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    y.fill_(3.0)
    ops.ffn2_fp8(a, None, nobody, n, w2, s2, None, y)
    assert (y == 3.0).all()
    empty = ops.linear_fp8(x[:0], w1[0], s1[0])
    assert empty.shape == (0, 128)
    h, hs = ops.ffn1_fp8(x[:0], None, nobody, 0, w1, s1, None)
    assert h.shape == (0, 128) and hs.shape == (0, 1)


@pytest.mark.parametrize("rows", [3, 60, 700])
def test_codes_that_are_no_numbers(rows):
    """A NaN code spoils its row (or its column) and nothing else; infinite and zero scales act as numbers."""
    from ccfuser_amd import ops
    x, w = _randn(21, rows, 256).half(), _randn(22, 512, 256, std=0.05).half()
    wq, ws = ops.quantize_weight(w)
    clean = ops.linear_fp8(x, wq, ws)
    x[1, 77] = float("nan")
    x[2, 5] = float("inf")
    y = ops.linear_fp8(x, wq, ws)
    assert y[1].isnan().all() and y[2].isnan().all()
    keep = [i for i in range(rows) if i not in (1, 2)]
    assert torch.equal(y[keep], clean[keep])
    ws[0, 1] = 0.0
    assert ops.linear_fp8(x, wq, ws)[keep].isfinite().all()


def test_in_a_graph_and_on_another_stream():
    from ccfuser_amd import ops
    x = _randn(23, 700, 512).half()
    w, s = ops.quantize_weight(_randn(24, 1024, 512, std=0.02).half())
    eager = ops.linear_fp8(x, w, s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        aside = ops.linear_fp8(x, w, s)
    side.synchronize()
    assert torch.equal(eager, aside)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.linear_fp8(x, w, s)
    for seed in (25, 26, 27):
        x.copy_(_randn(seed, 700, 512))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.linear_fp8(x, w, s))


def test_refusals():
    from ccfuser_amd import _lib, ops
    x = _randn(28, 4, 256).half()
    w, s = ops.quantize_weight(_randn(29, 64, 256).half())
    w3, s3 = ops.quantize_weight(_randn(29, 2, 64, 256).half())
    b = torch.zeros(64, dtype=torch.float16, device="cuda")
    off = torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    for bad in (lambda: ops.linear_fp8(x, w.float(), s), lambda: ops.linear_fp8(x.float(), w, s), lambda: ops.linear_fp8(x, w, s.half()),
                lambda: ops.linear_fp8(x, w, s, b.float()), lambda: ops.linear_fp8(x, w, s, dtype=torch.float32),
                lambda: ops.linear_fp8(x, w, s, b, dtype=torch.bfloat16), lambda: ops.ffn1_fp8(x, None, off.long(), 4, w3, s3, None)):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: ops.linear_fp8(x[:, :128].contiguous(), w, s), lambda: ops.linear_fp8(x, w, s[:, :1].contiguous()),
                lambda: ops.linear_fp8(x, w.t(), s), lambda: ops.linear_fp8(x, w, s, b[:32].contiguous()),
                lambda: ops.linear_fp8(x, w.cpu(), s.cpu()), lambda: ops.linear_fp8(x, w, s, b.cpu()),
                lambda: ops.ffn1_fp8(x, None, off[:2].contiguous(), 4, w3, s3, None), lambda: ops.ffn1_fp8(x, None, off, 5, w3, s3, None),
                lambda: ops.ffn1_fp8(x, off, off, 4, w3, s3, None), lambda: ops.ffn1_fp8(x, None, off, 4, w3, s3, b[None]),
                lambda: ops.ffn2_fp8(x[:, :64].contiguous(), None, off, 4, w3, s3, None, x)):
        with pytest.raises(ValueError):
            bad()
    odd, odd_s = ops.quantize_weight(_randn(30, 64, 200).half())
    with pytest.raises(_lib.CcfError, match="multiples of 16"):
        ops.linear_fp8(x[:, :200].contiguous(), odd, odd_s)
    odd, odd_s = ops.quantize_weight(_randn(30, 60, 256).half())
    with pytest.raises(_lib.CcfError, match="multiples of 16"):
        ops.linear_fp8(x, odd, odd_s)
