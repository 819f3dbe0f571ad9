"""The MoE layer for a few tokens, and on experts in 8 bits, against float64.

The choice and the scores have to be the gate's own, bit for bit.  Tolerances, u = 2^-24: a sum of K products is off by at
most 2 (K + 8) u of the sum of magnitudes, in any order; the GELU (Lipschitz constant 1.13) by 5e-6 |v| + 1e-8; fp16 by half
a step, 2^-11 and 2^-25.  What h is off by passes through |w2|, scores add up what the experts' outputs are off by.

In 8 bits the reference takes the activations that ``ffn1_fp8`` leaves (tested on their own).  A kernel of another order of
sums may round an element to the neighbouring code where the exact value is within its error of the border between the two:
such elements, found in float64, may each be off by that step."""
import pytest
import torch

from test_gpu_gemm8 import _product, _row_values, _weight_values

pytestmark = pytest.mark.gpu
U = 2.0 ** -24

SIZES = [(1, 64, 64, 1, 1), (1, 256, 1024, 4, 1), (2, 128, 192, 8, 8), (3, 192, 320, 5, 3), (16, 256, 448, 8, 2), (17, 128, 192, 33, 8),
         (32, 320, 512, 8, 2), (13, 1024, 1024, 16, 2), (1, 4096, 1536, 8, 2), (32, 64, 128, 600, 4), (5, 768, 2048, 64, 2),
         (1, 2048, 64, 1024, 8)]


def _randn(seed, *shape, std=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).half().cuda()


def _layer(T, d, f, E, k, seed=1):
    std = 1.0 / d ** 0.5
    return dict(x=_randn(seed, T, d), wg=_randn(seed + 1, E, d, std=std), bg=_randn(seed + 2, E, std=0.1),
                w1=_randn(seed + 3, E, f, d, std=std), b1=_randn(seed + 4, E, f, std=0.3),
                w2=_randn(seed + 5, E, d, f, std=2.0 / f ** 0.5), b2=_randn(seed + 6, E, d, std=0.3))


def _gelu64(v):
    return 0.5 * v * (1 + torch.erf(v * 0.5 ** 0.5))


def _half_step(ref):
    return ref.abs() * 2.0 ** -11 + 2.0 ** -25


def _fp16_reference(l, idx, score):
    """(out, bound) in float64 for a given choice; entries of idx that are no expert count for nothing.  Beyond 16 tokens an
    expert's output is itself rounded to fp16 before its score multiplies it: score times half a step of it, no more."""
    T, k = idx.shape
    x = l["x"].double()
    out = torch.zeros_like(x)
    off = torch.zeros_like(x)
    for e in idx[idx >= 0].unique().tolist():
        t, s = (idx == e).nonzero(as_tuple=True)
        w1, w2, b1, b2 = (l[n][e].double() for n in ("w1", "w2", "b1", "b2"))
        v = x[t] @ w1.t() + b1
        lost = 2 * (x.shape[1] + 8) * U * (x[t].abs() @ w1.abs().t() + b1.abs())
        h = _gelu64(v)
        h_off = 1.13 * lost + 5e-6 * v.abs() + 1e-8 + _half_step(h)
        g = score[t, s].double()[:, None]
        out.index_add_(0, t, g * (h @ w2.t() + b2))
        y_off = h_off @ w2.abs().t() + 2 * (h.shape[1] + 16) * U * (h.abs() @ w2.abs().t() + b2.abs())
        if T > 16:
            y_off = y_off + _half_step((h @ w2.t() + b2).abs() + y_off)
        off.index_add_(0, t, g * y_off)
    return out, off * 1.01


@pytest.mark.parametrize("T,d,f,E,k", SIZES)
def test_layer_in_16_bits(T, d, f, E, k):
    from ccfuser_amd import ops
    l = _layer(T, d, f, E, k)
    out, r = ops.moe_forward_few(*l.values(), k, return_routing=True)
    idx, score = ops.gate_topk_softmax(l["x"], l["wg"], l["bg"], k)
    assert torch.equal(r["idx"], idx) and torch.equal(r["score"], score)
    ref, off = _fp16_reference(l, idx, score)
    assert ((out.double() - ref).abs() <= off + _half_step(ref)).all()
    assert torch.equal(out, ops.moe_forward_few(*l.values(), k))
    # next to the layer of any size: two roundings of an expert's output apart
    near = ops.moe_forward(*l.values(), k)
    assert (near.double() - out.double()).norm() <= 4 * 2.0 ** -11 * k ** 0.5 * ref.norm() + off.norm()


def _codes_of_layer(l):
    from ccfuser_amd import ops
    w1, s1 = ops.quantize_weight(l["w1"])
    w2, s2 = ops.quantize_weight(l["w2"])
    # scales of any value, as a checkpoint has them
    jitter = lambda s, seed: s * (1.0 + 0.3 * torch.rand(s.shape, generator=torch.Generator().manual_seed(seed)).cuda())
    return w1, jitter(s1, 50), w2, jitter(s2, 51)


def _fp8_reference(l, q, idx, score, x_fp8):
    from ccfuser_amd import ops
    w1, s1, w2, s2 = q
    T, d = l["x"].shape
    f = w1.shape[1]
    xv = _row_values(*x_fp8)
    out, off = torch.zeros(T, d, dtype=torch.float64, device="cuda"), torch.zeros(T, d, dtype=torch.float64, device="cuda")
    for e in idx[idx >= 0].unique().tolist():
        t, s = (idx == e).nonzero(as_tuple=True)
        n = t.numel()
        offsets = torch.tensor([0, n], dtype=torch.int32, device="cuda")
        h, hs = ops.ffn1_fp8(x_fp8, t.to(torch.int32), offsets, n, w1[e:e + 1], s1[e:e + 1], l["b1"][e:e + 1])
        v, lost = _product(xv[t], _weight_values(w1[e], s1[e]), l["b1"][e])
        exact, slack = _gelu64(v), 1.13 * lost + 5e-6 * v.abs() + 1e-8
        scale = hs.double().repeat_interleave(128, -1)[:, :f]
        to = lambda y: y.clamp(-448 * scale, 448 * scale).div(scale).float().to(torch.float8_e4m3fn).double() * scale
        step = (to(exact + slack) - to(exact - slack)).abs()
        top = torch.nn.functional.pad(exact.abs() + slack, (0, -f % 128)).view(n, -1, 128).amax(-1)
        border = (top >= 448 * hs.double()) | (torch.nn.functional.pad(exact.abs() - slack, (0, -f % 128)).view(n, -1, 128).amax(-1)
                                               <= 224 * hs.double())
        step = step + border.repeat_interleave(128, -1)[:, :f] * scale * 2.0 ** -9       # subnormals of a scale twice or half as large
        mine = _row_values(h, hs)
        y, y_off = _product(mine, _weight_values(w2[e], s2[e]), l["b2"][e])
        g = score[t, s].double()[:, None]
        out.index_add_(0, t, g * y)
        off.index_add_(0, t, g * (y_off + step @ _weight_values(w2[e], s2[e]).abs().t()))
    return out, off * 1.01


@pytest.mark.parametrize("T,d,f,E,k", SIZES)
def test_layer_in_8_bits_of_few_tokens(T, d, f, E, k):
    from ccfuser_amd import ops
    l = _layer(T, d, f, E, k, seed=20)
    q = _codes_of_layer(l)
    x_fp8 = ops.quantize_rows(l["x"])
    args = (l["x"], l["wg"], l["bg"], q[0], q[1], l["b1"], q[2], q[3], l["b2"], k)
    out, r = ops.moe_forward_fp8(*args, return_routing=True)
    idx, score = ops.gate_topk_softmax(l["x"], l["wg"], l["bg"], k)
    assert torch.equal(r["idx"], idx) and torch.equal(r["score"], score)
    rounded = lambda x_fp8: _outputs_half_steps(l, q, idx, score, x_fp8) if T > 16 else 0           # as in _fp16_reference
    ref, off = _fp8_reference(l, q, idx, score, x_fp8)
    assert ((out.double() - ref).abs() <= off + _half_step(ref) + rounded(x_fp8)).all()
    assert torch.equal(out, ops.moe_forward_fp8(*args, x_fp8=x_fp8))
    assert torch.equal(out, ops.moe_forward_fp8(*args, capacity=T))
    # another norm's rows for the experts than for the gate
    other = ops.quantize_rows(l["x"] * 0.5)
    ref, off = _fp8_reference(l, q, idx, score, other)
    assert ((ops.moe_forward_fp8(*args, x_fp8=other).double() - ref).abs() <= off + _half_step(ref) + rounded(other)).all()


@pytest.mark.parametrize("T,d,f,E,k,capacity", [(33, 128, 192, 4, 1, -1), (100, 256, 512, 8, 2, -1), (20, 256, 320, 4, 2, 5),
                                                (1999, 192, 320, 8, 2, -1), (700, 320, 576, 16, 3, 90), (5000, 256, 512, 4, 2, -1)])
def test_layer_in_8_bits_of_any_size(T, d, f, E, k, capacity):
    from ccfuser_amd import ops
    l = _layer(T, d, f, E, k, seed=40)
    q = _codes_of_layer(l)
    x_fp8 = ops.quantize_rows(l["x"])
    args = (l["x"], l["wg"], l["bg"], q[0], q[1], l["b1"], q[2], q[3], l["b2"], k)
    out, r = ops.moe_forward_fp8(*args, capacity=capacity, return_routing=True)
    idx, score = ops.gate_topk_softmax(l["x"], l["wg"], l["bg"], k)
    kept = ops.route(idx, E, k, capacity)["idx_kept"].view(T, k)
    assert torch.equal(r["idx"], kept) and torch.equal(r["score"], score)
    ref, off = _fp8_reference(l, q, kept, score, x_fp8)
    # an expert's output is rounded to fp16 before the combine
    assert ((out.double() - ref).abs() <= off + _half_step(ref) + _outputs_half_steps(l, q, kept, score, x_fp8)).all()
    assert torch.equal(out, ops.moe_forward_fp8(*args, capacity=capacity, x_fp8=x_fp8))


def _outputs_half_steps(l, q, idx, score, x_fp8):
    """sum over a token's slots of score times half a step of the expert's output."""
    total = torch.zeros(l["x"].shape, dtype=torch.float64, device="cuda")
    for s in range(idx.shape[1]):
        one = torch.full_like(idx, -1)
        one[:, s] = idx[:, s]
        y, off = _fp8_reference(l, q, one, torch.ones_like(score), x_fp8)
        total += score[:, s].double()[:, None] * _half_step(y.abs() + off)
    return total


def test_without_biases_and_with_spare_experts():
    from ccfuser_amd import ops
    l = _layer(4, 128, 192, 6, 2, seed=60)
    gate = (l["wg"][:4].contiguous(), l["bg"][:4].contiguous())
    a = ops.moe_forward_few(l["x"], *gate, l["w1"], l["b1"], l["w2"], l["b2"], 2, spare_experts=True)
    b = ops.moe_forward_few(l["x"], *gate, *(l[n][:4].contiguous() for n in ("w1", "b1", "w2", "b2")), 2)
    assert torch.equal(a, b)
    c = ops.moe_forward_few(l["x"], gate[0], None, *(l[n][:4].contiguous() for n in ("w1", "b1", "w2", "b2")), 2)
    assert torch.equal(c, ops.moe_forward_few(l["x"], gate[0], torch.zeros_like(gate[1]), *(l[n][:4].contiguous() for n in
                                                                                         ("w1", "b1", "w2", "b2")), 2))
    q = _codes_of_layer(l)
    for T in (4, 50):
        x = _randn(70, T, 128)
        none = ops.moe_forward_fp8(x, l["wg"], l["bg"], q[0], q[1], None, q[2], q[3], None, 2)
        zero = ops.moe_forward_fp8(x, l["wg"], l["bg"], q[0], q[1], l["b1"] * 0, q[2], q[3], l["b2"] * 0, 2)
        assert torch.equal(none, zero)
    assert ops.moe_forward_few(l["x"][:0], *(l[n] for n in ("wg", "bg", "w1", "b1", "w2", "b2")), 2).shape == (0, 128)
    assert ops.moe_forward_fp8(l["x"][:0], l["wg"], l["bg"], q[0], q[1], None, q[2], q[3], None, 2).shape == (0, 128)


def test_tokens_that_are_no_numbers_keep_to_themselves():
    from ccfuser_amd import ops
    l = _layer(6, 128, 192, 8, 2, seed=80)
    q = _codes_of_layer(l)
    run16 = lambda x: ops.moe_forward_few(x, *(l[n] for n in ("wg", "bg", "w1", "b1", "w2", "b2")), 2)
    run8 = lambda x: ops.moe_forward_fp8(x, l["wg"], l["bg"], q[0], q[1], l["b1"], q[2], q[3], l["b2"], 2)
    for run in (run16, run8):
        clean = run(l["x"])
        bad = l["x"].clone()
        bad[2, 5] = float("nan")
        bad[4, 9] = float("inf")
        out = run(bad)
        keep = [0, 1, 3, 5]
        assert torch.equal(out[keep], clean[keep])
    # weights of an expert that are no numbers spoil the tokens that chose it and no other
    idx, _ = ops.gate_topk_softmax(l["x"], l["wg"], l["bg"], 2)
    e = int(idx[0, 0])
    hit = (idx == e).any(1)
    w2 = l["w2"].clone()
    w2[e, 7] = float("nan")
    out = ops.moe_forward_few(l["x"], l["wg"], l["bg"], l["w1"], l["b1"], w2, l["b2"], 2)
    assert out[hit][:, 7].isnan().all() and out[~hit].isfinite().all()


def test_in_a_graph_and_on_another_stream():
    from ccfuser_amd import ops
    l = _layer(9, 256, 512, 8, 2, seed=90)
    q = _codes_of_layer(l)

    def both():
        return (ops.moe_forward_few(*l.values(), 2),
                ops.moe_forward_fp8(l["x"], l["wg"], l["bg"], q[0], q[1], l["b1"], q[2], q[3], l["b2"], 2),
                ops.moe_forward_fp8(big, l["wg"], l["bg"], q[0], q[1], l["b1"], q[2], q[3], l["b2"], 2, 30))

    big = _randn(99, 200, 256)
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
    for seed in (91, 92, 93):
        l["x"].copy_(_randn(seed, 9, 256))
        big.copy_(_randn(seed + 10, 200, 256))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(both(), out))


def test_refusals():
    from ccfuser_amd import _lib, ops
    l = _layer(4, 128, 192, 4, 2, seed=100)
    q = _codes_of_layer(l)
    few = lambda k=2, **o: ops.moe_forward_few(*{**l, **o}.values(), k)
    eight = lambda k=2, x=l["x"], w1=q[0], s1=q[1], b1=l["b1"], **o: ops.moe_forward_fp8(x, l["wg"], l["bg"], w1, s1, b1, q[2], q[3],
                                                                                        l["b2"], k, **o)
    with pytest.raises(ValueError, match="32 tokens"):
        few(x=_randn(101, 33, 128))
    with pytest.raises(TypeError):
        few(x=l["x"].float())
    with pytest.raises(TypeError):
        eight(x=l["x"].float())
    with pytest.raises(TypeError):
        eight(w1=l["w1"])
    for call in (lambda: few(k=0), lambda: few(k=5), lambda: few(w1=l["w1"][:3].contiguous(), b1=l["b1"][:3].contiguous()),
                 lambda: few(wg=l["wg"][:, :64].contiguous()), lambda: few(x=l["x"].cpu()), lambda: few(b2=l["b2"].cpu()),
                 lambda: eight(k=5), lambda: eight(s1=q[1][:, :1].contiguous()), lambda: eight(b1=l["b1"][:, :64].contiguous()),
                 lambda: eight(x_fp8=ops.quantize_rows(_randn(102, 5, 128))), lambda: eight(x=l["x"][:, ::2])):
        with pytest.raises(ValueError):
            call()
    odd = _layer(4, 96, 192, 4, 2, seed=103)
    with pytest.raises(_lib.CcfError, match="multiple of 64"):
        ops.moe_forward_few(*odd.values(), 2)
    oq = _codes_of_layer(odd)
    with pytest.raises(_lib.CcfError, match="multiple of 64"):
        ops.moe_forward_fp8(odd["x"], odd["wg"], odd["bg"], oq[0], oq[1], None, oq[2], oq[3], None, 2)
    with pytest.raises(_lib.CcfError, match="workspace"):
        ops.moe_forward_few(*l.values(), 2, workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    with pytest.raises(_lib.CcfError, match="workspace"):
        eight(workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
