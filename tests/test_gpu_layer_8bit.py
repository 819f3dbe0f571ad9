"""The norm in front of the MoE layer, the few-token layer and experts in 8 bits, as a transformer block's module runs them."""
import pytest
import torch

from test_gpu_few_layer import _fp8_reference, _half_step, _layer, _codes_of_layer, _outputs_half_steps

pytestmark = pytest.mark.gpu


def _mlp(l, k, **kw):
    from ccfuser_amd.mix_moe import MixMOETransformerMLP
    E, f, d = l["w1"].shape
    mlp = MixMOETransformerMLP("naive", {"num_local_expert": E, "hidden_size": f}, d, 0, 1, total_batch_size=l["x"].shape[0], top_k=k,
                               popular_expert_num=1, **kw).half().cuda()
    with torch.no_grad():
        mlp.gate.gate.weight.copy_(l["wg"])
        mlp.gate.gate.bias.copy_(l["bg"])
        for lin, w, b in ((mlp.experts.htoh4, l["w1"], l["b1"]), (mlp.experts.h4toh, l["w2"], l["b2"])):
            lin.weight[:E].copy_(w)
            lin.bias[:E].copy_(b)
        if mlp.norm is not None:
            mlp.norm.weight.copy_(1 + 0.1 * torch.randn(d, generator=torch.Generator().manual_seed(9)).cuda())
    return mlp


@pytest.mark.parametrize("T,d,f,E,k", [(1, 256, 512, 8, 2), (32, 128, 192, 4, 1), (300, 256, 320, 4, 2)])
def test_residual_norm_and_layer(T, d, f, E, k):
    """total = x + residual, y = norm(total), its codes to the experts and y itself to the gate; the norm is tested on its own,
    so the layer's reference starts at its outputs."""
    from ccfuser_amd import ops
    l = _layer(T, d, f, E, k, seed=60)
    q = _codes_of_layer(l)
    residual = l["x"].flip(0) * 0.5
    weight = torch.ones(d, dtype=torch.float16, device="cuda") * 1.25
    n = ops.rms_norm(l["x"], weight, 1e-5, residual=residual, want_fp8=True)
    exact = (l["x"].double() + residual.double()).half().double()
    y = exact * torch.rsqrt((exact * exact).mean(-1, keepdim=True) + 1e-5) * 1.25
    assert torch.equal(n.total.double(), exact)
    # fp32 sums of d squares, a root and two products: (d + 16) 2^-24 in relative terms, and the rounding to fp16
    assert ((n.y.double() - y).abs() <= y.abs() * (d + 16) * 2.0 ** -24 + _half_step(y) * 1.001).all()
    l["x"] = n.y
    x_fp8 = (n.codes, n.scale)
    out, r = ops.moe_forward_fp8(n.y, l["wg"], l["bg"], q[0], q[1], l["b1"], q[2], q[3], l["b2"], k, x_fp8=x_fp8, return_routing=True)
    ref, off = _fp8_reference(l, q, r["idx"], r["score"], x_fp8)
    extra = _outputs_half_steps(l, q, r["idx"], r["score"], x_fp8) if T > 16 else 0
    assert ((out.double() - ref).abs() <= off + _half_step(ref) + extra).all()


@pytest.mark.parametrize("T", [1, 7, 200])
@pytest.mark.parametrize("pre_norm", [False, True])
def test_module_on_experts_in_8_bits(T, pre_norm):
    from ccfuser_amd import ops
    k = 2
    l = _layer(T, 256, 512, 8, k, seed=70)
    mlp = _mlp(l, k, pre_norm=pre_norm)
    with torch.no_grad():
        before = mlp(l["x"])
        assert mlp.quantize_experts() is mlp
        out = mlp(l["x"])
        w1, s1 = ops.quantize_weight(l["w1"])
        w2, s2 = ops.quantize_weight(l["w2"])
        x, x_fp8 = l["x"], None
        if pre_norm:
            n = ops.rms_norm(x, mlp.norm.weight, mlp.norm.eps, want_fp8=True)
            x, x_fp8 = n.y, (n.codes, n.scale)
        assert torch.equal(out, ops.moe_forward_fp8(x, l["wg"], l["bg"], w1, s1, l["b1"], w2, s2, l["b2"], k, x_fp8=x_fp8))
        assert not torch.equal(out, before)
        assert torch.equal(mlp(l["x"].view(1, T, -1)), out.view(1, T, -1))
    # with a gradient the stored weights
    x = l["x"].clone().requires_grad_()
    y = mlp(x)
    y.float().square().sum().backward()
    assert x.grad is not None and mlp.experts.htoh4.weight.grad is not None and (not pre_norm or mlp.norm.weight.grad is not None)
    with torch.no_grad():
        mlp.experts.htoh4.weight.mul_(2)
        with pytest.raises(RuntimeError, match="changed"):
            mlp(l["x"])
        mlp.experts.htoh4.weight.mul_(0.5)
        assert torch.equal(mlp.quantize_experts()(l["x"]), out)
        mlp.quantize_experts()
        mlp.experts.h4toh.weight = torch.nn.Parameter(mlp.experts.h4toh.weight.clone())
        with pytest.raises(RuntimeError, match="changed"):
            mlp(l["x"])
        assert torch.equal(mlp.quantize_experts(False)(l["x"]), before)
    mlp.close()


def test_module_with_norm_equals_its_parts():
    from ccfuser_amd import ops
    l = _layer(40, 128, 192, 4, 2, seed=80)
    plain, normed = _mlp(l, 2), _mlp(l, 2, pre_norm=True)
    with torch.no_grad():
        y = ops.rms_norm(l["x"], normed.norm.weight, normed.norm.eps).y
        assert torch.equal(normed(l["x"]), plain(y))
        normed.async_expert_assignment(l["x"])
        asynchronous = normed(l["x"])
        plain.async_expert_assignment(y)
        assert torch.equal(asynchronous, plain(y))
    assert "norm.weight" in normed.state_dict() and not any("norm" in n for n in plain.state_dict())
    # the gradient through the norm is the norm's of the layer's
    x = l["x"].clone().requires_grad_()
    g = torch.randn_like(l["x"])
    grad_x, grad_w = torch.autograd.grad(normed(x), (x, normed.norm.weight), g)
    leaf = y.clone().requires_grad_()
    (grad_y,) = torch.autograd.grad(plain(leaf), leaf, g)
    n = ops.rms_norm(l["x"], normed.norm.weight, normed.norm.eps, want_rstd=True)
    want_x, want_w = ops.rms_norm_backward(grad_y, n.total, normed.norm.weight.detach(), n.rstd)
    assert torch.equal(grad_x, want_x) and torch.equal(grad_w, want_w)
    for m in (plain, normed):
        m.close()


@pytest.mark.parametrize("T", [1, 13, 32, 33])
def test_module_of_few_tokens(T):
    from ccfuser_amd import ops
    l = _layer(T, 256, 512, 8, 2, seed=90)
    few, any_size = _mlp(l, 2, few_tokens=32), _mlp(l, 2)
    with torch.no_grad():
        args = [l[n] for n in ("x", "wg", "bg", "w1", "b1", "w2", "b2")]
        out = few(l["x"])
        assert torch.equal(out, ops.moe_forward_few(*args, 2) if T <= 32 else ops.moe_forward(*args, 2))
        assert torch.equal(any_size(l["x"]), ops.moe_forward(*args, 2))
    limited = _mlp(l, 2, few_tokens=32, capacity_factor=1.0)
    with torch.no_grad():
        assert torch.equal(limited(l["x"]), ops.moe_forward(*args, 2, -(-2 * T // 8)))
    for m in (few, any_size, limited):
        m.close()


def test_a_block_in_a_graph():
    """norm -> layer in 8 bits, captured once and replayed on new inputs between eager calls."""
    l = _layer(24, 256, 512, 8, 2, seed=100)
    mlp = _mlp(l, 2, pre_norm=True).quantize_experts()
    x = l["x"].clone()
    with torch.no_grad():
        mlp(x)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = mlp(x)
        for i in range(4):
            x.copy_(l["x"].roll(i, 0) * (1 + i))
            graph.replay()
            torch.cuda.synchronize()
            got = out.clone()
            assert torch.equal(got, mlp(x.clone()))
    mlp.close()


def test_module_refusals():
    from ccfuser_amd.mix_moe import MixMOETransformerMLP
    l = _layer(2, 64, 64, 2, 1)
    with pytest.raises(ValueError, match="few_tokens"):
        _mlp(l, 1, few_tokens=33)
    staged = _mlp(l, 1, fused=False)
    with pytest.raises(ValueError, match="fused"):
        staged.quantize_experts()
    staged.close()


@pytest.mark.parametrize("form", [0, 1, 4])
@pytest.mark.parametrize("rows,k,n", [(1, 2048, 512), (16, 4096, 136), (5, 2080, 264), (16, 48, 8), (17, 2048, 64), (1, 144, 1000)])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
def test_product_of_rows_in_16_bits(form, rows, k, n, dt):
    """The codes that a product makes of its rows are those of ``quantize_rows``, so the results are the same bits; rows of
    zeros, subnormals, infinities and NaN, and a view that is not 16-byte aligned, among them."""
    from ccfuser_amd import ops
    g = torch.Generator().manual_seed(rows + k)
    x = torch.randn(rows * k + 1, generator=g)
    x[: k // 2] *= 2.0 ** -20
    w, s = ops.quantize_weight(torch.randn(n, k, generator=g).cuda())
    out = torch.bfloat16 if dt == torch.float32 else None
    ops.set_option("fp8_form", form)
    try:
        for at in (0, 1):
            v = x.to(dt).cuda()[at:at + rows * k].view(rows, k)
            for special in (None, 0.0, float("inf"), float("nan")):
                if special is not None:
                    v = v.clone() if at == 0 else v
                    v[rows // 2, k // 2] = special
                want = ops.linear_fp8(ops.quantize_rows(v), w, s, dtype=out or dt)
                got = ops.linear_fp8(v, w, s, dtype=out)
                assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())
    finally:
        ops.set_option("fp8_form", 0)


def test_product_of_no_rows():
    from ccfuser_amd import ops
    w, s = ops.quantize_weight(torch.randn(64, 128).half().cuda())
    x = torch.empty(0, 128, dtype=torch.float16, device="cuda")
    for rows in (x, ops.quantize_rows(x)):
        assert ops.linear_fp8(rows, w, s).shape == (0, 64)
    l = _layer(1, 64, 64, 2, 1)
    q = [t for n in ("w1", "w2") for t in ops.quantize_weight(l[n])]
    none = l["x"][:0]
    assert ops.moe_forward_few(none, *list(l.values())[1:], 1).shape == (0, 64)
    assert ops.moe_forward_fp8(none, l["wg"], l["bg"], q[0], q[1], l["b1"], q[2], q[3], l["b2"], 1).shape == (0, 64)


def test_two_products_at_once():
    """Calls on two streams share nothing: each result is the one that the call gives alone."""
    from ccfuser_amd import ops
    g = torch.Generator().manual_seed(3)
    w, s = ops.quantize_weight(torch.randn(2048, 2048, generator=g).half().cuda())
    xs = [torch.randn(r, 2048, generator=g).half().cuda() for r in (3, 16, 40, 700)]
    l = _layer(9, 256, 512, 8, 2, seed=120)
    args = [l[n] for n in ("x", "wg", "bg", "w1", "b1", "w2", "b2")]
    alone = [ops.linear_fp8(x, w, s) for x in xs] + [ops.moe_forward_few(*args, 2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = []
        for i in range(5):
            with torch.cuda.stream(streams[i % 2]):
                got.append(ops.linear_fp8(xs[i], w, s) if i < 4 else ops.moe_forward_few(*args, 2))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, alone))


def test_norm_is_differentiable_once():
    """A graph of the backward may be asked for, and what it holds of the norm is refused, not taken for a constant."""
    from ccfuser_amd.mix_moe import rms_norm
    x = torch.randn(4, 64).half().cuda().requires_grad_()
    w = torch.ones(64).half().cuda().requires_grad_()
    y = rms_norm(x, w)
    g = torch.randn_like(y).requires_grad_()
    plain = torch.autograd.grad(y, (x, w), g, retain_graph=True)
    first = torch.autograd.grad(y, (x, w), g, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(plain, first))
    with pytest.raises(RuntimeError, match="once_differentiable"):
        first[0].sum().backward()
