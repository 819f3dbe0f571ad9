"""Timing cases of the operators around a MoE layer in 8 bits: what a program that serves or trains such a block calls.

Five paths:

``norm``    root-mean-square norm with the residual's addition; the result in 16 bits for the router and in 8 bits with a
            scale for each block of 128 for the experts (serving)
``train``   the same norm without the 8-bit output, forward and backward
``linear``  a dense product in 8-bit floating point: activations of 16 bits that the call quantises by rows and blocks of
            128 (their scales are powers of two, so that codes of 16-bit values are exact), weights that the program holds
            in 8 bits with any scale for each 128 x 128 block
``layer8``  the whole MoE layer on experts in 8 bits
``few``     the whole MoE layer for a few tokens on experts in 16 bits

``listed()`` are fixed cases, ``draw()`` makes more of the same ranges.  Widths are the repository's own
(``ccfuser_amd/workloads.py``) and generic ones.
"""
import math

import torch

own = False

BLOCK = 128                  # elements that share a scale
FP8_MAX = 448.0              # largest finite value of e4m3
EPS = 1e-5
_TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _norm(name, kind, rows, d, dtype):
    c = {"kind": kind, "rows": rows, "d": d, "dtype": dtype}
    return dict(c, name=name) if name else c


def _linear(name, rows, k, n, dtype, bias):
    c = {"kind": "linear", "rows": rows, "d": k, "f": n, "dtype": dtype, "bias": bias}
    return dict(c, name=name) if name else c


def _layer(name, kind, rows, d, f, experts, top_k):
    c = {"kind": kind, "rows": rows, "d": d, "f": f, "experts": experts, "top_k": top_k}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one token being decoded, in front of the router and the experts: a launch and a chain of loads
        _norm("norm_1", "norm", 1, 4096, "fp16"),
        # a full prefill batch of the repository's benchmark: bytes
        _norm("norm_4096", "norm", 4096, 4096, "fp16"),
        # a training step of a GPT-2 / BERT sized block on an odd number of tokens
        _norm("norm_train_1999", "train", 1999, 768, "fp16"),
        # a training step of a large block in bf16
        _norm("norm_train_16384", "train", 16384, 4096, "bf16"),
        # a dense layer beside the experts for one token: weight bytes
        _linear("linear_1", 1, 4096, 14336, "fp16", True),
        # a short prompt of odd length, a small layer
        _linear("linear_333", 333, 1024, 4096, "bf16", True),
        # a full prefill batch through a large dense layer: the matrix cores
        _linear("linear_8192", 8192, 4096, 14336, "fp16", False),
        # one token through a layer with experts in 8 bits: half the weight bytes of 16 bits
        _layer("layer8_1", "layer8", 1, 4096, 14336, 8, 2),
        # a short prompt of odd length through encoder-sized experts
        _layer("layer8_555", "layer8", 555, 1024, 4096, 8, 2),
        # the repository's benchmark shape in 8 bits
        _layer("layer8_4096", "layer8", 4096, 4096, 14336, 8, 2),
        # one token through experts in 16 bits
        _layer("few_1", "few", 1, 4096, 14336, 8, 2),
        # a small decoding batch through smaller experts
        _layer("few_13", "few", 13, 2048, 8192, 8, 2),
    ]


_MODELS = ((256, 1024), (768, 2048), (1024, 4096), (2048, 8192), (4096, 14336))
_MAX_NORM = 16384 * 4096                    # elements of the largest norm
_MAX_LINEAR = 8192 * 4096 * 14336           # products of the largest dense layer
_MAX_ROUTED = 2 * 4096 * 4096 * 14336       # products of one of the largest layer's two matrices


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("norm", "train", "linear", "layer8", "few"))
    if kind in ("norm", "train"):
        d = rng.choice((rng.choice((256, 768, 1024, 2048, 4096)), _log_int(rng, 65, 8192), 8 * _log_int(rng, 16, 1024)))
        rows = _log_int(rng, 1, min(32768, _MAX_NORM // d))
        return _norm(None, kind, rows, d, rng.choice(("fp16", "bf16", "fp16", "bf16", "fp32")))
    if kind == "linear":
        k = rng.choice((256, 768, 1024, 4096, 16 * _log_int(rng, 16, 512)))
        n = rng.choice((1024, 2048, 4096, 14336, 8 * _log_int(rng, 32, 1792)))
        rows = _log_int(rng, 1, min(8192, _MAX_LINEAR // (k * n)))
        return _linear(None, rows, k, n, rng.choice(("fp16", "bf16")), rng.random() < 0.5)
    if rng.random() < 0.4:
        d, f = rng.choice(_MODELS)
    else:                                                   # any multiple of 64
        d = 64 * _log_int(rng, 4, 64)
        f = 64 * int(round(d * rng.uniform(2.0, 3.5) / 64))
    experts = rng.choice((4, 8, 8, 16, 32))
    while experts * d * f > 8 * 4096 * 14336:
        experts //= 2
    top_k = rng.choice((1, 2, 2, 3))
    if kind == "few":
        return _layer(None, kind, rng.randint(1, 32), d, f, experts, top_k)
    rows = _log_int(rng, 1, min(8192, _MAX_ROUTED // (d * f * top_k)))
    return _layer(None, kind, rows, d, f, experts, top_k)


# ---------------------------------------------------------------- inputs
def _blocks(t):
    """t [..., R, K] as [..., R, K / 128, 128], the last block filled with zeros."""
    pad = -t.shape[-1] % BLOCK
    return torch.nn.functional.pad(t, (0, pad)).unflatten(-1, (-1, BLOCK))


def _weight_in_8_bits(w):
    """(codes, scales) of a weight [..., N, K]: a scale for each 128 x 128 block, as a checkpoint in 8 bits holds them."""
    n, k = w.shape[-2:]
    tiles = _blocks(torch.nn.functional.pad(w, (0, 0, 0, -n % BLOCK))).unflatten(-3, (-1, BLOCK))      # [..., nb, 128, kb, 128]
    scale = (tiles.abs().amax(dim=(-3, -1)).float() / FP8_MAX).clamp_min(1e-30)
    codes = (tiles / scale[..., :, None, :, None]).to(torch.float8_e4m3fn)
    return codes.flatten(-2).flatten(-3, -2)[..., :n, :k].contiguous(), scale


class _Maker:
    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda").manual_seed(seed)

    def randn(self, *shape, std=1.0, dtype=torch.float16):
        return torch.empty(*shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=self.gen)


def prepare(case, seed):
    mk = _Maker(seed)
    kind, rows, d = case["kind"], case["rows"], case["d"]
    st = {"kind": kind, "case": case}
    if kind in ("norm", "train"):
        dt = _TYPES[case["dtype"]]
        # a residual stream is several times wider than what a block adds to it, and some of its channels far more
        wide = 1.0 + 15.0 * (torch.rand(d, generator=mk.gen, device="cuda") < 0.01).float()
        st["x"] = mk.randn(rows, d, dtype=dt)
        st["residual"] = (mk.randn(rows, d, std=3.0, dtype=torch.float32) * wide).to(dt)
        st["w"] = (1.0 + mk.randn(d, std=0.1, dtype=torch.float32)).to(dt)
        if kind == "train":
            for n in ("x", "residual", "w"):
                st[n].requires_grad_(True)
            st["grad_y"] = mk.randn(rows, d, std=0.1, dtype=dt)
            st["grad_total"] = mk.randn(rows, d, std=0.1, dtype=dt)
        return st
    f = case["f"]
    if kind == "linear":
        dt = _TYPES[case["dtype"]]
        st["x"] = mk.randn(rows, d, dtype=dt)
        st["wq"], st["ws"] = _weight_in_8_bits(mk.randn(f, d, std=0.02))
        st["bias"] = mk.randn(f, std=0.02, dtype=dt) if case["bias"] else None
        return st
    E = case["experts"]
    st["x"] = mk.randn(rows, d)
    st["wg"], st["bg"] = mk.randn(E, d, std=0.02), mk.randn(E, std=0.02)
    st["b1"], st["b2"] = mk.randn(E, f, std=0.02), mk.randn(E, d, std=0.02)
    if kind == "few":
        st["w1"], st["w2"] = mk.randn(E, f, d, std=0.02), mk.randn(E, d, f, std=0.02)
    else:
        st["w1q"], st["w1s"] = _weight_in_8_bits(mk.randn(E, f, d, std=0.02))
        st["w2q"], st["w2s"] = _weight_in_8_bits(mk.randn(E, d, f, std=0.02))
    return st


# ------------------------------------------------------------ plain forms
def _rows_in_8_bits(t):
    """(codes, scales) of rows [R, K] held in 32 bits: for each row and block of 128 the least power of two that leaves no
    value beyond 448 = 0.875 * 2^9."""
    b = _blocks(t)
    part, power = torch.frexp(b.abs().amax(-1))
    power = (power - 9 + (part > 0.875).int()).clamp_min(-126)
    scale = torch.ldexp(torch.ones_like(part), power)
    codes = torch.ldexp(b, -power[..., None]).to(torch.float8_e4m3fn)
    return codes.flatten(-2)[:, :t.shape[-1]], scale


def _values(codes, scale):
    """What codes of rows stand for, in 32 bits."""
    k = codes.shape[-1]
    return codes.float() * scale.repeat_interleave(BLOCK, -1)[..., :k]


def _weight_values(codes, scale):
    n = codes.shape[-2]
    return _values(codes, scale.repeat_interleave(BLOCK, -2)[..., :n, :])


def _through_8_bits(t):
    return _values(*_rows_in_8_bits(t))


def _gelu(v):
    return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))


def _choice(x, wg, bg, top_k):
    """Experts and weights of every token; logits are rounded to the input's type, ties go to the lowest expert."""
    logits = (x.float() @ wg.float().t() + bg.float()).to(x.dtype).float()
    value, idx = logits.sort(dim=-1, descending=True, stable=True)
    score = torch.softmax(value[:, :top_k], dim=-1).to(x.dtype).float()
    return idx[:, :top_k], score


def _experts(rows, owner, weight, bias):
    """rows[r] times the weight of expert owner[r] (an index into weight) and its bias; rows sorted by owner."""
    count = torch.bincount(owner, minlength=weight.shape[0])
    at = torch.arange(owner.numel(), device=owner.device) - (count.cumsum(0) - count)[owner]
    padded = rows.new_zeros(weight.shape[0], int(count.max()), rows.shape[1])
    padded[owner, at] = rows
    return torch.bmm(padded, weight.transpose(1, 2))[owner, at] + bias[owner]


def _plain_layer(st, in_8_bits):
    x, k = st["x"], st["case"]["top_k"]
    T = x.shape[0]
    idx, score = _choice(x, st["wg"], st["bg"], k)
    present, owner = idx.reshape(-1).unique(return_inverse=True)
    owner, order = owner.sort(stable=True)
    rows = (_through_8_bits(x.float()) if in_8_bits else x.float())[order // k]
    if in_8_bits:
        w1 = _weight_values(st["w1q"].view(torch.uint8)[present].view(torch.float8_e4m3fn), st["w1s"][present])
        w2 = _weight_values(st["w2q"].view(torch.uint8)[present].view(torch.float8_e4m3fn), st["w2s"][present])
    else:
        w1, w2 = st["w1"][present].float(), st["w2"][present].float()
    h = _gelu(_experts(rows, owner, w1, st["b1"][present].float()))
    y = _experts(_through_8_bits(h) if in_8_bits else h, owner, w2, st["b2"][present].float())
    flat = torch.empty_like(y)
    flat[order] = y
    return (flat.view(T, k, -1) * score[:, :, None]).sum(1).to(x.dtype)


def _plain_norm(x, residual, w):
    total = (x.float() + residual.float()).to(x.dtype)
    t = total.float()
    y = t * (t.square().mean(-1, keepdim=True) + EPS).rsqrt() * w.float()
    return total, y


def run(state):
    kind, case = state["kind"], state["case"]
    if own:
        return _own(state, kind, case)
    if kind == "norm":
        total, y = _plain_norm(state["x"], state["residual"], state["w"])
        codes, scale = _rows_in_8_bits(y)
        return {"y": y.to(total.dtype), "total": total, "codes": codes, "scale": scale}
    if kind == "train":
        x, residual, w = (state[n].detach().requires_grad_(True) for n in ("x", "residual", "w"))
        total, y = _plain_norm(x, residual, w)
        y = y.to(x.dtype)
        g = torch.autograd.grad((y, total), (x, residual, w), (state["grad_y"], state["grad_total"]))
        return {"y": y.detach(), "total": total.detach(), "x": g[0], "residual": g[1], "w": g[2]}
    if kind == "linear":
        y = _through_8_bits(state["x"].float()) @ _weight_values(state["wq"], state["ws"]).t()
        if state["bias"] is not None:
            y = y + state["bias"].float()
        return y.to(state["x"].dtype)
    return _plain_layer(state, kind == "layer8")


def _own(st, kind, case):
    from ccfuser_amd import ops
    if kind == "norm":
        n = ops.rms_norm(st["x"], st["w"], EPS, residual=st["residual"], want_fp8=True)
        return {"y": n.y, "total": n.total, "codes": n.codes, "scale": n.scale}
    if kind == "train":
        from ccfuser_amd.mix_moe import rms_norm
        y, total = rms_norm(st["x"], st["w"], EPS, residual=st["residual"])
        g = torch.autograd.grad((y, total), (st["x"], st["residual"], st["w"]), (st["grad_y"], st["grad_total"]))
        return {"y": y.detach(), "total": total.detach(), "x": g[0], "residual": g[1], "w": g[2]}
    if kind == "linear":
        return ops.linear_fp8(st["x"], st["wq"], st["ws"], st["bias"])
    if kind == "few":
        return ops.moe_forward_few(st["x"], st["wg"], st["bg"], st["w1"], st["b1"], st["w2"], st["b2"], case["top_k"])
    return ops.moe_forward_fp8(st["x"], st["wg"], st["bg"], st["w1q"], st["w1s"], st["b1"], st["w2q"], st["w2s"], st["b2"],
                               case["top_k"])


# ------------------------------------------------------------- 64 bits
def _exact_codes(t):
    """Codes and scales of rows in 64 bits, and what they stand for."""
    k = t.shape[1]
    full = torch.zeros(t.shape[0], (k + BLOCK - 1) // BLOCK * BLOCK, dtype=torch.float64, device=t.device)
    full[:, :k] = t
    full = full.view(t.shape[0], -1, BLOCK)
    top = full.abs().max(dim=2).values
    scale = torch.full_like(top, 2.0 ** -126)
    for p in range(-125, 121):                               # the least power of two with top / scale <= 448
        scale[top > FP8_MAX * 2.0 ** (p - 1)] = 2.0 ** p
    codes = (full / scale[:, :, None]).to(torch.float8_e4m3fn).double()
    return (codes.view(t.shape[0], -1)[:, :k], scale, (codes * scale[:, :, None]).view(t.shape[0], -1)[:, :k])


def _exact_weight(codes, scale):
    """A weight [N, K] from its codes and the scales of its 128 x 128 blocks."""
    n = torch.arange(codes.shape[0], device=codes.device) // BLOCK
    k = torch.arange(codes.shape[1], device=codes.device) // BLOCK
    return codes.double() * scale.double()[n][:, k]


def exact(case, seed):
    st = prepare(case, seed)
    kind, rows, d = case["kind"], case["rows"], case["d"]
    if kind in ("norm", "train"):
        if rows * d > (1 << 26):
            return None
        total = (st["x"].detach().double() + st["residual"].detach().double()).to(st["x"].dtype)
        t, w = total.double(), st["w"].detach().double()
        r = 1.0 / torch.sqrt((t * t).sum(1, keepdim=True) / d + EPS)
        y = t * r * w
        if kind == "norm":
            codes, scale, _ = _exact_codes(y)
            return {"y": y, "total": total.double(), "codes": codes, "scale": scale}
        g = st["grad_y"].double()
        gx = st["grad_total"].double() + r * (g * w - t * r * r * (g * w * t).sum(1, keepdim=True) / d)
        return {"y": y, "total": total.double(), "x": gx, "residual": gx, "w": (g * t * r).sum(0)}
    if kind == "linear":
        y = _exact_codes(st["x"].double())[2] @ _exact_weight(st["wq"], st["ws"]).T
        return y if st["bias"] is None else y + st["bias"].double()
    x, k = st["x"].double(), case["top_k"]
    logits = (x @ st["wg"].double().T + st["bg"].double()).to(torch.float16).double()
    out = torch.zeros(rows, d, dtype=torch.float64, device="cuda")
    # the k largest, one after the other, the lowest expert first among equals
    left, chosen, top = logits.clone(), [], None
    for _ in range(k):
        best = left.max(dim=1).values
        e = (left == best[:, None]).double().argmax(dim=1)
        chosen.append((e, best))
        left.scatter_(1, e[:, None], -math.inf)
    top = torch.stack([b for _, b in chosen], 1)
    score = torch.exp(top - top[:, :1])
    score = (score / score.sum(1, keepdim=True)).to(torch.float16).double()
    for e in range(case["experts"]):
        for s in range(k):
            mine = (chosen[s][0] == e).nonzero()[:, 0]
            if not mine.numel():
                continue
            if kind == "few":
                w1, w2, v = st["w1"][e].double(), st["w2"][e].double(), x[mine]
            else:
                w1, w2 = _exact_weight(st["w1q"][e], st["w1s"][e]), _exact_weight(st["w2q"][e], st["w2s"][e])
                v = _exact_codes(x[mine])[2]
            h = v @ w1.T + st["b1"][e].double()
            h = h * 0.5 * torch.special.erfc(-h / math.sqrt(2.0))
            if kind == "layer8":
                h = _exact_codes(h)[2]
            out[mine] += score[mine, s][:, None] * (h @ w2.T + st["b2"][e].double())
    return out


# ---------------------------------------------------------------- work
def work(case):
    """Inputs and touched weights read once, outputs written once; the products of the rows."""
    kind, rows, d = case["kind"], case["rows"], case["d"]
    if kind in ("norm", "train"):
        size, n = torch.finfo(_TYPES[case["dtype"]]).bits // 8, float(rows * d)
        if kind == "norm":
            return {"bytes": n * (4 * size + 1) + 4.0 * rows * ((d + BLOCK - 1) // BLOCK) + size * d, "flops": 6.0 * n}
        # forward: x, residual, y, total; backward: both gradients, total, and the one that x and residual share
        return {"bytes": 8.0 * n * size + 3.0 * size * d, "flops": 16.0 * n}
    f = case["f"]
    if kind == "linear":
        return {"bytes": 2.0 * rows * (d + f) + d * f + d * f / 4096.0, "flops": 2.0 * rows * d * f}
    E, k = case["experts"], case["top_k"]
    touched = E * (1.0 - (1.0 - k / E) ** rows)                     # experts that get a row, loads being even
    element = 2.0 if kind == "few" else 1.0
    return {"bytes": 4.0 * rows * d + 2.0 * E * d + touched * (2 * element * d * f + 2.0 * (d + f)),
            "flops": 4.0 * rows * k * d * f + 2.0 * rows * d * E}
