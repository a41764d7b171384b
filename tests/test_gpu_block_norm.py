"""kernels.moe.block_norm, block_norm_add and mul_merge_k_norm_add, forward and backward, against the definition in 64 bits."""
import itertools

import pytest
import torch

from fast_moe_amd.kernels import moe
from fast_moe_amd.kernels.hip import ops

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
HALF_STEP = {BF16: 2.0 ** -8, F32: 2.0 ** -24}      # the most that one rounding moves a value by, relative to it
# fp32 inside: sums of up to 8192 terms as trees (at most 8 in a lane, 6 steps in a wave, 16 waves), products of a dozen factors, each within a few
# 2^-24; a sum over rows takes up to 300 steps of that.  512 * 2^-24 of the sum of magnitudes bounds them all.
SUMS = 2.0 ** -15
EPS = 1e-6


def make(T, D, dtype, norm="rms", gate="none", K=0, param_dtype=None, after=True, nxt=True, scale="tensor", seed=0):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s, scale=1.0, dt=dtype: (torch.randn(*s, generator=g) * scale).to(dt).cuda()
    pd = param_dtype or dtype
    p = {"y": rnd(T * max(1, K), D, scale=2.0) + 0.25, "residual": rnd(T, D)}
    if after:
        p["weight"] = (1 + rnd(D, scale=0.2, dt=F32)).to(pd)
    if nxt:
        p["next_weight"] = (1 + rnd(D, scale=0.2, dt=F32)).to(pd)
    if norm == "layer":
        if after:
            p["bias"] = rnd(D, scale=0.3, dt=pd)
        if nxt:
            p["next_bias"] = rnd(D, scale=0.3, dt=pd)
    if gate != "none":
        p["gate"] = rnd(*{"token": (T, 1), "token1d": (T,), "element": (T, D)}[gate])
    if scale == "tensor":
        p["scale"] = rnd(D, scale=0.7, dt=pd)
    merge = None
    if K:
        order = torch.randperm(T * K, generator=g)
        merge = {"gate_index": order.cuda(), "index": (order // K).cuda(), "reverse": torch.argsort(order).view(T, K).sort(dim=1).values.cuda()}
        p["merge"] = (torch.rand(T, K, generator=g) + 0.1).to(dtype).cuda()
    return p, merge


def call(p, merge, norm, sigmoid, scale=None):
    kw = dict(weight=p.get("weight"), bias=p.get("bias"), gate=p.get("gate"), gate_sigmoid=sigmoid, scale=p.get("scale", scale),
              next_weight=p.get("next_weight"), next_bias=p.get("next_bias"), eps=EPS, norm=norm)
    if merge:
        return moe.mul_merge_k_norm_add(merge["index"], merge["reverse"], p["y"], p["residual"], p.get("merge"), merge["gate_index"], **kw)
    return moe.block_norm_add(p["y"], p["residual"], **kw)


def formula(p, merge, norm, sigmoid, d_out=None, d_next=None, scale=None):
    """-> {name: (value, sum of the magnitudes it is made of)} in 64 bits, gradients (by operand) among them."""
    v = {n: t.detach().double().cpu() for n, t in p.items()}
    layer = norm == "layer"
    mean = lambda a: a.mean(dim=1, keepdim=True)
    T, D = v["residual"].shape
    y, my = v["y"], v["y"].abs()
    if merge:
        idx, tok = merge["gate_index"].cpu(), merge["index"].cpu()
        share = v["merge"].flatten()[idx][:, None]
        y = torch.zeros(T, D, dtype=torch.float64).index_add_(0, tok, v["y"] * share)
        my = torch.zeros(T, D, dtype=torch.float64).index_add_(0, tok, v["y"].abs() * share)
    one = torch.ones(1, 1, dtype=torch.float64)

    def unit(a, ma):
        m = mean(a) if layer else 0 * one
        r = 1 / torch.sqrt(mean((a - m) ** 2) + EPS)
        return (a - m) * r, r, (ma + mean(ma) * layer) * r      # (value, reciprocal, magnitude)

    def back(d, md, a, r):
        return (r * (d - a * mean(d * a) - mean(d) * layer), r * (md + a.abs() * mean(md * a.abs()) + mean(md) * layer))

    w, b = v.get("weight", one), v.get("bias", 0 * one)
    a, ra, ma = unit(y, my) if "weight" in v else (y, one, my)
    z, mz = a * w + b, ma * w.abs() + b.abs()
    gate = one
    if "gate" in v:
        gate = v["gate"].reshape(T, -1)
        gate = torch.sigmoid(gate) if sigmoid else gate
    s = v.get("scale", one * (1 if scale is None else scale))
    out, mo = v["residual"] + s * gate * z, v["residual"].abs() + (s * gate).abs() * mz
    res = {"out": (out, mo)}
    bb = None
    if "next_weight" in v:
        bb, rb, mb = unit(out, mo)
        nb = v.get("next_bias", 0 * one)
        res["next"] = (bb * v["next_weight"] + nb, mb * v["next_weight"].abs() + nb.abs())
    if d_out is None and d_next is None:
        return res
    d = md = torch.zeros(T, D, dtype=torch.float64)
    if d_out is not None:
        d = d_out.double().cpu()
        md = d.abs()
    if d_next is not None and bb is not None:
        dn = d_next.double().cpu()
        e, me = back(dn * v["next_weight"], (dn * v["next_weight"]).abs(), bb, rb)
        d, md = d + e, md + me * (mb.abs() + 1) / (bb.abs() + 1)
        res["d_next_weight"], res["d_next_bias"] = ((dn * bb).sum(0), (dn.abs() * mb).sum(0)), (dn.sum(0), dn.abs().sum(0))
    dz, mdz = d * s * gate, md * (s * gate).abs()
    da, mda = dz * w, mdz * w.abs()
    dy, mdy = back(da, mda, a, ra) if "weight" in v else (da, mda)
    dg, mdg = d * s * z, md * s.abs() * mz
    if sigmoid:
        dg, mdg = dg * gate * (1 - gate), mdg * gate
    if "gate" in v and v["gate"].numel() != T * D:
        dg, mdg = dg.sum(dim=1), mdg.sum(dim=1)
    res.update(d_residual=(d, md), d_weight=((dz * a).sum(0), (mdz * ma).sum(0)), d_bias=(dz.sum(0), mdz.sum(0)),
               d_scale=((d * gate * z).sum(0), (md * gate.abs() * mz).sum(0)), d_gate=(dg, mdg), d_y=(dy, mdy))
    if merge:
        rows, mrows = dy[tok], mdy[tok]
        flat, mflat = torch.empty(len(idx), dtype=torch.float64), torch.empty(len(idx), dtype=torch.float64)
        flat[idx], mflat[idx] = (rows * v["y"]).sum(1), (mrows * v["y"].abs()).sum(1)
        res.update(d_y=(rows * share, mrows * share), d_merge=(flat, mflat))
    return res


def close(what, got, want, rounded=0.0):
    """``rounded``: what operands that were rounded on the way (the merged rows kept for the backward pass, their gradients) may add."""
    value, magnitude = want
    got = got.detach()
    bound = HALF_STEP[got.dtype] * value.abs() + (SUMS + rounded) * magnitude + 1e-30
    err = (got.double().cpu().reshape(value.shape) - value).abs()
    assert (err <= bound).all(), f"{what}: {int((err > bound).sum())} of {err.numel()} off, worst {(err / bound).max():.3g} of the bound"


SIZES = [(1, 1), (1, 8), (3, 7), (5, 64), (2, 512), (7, 520), (33, 1001), (4, 2048), (9, 4096), (2, 4100), (3, 8192), (300, 96), (5000, 24)]


@pytest.mark.parametrize("T,D", SIZES)
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("norm,gate,sigmoid", [("rms", "none", False), ("layer", "token", True), ("rms", "element", True), ("layer", "element", False),
                                               ("rms", "token1d", False)])
def test_block_norm_add_forward_and_backward(T, D, dtype, norm, gate, sigmoid):
    p, _ = make(T, D, dtype, norm, gate, seed=T + D)
    plain = call(p, None, norm, sigmoid)
    for t in p.values():
        t.requires_grad_(True)
    out, nxt = call(p, None, norm, sigmoid)
    assert torch.equal(out, plain[0]) and torch.equal(nxt, plain[1])
    d_out, d_next = (torch.randn(T, D, device="cuda").to(dtype) for _ in range(2))
    torch.autograd.backward((out, nxt), (d_out, d_next))
    want = formula(p, None, norm, sigmoid, d_out, d_next)
    close("out", out, want["out"])
    close("next", nxt, want["next"])
    for n, t in p.items():
        assert t.grad.shape == t.shape and t.grad.dtype == t.dtype
        close("d_" + n, t.grad, want["d_" + n])


@pytest.mark.parametrize("T,D,K", [(1, 64, 1), (4, 100, 2), (37, 2048, 8), (3, 1001, 3), (130, 72, 5), (2, 8192, 64)])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("norm,gate", [("rms", "none"), ("layer", "token")])
def test_merged_rows_forward_and_backward(T, D, K, dtype, norm, gate):
    p, merge = make(T, D, dtype, norm, gate, K=K, seed=T + D)
    plain = call(p, merge, norm, True)
    for t in p.values():
        t.requires_grad_(True)
    out, nxt = call(p, merge, norm, True)
    assert torch.equal(out, plain[0]) and torch.equal(nxt, plain[1])
    d_out, d_next = (torch.randn(T, D, device="cuda").to(dtype) for _ in range(2))
    torch.autograd.backward((out, nxt), (d_out, d_next))
    want = formula(p, merge, norm, True, d_out, d_next)
    close("out", out, want["out"])
    close("next", nxt, want["next"])
    # the merged rows and their gradients are kept in the rows' dtype: a rounding each (the merge weights' gradients take the second times
    # the rows, and round every product)
    for n, t in p.items():
        close("d_" + n, t.grad, want["d_" + n], rounded=4 * HALF_STEP[dtype])


@pytest.mark.parametrize("after,nxt,scale", list(itertools.product((True, False), (True, False), ("tensor", 0.5, None))))
def test_parts_left_out(after, nxt, scale):
    T, D = 6, 200
    p, _ = make(T, D, F32, "layer", "token", after=after, nxt=nxt, scale=scale, seed=3)
    for t in p.values():
        t.requires_grad_(True)
    number = None if scale == "tensor" else scale
    out, normed = call(p, None, "layer", True, number)
    assert (normed is None) == (not nxt)
    d_out, d_next = (torch.randn(T, D, device="cuda") for _ in range(2))
    torch.autograd.backward((out, normed) if nxt else (out,), (d_out, d_next) if nxt else (d_out,))
    want = formula(p, None, "layer", True, d_out, d_next if nxt else None, scale=number)
    close("out", out, want["out"])
    for n, t in p.items():
        close("d_" + n, t.grad, want["d_" + n])


@pytest.mark.parametrize("which", ["out", "next"])
def test_only_one_output_is_used(which):
    T, D = 5, 96
    p, _ = make(T, D, F32, "rms", "element", seed=4)
    for t in p.values():
        t.requires_grad_(True)
    out, nxt = call(p, None, "rms", True)
    d = torch.randn(T, D, device="cuda")
    (out if which == "out" else nxt).backward(d)
    want = formula(p, None, "rms", True, d if which == "out" else None, d if which == "next" else None)
    for n, t in p.items():
        if which == "out" and n.startswith("next"):
            assert t.grad is None or not t.grad.any()
        else:
            close("d_" + n, t.grad, want["d_" + n])


@pytest.mark.parametrize("T,D", [(1, 5), (4, 128), (65, 1000), (3, 8192)])
@pytest.mark.parametrize("dtype,param", [(BF16, BF16), (BF16, F32), (F32, F32)])
@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_block_norm(T, D, dtype, param, norm):
    g = torch.Generator().manual_seed(D)
    x = (torch.randn(T, D, generator=g) + 0.5).to(dtype).cuda().requires_grad_(True)
    w = (1 + 0.2 * torch.randn(D, generator=g)).to(param).cuda().requires_grad_(True)
    b = (0.2 * torch.randn(D, generator=g)).to(param).cuda().requires_grad_(True) if norm == "layer" else None
    got = moe.block_norm(x, w, b, eps=EPS, norm=norm)
    d = torch.randn(T, D, device="cuda").to(dtype)
    got.backward(d)
    p = {"y": torch.zeros_like(x), "residual": x, "next_weight": w, **({} if b is None else {"next_bias": b})}
    want = formula(p, None, norm, False, None, d)
    close("next", got, want["next"])
    close("d_x", x.grad, want["d_residual"])
    close("d_weight", w.grad, want["d_next_weight"])
    if b is not None:
        close("d_bias", b.grad, want["d_next_bias"])


@pytest.mark.parametrize("param", [F32, BF16])
def test_parameters_of_another_dtype_and_strided_operands(param):
    T, D = 9, 256
    p, _ = make(T, D, BF16, "layer", "element", param_dtype=param, seed=8)
    want = call(p, None, "layer", True)
    w64 = formula(p, None, "layer", True)
    close("out", want[0], w64["out"])
    close("next", want[1], w64["next"])
    wide = torch.zeros(T, 3 * D + 8, dtype=BF16, device="cuda")
    wide[:, :D], wide[:, D:2 * D], wide[:, 2 * D:3 * D] = p["y"], p["residual"], p["gate"]
    q = dict(p, y=wide[:, :D], residual=wide[:, D:2 * D], gate=wide[:, 2 * D:3 * D])
    got = call(q, None, "layer", True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    odd = torch.zeros(T, D + 3, dtype=BF16, device="cuda")           # rows at odd addresses
    odd[:, 1:D + 1] = p["y"]
    got = call(dict(p, y=odd[:, 1:D + 1]), None, "layer", True)
    close("out", got[0], w64["out"])
    turned = dict(p, y=p["y"].t().contiguous().t(), residual=p["residual"].t().contiguous().t())
    got = call(turned, None, "layer", True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_gradients_against_differences():
    """Directional derivatives of the 64-bit formula's forward pass by central differences (error h^2) against the gradients."""
    T, D = 4, 48
    for K in (0, 3):
        p, merge = make(T, D, F32, "layer", "element", K=K, seed=20 + K)
        for t in p.values():
            t.requires_grad_(True)
        out, nxt = call(p, merge, "layer", True)
        d_out, d_next = (torch.randn(T, D, device="cuda") for _ in range(2))
        torch.autograd.backward((out, nxt), (d_out, d_next))
        loss = lambda q: ((formula(q, merge, "layer", True)["out"][0] * d_out.double().cpu()).sum()
                          + (formula(q, merge, "layer", True)["next"][0] * d_next.double().cpu()).sum())
        for n, t in p.items():
            direction, h = torch.randn(t.shape, dtype=torch.float64), 1e-4
            moved = lambda sign: {**{m: u.detach().double().cpu() for m, u in p.items()}, n: t.detach().double().cpu() + sign * h * direction}
            slope = (loss(moved(1)) - loss(moved(-1))) / (2 * h)
            got = (t.grad.double().cpu() * direction).sum()
            scale = (t.grad.double().cpu() * direction).abs().sum()
            assert (got - slope).abs() <= 1e-5 * scale + 1e-6, (n, K, got, slope)


def test_rows_of_zeros_and_what_is_not_finite():
    p, _ = make(6, 128, BF16, "rms", "none", seed=1)
    p["y"][2] = 0
    p["residual"][2] = 0
    clean = call(p, None, "rms", False)
    assert not clean[0][2].any() and not clean[1][2].any()
    p["y"][4, 7] = float("inf")
    got = call(p, None, "rms", False)
    rest = torch.arange(6) != 4
    assert torch.equal(got[0][rest], clean[0][rest]) and torch.equal(got[1][rest], clean[1][rest]) and not got[0][4].isfinite().all()


def test_no_rows():
    p, _ = make(0, 64, BF16, "layer", "token")
    for t in p.values():
        t.requires_grad_(True)
    out, nxt = call(p, None, "layer", True)
    assert out.shape == nxt.shape == (0, 64)
    (out.sum() + nxt.sum()).backward()
    assert not p["weight"].grad.any() and p["y"].grad.shape == (0, 64)


def test_merge_leaves_out_rows_that_are_not_there():
    p, merge = make(5, 64, F32, "rms", "none", K=3, seed=2)
    merge["reverse"][1, 2] = -1                              # a slot that no row names
    merge["reverse"][3] = -1                                 # a token without any
    row = torch.ones(15, dtype=torch.bool)
    with torch.no_grad():
        got = call(p, merge, "rms", False)
        y = ops.combine(p["y"], merge["reverse"], p["merge"], merge["gate_index"])
    alone = moe.block_norm_add(y, p["residual"], weight=p["weight"], scale=p["scale"], next_weight=p["next_weight"], eps=EPS)
    assert (got[0] - alone[0]).abs().max() <= 1e-5 and (got[1] - alone[1]).abs().max() <= 1e-5      # (another order of sums)
    assert torch.equal(got[0][3], p["residual"][3])


def test_same_bits_each_time_and_from_a_graph():
    T, D = 700, 1024
    p, _ = make(T, D, BF16, "rms", "token", seed=11)
    d_out, d_next = (torch.randn(T, D, device="cuda").to(BF16) for _ in range(2))
    args = ops.NormArgs(p["weight"], None, p["gate"], True, p["scale"], p["next_weight"])
    need = {n: True for n in ("y", "residual", "gate", "scale", "weight", "next_weight")}

    def both():
        out, nxt, _, stats = ops.norm_add(p["y"], p["residual"], args, for_backward=True)
        return [out, nxt, *(t for t in ops.norm_add_bwd(p["y"], p["residual"], args, stats, d_out, d_next, need).values() if t is not None)]
    want = both()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(both(), want))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    for seed in (1, 2, 3):
        p["y"].copy_(make(T, D, BF16, seed=seed)[0]["y"])
        want = both()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals():
    p, merge = make(4, 64, BF16, "layer", "token", K=2)
    ok = dict(weight=p["weight"], bias=p["bias"], scale=p["scale"])
    y, r = p["y"][:4], p["residual"]
    for bad, match in ((dict(y=y[:3]), "y must be"), (dict(y=y.float()), "y must be"), (dict(weight=p["weight"][:32]), r"weight must be \[64\]"),
                       (dict(weight=p["weight"].float()), "one dtype"), (dict(weight=None), "goes with its weight"), (dict(norm="batch"), "norm must be"),
                       (dict(gate=p["gate"][:3]), "gate must be"), (dict(gate=p["gate"].float()), "gate must be"),
                       (dict(residual=r.cpu()), "GPU")):
        kw = dict(ok, **{k: v for k, v in bad.items() if k not in ("y", "residual")})
        with pytest.raises(ValueError, match=match):
            moe.block_norm_add(bad.get("y", y), bad.get("residual", r), **kw)
    big = torch.zeros(1, 8193, dtype=BF16, device="cuda")
    with pytest.raises(ValueError, match="8192 columns"):
        moe.block_norm_add(big, big)
    with pytest.raises(NotImplementedError, match="bf16 or fp32"):
        moe.block_norm_add(y.half(), r.half())
    with pytest.raises(AssertionError, match="mul_merge_k_norm_add"):
        moe.mul_merge_k_norm_add(merge["index"][:7], merge["reverse"], p["y"], r)
    with pytest.raises(NotImplementedError, match="not available"):
        moe.block_norm(r, p["weight"], kernel=moe.KernelType.PYTORCH)


@pytest.mark.parametrize("T,D", [(3, 7), (5, 64), (4, 2048), (3, 8192)])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("gate", ["none", "token", "element"])
def test_rms_norm_with_biases(T, D, dtype, gate):
    p, _ = make(T, D, dtype, "layer", gate, seed=T + D + 1)         # (both biases, which "rms" takes as well)
    for t in p.values():
        t.requires_grad_(True)
    out, nxt = call(p, None, "rms", False)
    d_out, d_next = (torch.randn(T, D, device="cuda").to(dtype) for _ in range(2))
    torch.autograd.backward((out, nxt), (d_out, d_next))
    want = formula(p, None, "rms", False, d_out, d_next)
    close("out", out, want["out"])
    close("next", nxt, want["next"])
    for n, t in p.items():
        close("d_" + n, t.grad, want["d_" + n])


def test_gradients_against_differences():
    T, D, step = 3, 24, 2.0 ** -6
    p, _ = make(T, D, F32, "layer", "element", seed=11)
    g = torch.Generator().manual_seed(12)
    d_out, d_next = (torch.randn(T, D, generator=g).cuda() for _ in range(2))
    for t in p.values():
        t.requires_grad_(True)
    torch.autograd.backward(call(p, None, "layer", True), (d_out, d_next))
    for n, t in p.items():
        direction = torch.randn(t.shape, generator=g).cuda()

        def loss(by):
            out, nxt = call({m: (v + by * direction if m == n else v).detach() for m, v in p.items()}, None, "layer", True)
            return ((out.double() * d_out).sum() + (nxt.double() * d_next).sum()).item()

        slope = (8 * (loss(step) - loss(-step)) - (loss(2 * step) - loss(-2 * step))) / (12 * step)      # error of step^4 = 2^-24 of the fifth derivative
        want = (t.grad.double() * direction).sum().item()
        # values of a few units in fp32, 150 of them, differences over 2^-6: 2^-24 * 4 * 12 * 64 of noise; the fifth derivative of a norm or sigmoid of
        # such rows is within a few hundred
        assert abs(slope - want) <= 2e-3 * (1 + abs(want)), (n, slope, want)


def test_no_rows_strided_operands_and_no_second_derivative():
    p, _ = make(1, 64, F32, "layer", "token", seed=1)
    p = {n: (t if t.ndim == 1 else t[:0]).detach().requires_grad_(True) for n, t in p.items()}
    out, nxt = call(p, None, "layer", False)
    torch.autograd.backward((out, nxt), (torch.ones_like(out), torch.ones_like(nxt)))
    assert out.shape == nxt.shape == (0, 64) and all(t.grad.shape == t.shape and not t.grad.any() for t in p.values())

    T, D, K = 5, 96, 2
    p, merge = make(T, D, BF16, "layer", "element", K=K, seed=2)
    wide = {n: torch.zeros(t.shape[0], t.shape[1] + 7, dtype=t.dtype, device="cuda") for n, t in p.items() if n in ("y", "residual", "gate")}
    for n in wide:
        wide[n][:, 3:-4] = p[n]
    views = {n: wide[n][:, 3:-4] if n in wide else t for n, t in p.items()}
    views["weight"] = torch.stack((p["weight"], p["weight"]), dim=1)[:, 0]
    got, grads = [], []
    for q in (p, views):
        leaves = {n: t.detach().requires_grad_(True) for n, t in q.items()}
        o = call(leaves, merge, "layer", True)
        torch.autograd.backward(o, [torch.full_like(t, 0.5) for t in o])
        got.append(o)
        grads.append([t.grad for t in leaves.values()])
    assert all(torch.equal(a, b) for a, b in zip(*got)) and all(torch.equal(a, b) for a, b in zip(*grads))

    x = torch.randn(4, 64, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    grad, = torch.autograd.grad(moe.block_norm(x, w).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):       # (never a gradient of a gradient that leaves a part of it out)
        grad.sum().backward()


@pytest.mark.parametrize("T,D,K", [(5, 1001, 3), (9, 2048, 8), (3, 4100, 2)])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("norm,sigmoid", [("rms", True), ("layer", False)])
def test_merged_rows_with_a_gate_for_each_element(T, D, K, dtype, norm, sigmoid):
    p, merge = make(T, D, dtype, norm, "element", K=K, param_dtype=F32, seed=T + D)
    for t in p.values():
        t.requires_grad_(True)
    out, nxt = call(p, merge, norm, sigmoid)
    d_out, d_next = (torch.randn(T, D, device="cuda").to(dtype) for _ in range(2))
    torch.autograd.backward((out, nxt), (d_out, d_next))
    want = formula(p, merge, norm, sigmoid, d_out, d_next)
    close("out", out, want["out"])
    close("next", nxt, want["next"])
    for n, t in p.items():      # (the merged rows and their gradients rounded to the rows' dtype)
        close("d_" + n, t.grad, want["d_" + n], rounded=4 * HALF_STEP[dtype])


@pytest.mark.parametrize("T,D,K", [(17, 256, 2), (5, 1001, 3), (40, 2048, 8), (3, 6000, 2)])
@pytest.mark.parametrize("norm,gate", [("rms", "none"), ("layer", "element")])
def test_nothing_is_rounded_between_the_merge_and_its_gradients(T, D, K, norm, gate):
    # the merge weights' gradients are sums that cancel (the gradient of a normed row is at right angles to it): bf16 rounds them once, at the end
    p, merge = make(T, D, BF16, norm, gate, K=K, seed=T + D)
    for t in p.values():
        t.requires_grad_(True)
    d_out, d_next = (torch.randn(T, D, device="cuda").to(BF16) for _ in range(2))
    torch.autograd.backward(call(p, merge, norm, True), (d_out, d_next))
    want = formula(p, merge, norm, True, d_out, d_next)
    for n, t in p.items():
        close("d_" + n, t.grad, want["d_" + n])
