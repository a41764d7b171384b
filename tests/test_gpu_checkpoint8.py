"""SwiGLU pre-activations in 8 bits: the codes, what they stand for, and the backward pass on them, against the definitions in 64 bits."""
import pytest
import torch

from fast_moe_amd.kernels import moe
from fast_moe_amd.kernels.hip import ops
from tests.helpers import make_routing

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
HALF_STEP = {BF16: 2.0 ** -8, F32: 2.0 ** -24}
SIZES = [(1, 1), (1, 8), (3, 31), (2, 32), (5, 33), (4, 64), (7, 100), (129, 1408), (3, 2600), (1000, 40), (2, 4097)]


def codes(v):
    """codes, biased exponents and what they stand for, of rows in 64 bits (exact: only powers of two and one rounding to nearest even)."""
    v = v.double().cpu()
    R, H = v.shape
    P = (H + 31) // 32 * 32
    blocks = torch.nn.functional.pad(v, (0, P - H)).view(R, P // 32, 32)
    top = blocks.abs().amax(dim=2)
    e = torch.where(top > 0, (torch.frexp(top)[1] - 1).clamp_min(-127), -127)
    q = torch.round(torch.ldexp(blocks, 6 - e[:, :, None])).clamp(-127, 127)
    return q.view(R, P).to(torch.int8), (e + 127).to(torch.uint8), torch.ldexp(q, e[:, :, None] - 6).view(R, P)[:, :H]


def rows(R, H, dtype, seed, spread=True):
    g = torch.Generator().manual_seed(seed)
    v = torch.randn(R, H, generator=g)
    if spread:                      # columns over forty powers of two, blocks of zeros
        v = v * 2.0 ** torch.randint(-20, 20, (R, (H + 31) // 32), generator=g).repeat_interleave(32, dim=1)[:, :H]
        v[:, 32:64] = 0
    return v.to(dtype)


@pytest.mark.parametrize("R,H", SIZES)
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_codes_and_what_they_stand_for(R, H, dtype):
    g, u = rows(R, H, dtype, R + H), rows(R, H, dtype, R + H + 1)
    kept = moe.checkpoint_swiglu(g.cuda(), u.cuda())
    back = moe.read_checkpoint(kept)
    for m, v in enumerate((g, u)):
        q, e, stands = codes(v)
        assert torch.equal(kept.q[:, m].cpu(), q) and torch.equal(kept.e[:, m].cpu(), e)
        assert back[m].dtype == dtype and torch.equal(back[m].cpu().double(), stands)


def test_the_ends_of_the_range():
    v = torch.zeros(1, 7 * 32)
    v[0, 0:4] = torch.tensor([1.9921875, 1.9990234375, -1.9990234375, 1.0])         # above 127.5 / 64: held to 127
    v[0, 32:35] = torch.tensor([1.0, 0.5 / 64, 1.5 / 64])                           # ties to even: 0 and 2
    v[0, 64] = 2.0 ** -126
    v[0, 65] = 2.0 ** -130
    v[0, 96] = 2.0 ** -130                                                          # below the normal range
    v[0, 128] = torch.finfo(BF16).max
    v[0, 160:162] = torch.tensor([float("inf"), 1.0])
    v[0, 192:194] = torch.tensor([float("nan"), 1.0])
    for dtype in (BF16, F32):
        x = v.to(dtype)
        kept = moe.checkpoint_swiglu(x.cuda(), x.cuda())
        got = moe.read_checkpoint(kept)[0].cpu()
        q, e, stands = codes(x[:, :160])
        assert torch.equal(kept.q[0, 0, :160].cpu(), q[0]) and torch.equal(kept.e[0, 0, :5].cpu(), e[0])
        assert torch.equal(got[:, :160].double(), stands)
        assert got[0, 160:].isnan().all() and kept.e[0, 0, 5:].tolist() == [255, 255]


@pytest.mark.parametrize("R,H", SIZES)
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("weight", [None, BF16, F32])
def test_backward_on_the_codes(R, H, dtype, weight):
    g, u = rows(R, H, dtype, R + H, spread=False) * 3, rows(R, H, dtype, R + H + 1, spread=False)
    gen = torch.Generator().manual_seed(7)
    d = torch.randn(R, H, generator=gen).to(dtype)
    w = None if weight is None else torch.rand(R, generator=gen).to(weight)
    kept = moe.checkpoint_swiglu(g.cuda(), u.cuda())
    got = moe.swiglu_checkpoint_bwd(kept, d.cuda(), None if w is None else w.cuda())
    (_, _, gd), (_, _, ud) = codes(g), codes(u)
    ww, dd = (1.0 if w is None else w.double()[:, None]), d.double()
    s = torch.sigmoid(gd)
    act = gd * s
    want = (ww * dd * ud * (s + act * (1 - s)), ww * dd * act, ww * act * ud)
    # what cancels in the slope of silu: |s| + |act (1 - s)|
    mags = ((ww * dd * ud).abs() * (s + act.abs() * (1 - s)), want[1].abs(), want[2].abs())
    for a, b, m in zip(got, want, mags):
        assert a.dtype == dtype
        # one rounding to the type, on sigmoid and products within 16 steps of 2^-24
        bound = HALF_STEP[dtype] * b.abs() + 16 * 2.0 ** -24 * m + 1e-37
        assert ((a.double().cpu() - b).abs() <= bound).all(), ((a.double().cpu() - b).abs() / bound).max()
    dots = (act * ud * dd)
    bound = 2.0 ** -17 * dots.abs().sum(1) + 1e-37          # up to 65 values a lane, six steps between lanes, the factors' own: below 128 * 2^-24
    assert got[3].dtype == F32 and ((got[3].double().cpu() - dots.sum(1)).abs() <= bound).all()


def test_strided_rows_and_same_bits_each_time():
    R, H = 50, 96
    both = torch.randn(R, 2 * H + 8, device="cuda").to(BF16)
    want = moe.checkpoint_swiglu(both[:, :H].contiguous(), both[:, H:2 * H].contiguous())
    got = moe.checkpoint_swiglu(both[:, :H], both[:, H:2 * H])
    odd = torch.zeros(R, H + 3, device="cuda", dtype=BF16)
    odd[:, 1:H + 1] = both[:, :H]
    third = moe.checkpoint_swiglu(odd[:, 1:H + 1], both[:, H:2 * H])
    for k in (got, third):
        assert torch.equal(k.q, want.q) and torch.equal(k.e, want.e)
    d = torch.randn(R, H, device="cuda").to(BF16)
    first = moe.swiglu_checkpoint_bwd(want, d)
    wide = torch.zeros(R, H + 3, device="cuda", dtype=BF16)
    wide[:, 1:H + 1] = d
    for again in (moe.swiglu_checkpoint_bwd(want, d), moe.swiglu_checkpoint_bwd(want, wide[:, 1:H + 1])):
        assert all(torch.equal(a, b) for a, b in zip(again[:3], first[:3]))
    assert torch.equal(moe.swiglu_checkpoint_bwd(want, d)[3], first[3])
    joint = ops.swiglu_checkpoint_bwd(want, d, joint=True)
    assert torch.equal(joint[0], first[0]) and torch.equal(joint[1], first[1]) and ops.joint_rows(joint[0], joint[1]) is not None


def block(T, E, K, D, H, dtype, biases, seed=0, layout="nk"):
    r = make_routing(T, E, K, seed=seed)
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s, scale=1.0: (torch.randn(*s, generator=g) * scale).to(dtype).cuda()
    w = lambda i, o: rnd(E, o, i, scale=i ** -0.5).permute(0, 2, 1) if layout == "nk" else rnd(E, i, o, scale=i ** -0.5)
    p = {"x": rnd(T, D), "w": w(D, H), "wp": w(D, H), "wo": w(H, D), "gates": (torch.rand(T, K, generator=g) + 0.1).to(dtype).cuda()}
    for n, c in (("b", H), ("bp", H), ("bo", D)):
        p[n] = rnd(E, c, scale=0.2) if biases else None
    return {n: t.cuda() for n, t in r.items()}, p


def run_block(r, p, K, bits, dy):
    leaves = {n: t.detach().requires_grad_(True) for n, t in p.items() if t is not None}
    q = lambda n: leaves.get(n)
    y = moe.fused_jagged_bmm_swiglu_combine(r["offsets"], r["index"], q("x"), q("w"), q("b"), q("wp"), q("bp"), q("wo"), q("bo"), K, q("gates"),
                                            r["gate_index"], checkpoint_bits=bits)
    y.backward(dy)
    return y.detach(), {n: t.grad for n, t in leaves.items()}


def block_formula(r, p, K, dy, bits=True):
    """Gradients of the block in 64 bits with the pre-activations of the backward pass rounded to their 8-bit values."""
    v = {n: None if t is None else t.detach().double().cpu().requires_grad_(n not in ("w",)) for n, t in p.items()}
    v = {n: None if t is None else t.detach().double().cpu().requires_grad_(True) for n, t in p.items()}
    off, tok, gi = r["offsets"].cpu(), r["token_index"].cpu(), r["gate_index"].cpu()
    parts = []
    for e in range(off.numel() - 1):
        rows_ = slice(int(off[e]), int(off[e + 1]))
        x = v["x"][tok[rows_]]
        add = lambda n: 0 if v[n] is None else v[n][e]
        a, u = x @ v["w"][e] + add("b"), x @ v["wp"][e] + add("bp")
        if bits and a.numel():          # the value of the code, the gradient of the value (a straight line through the rounding)
            dt = p["x"].dtype
            a = a + (codes(a.detach().to(dt))[2] - a.detach())
            u = u + (codes(u.detach().to(dt))[2] - u.detach())
        parts.append((a * torch.sigmoid(a) * u) @ v["wo"][e] + add("bo"))
    value = torch.cat(parts) * v["gates"].flatten()[gi][:, None]
    y = torch.zeros(p["x"].shape[0], value.shape[1], dtype=torch.float64).index_add_(0, tok, value)
    y.backward(dy.double().cpu())
    return y.detach(), {n: t.grad for n, t in v.items() if t is not None}


@pytest.mark.parametrize("T,E,K,D,H", [(48, 4, 2, 64, 96), (100, 7, 3, 128, 200), (5, 6, 2, 40, 33), (300, 4, 2, 256, 128)])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("biases", [False, True])
def test_block_with_its_activations_in_8_bits(T, E, K, D, H, dtype, biases):
    r, p = block(T, E, K, D, H, dtype, biases, seed=T)
    dy = torch.randn(T, D, device="cuda").to(dtype)
    y, grads = run_block(r, p, K, 8, dy)
    plain_y, plain = run_block(r, p, K, None, dy)
    assert torch.equal(y, plain_y)                          # the forward pass is the same
    want = block_formula(r, p, K, dy)[1]
    # In norm.  fp32: sums in another order, and a code that falls the other way where a pre-activation lies next to a border (one step in 64 of its
    # block, for few values in a thousand).  bf16: five roundings of 2^-8 one after another at most (gathered rows, d_h, dg / du / h, the product's
    # rows, the result) and the pre-activations' own, whose codes move by a step where the rounding crosses a border.
    for n, g in grads.items():
        rel = ((g.double().cpu() - want[n]).norm() / want[n].norm()).item()
        assert rel <= (2e-3 if dtype == F32 else 6 * 2.0 ** -8), (n, rel)
        # against the block that keeps everything: a code is off by at most half a step of 1 / 64 of the block's power of two (1 / 128, rms a third of
        # that over values of rms about a third of it): 1.5 % for each of the two pre-activations, on top of the roundings
        rel = ((g.double() - plain[n].double()).norm() / plain[n].double().norm()).item()
        assert rel <= 0.03 + 6 * HALF_STEP[dtype], (n, rel)


def test_block_without_gates_or_some_gradients():
    r, p = block(40, 5, 2, 64, 64, BF16, False, seed=9)
    dy = torch.randn(40, 64, device="cuda").to(BF16)
    x, w = p["x"].clone().requires_grad_(True), p["wo"].detach().requires_grad_(True)
    y = moe.fused_jagged_bmm_swiglu_combine(r["offsets"], r["index"], x, p["w"], None, p["wp"], None, w, None, 2, checkpoint_bits=8)
    y.backward(dy)
    p["gates"] = torch.ones_like(p["gates"])
    want = block_formula(r, p, 2, dy)[1]
    for g, n in ((x.grad, "x"), (w.grad, "wo")):
        assert ((g.double().cpu() - want[n]).norm() / want[n].norm()).item() <= 6 * 2.0 ** -8
    with torch.no_grad():
        again = moe.fused_jagged_bmm_swiglu_combine(r["offsets"], r["index"], x, p["w"], None, p["wp"], None, w, None, 2, checkpoint_bits=8)
    assert torch.equal(again, y)


def test_block_keeps_less():
    r, p = block(2048, 8, 4, 256, 512, BF16, False, seed=1)
    kept = {}
    for bits in (None, 8):
        leaves = [t.detach().requires_grad_(True) for t in (p["x"], p["w"], p["wp"], p["wo"], p["gates"])]
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = moe.fused_jagged_bmm_swiglu_combine(r["offsets"], r["index"], leaves[0], leaves[1], None, leaves[2], None, leaves[3], None, 4, leaves[4],
                                                r["gate_index"], checkpoint_bits=bits)
        kept[bits] = torch.cuda.memory_allocated() - before
        del y
    rows_ = 2048 * 4
    assert kept[8] <= rows_ * 2 * 512 * 33 / 32 + 2048 * 256 * 2 + rows_ * 16 + (1 << 20) < kept[None] / 2.5


def test_expert_without_rows_and_no_rows_at_all():
    r, p = block(16, 6, 1, 64, 64, BF16, True, seed=3)
    topk = torch.zeros(16, 1, dtype=torch.int64)            # everything to expert 0
    from tests.helpers import o_routing
    meta = o_routing.routing_metadata(topk.numpy(), 6)
    r = {"index": torch.from_numpy(meta["gate_index"]).view(-1, 1).cuda(), "gate_index": torch.from_numpy(meta["gate_index"]).cuda(),
         "token_index": torch.from_numpy(meta["token_index"]).cuda(), "offsets": torch.from_numpy(meta["offsets"]).cuda()}
    dy = torch.randn(16, 64, device="cuda").to(BF16)
    _, grads = run_block(r, p, 1, 8, dy)
    want = block_formula(r, p, 1, dy)[1]
    for n, g in grads.items():
        assert ((g.double().cpu() - want[n]).norm() <= 6 * 2.0 ** -8 * want[n].norm()), n
        if n[0] in "wb":
            assert not g[1:].any()
    empty = torch.zeros(0, 96, dtype=BF16, device="cuda")
    kept = moe.checkpoint_swiglu(empty, empty)
    assert kept.q.shape == (0, 2, 96) and moe.read_checkpoint(kept)[0].shape == (0, 96)
    assert moe.swiglu_checkpoint_bwd(kept, empty)[3].shape == (0,)


def test_replays_from_a_graph():
    R, H = 200, 320
    g, u, d = (torch.randn(R, H, device="cuda").to(BF16) for _ in range(3))
    w = torch.rand(R, device="cuda")
    both = lambda: moe.swiglu_checkpoint_bwd(moe.checkpoint_swiglu(g, u), d, w)
    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    for _ in range(3):
        g.copy_(torch.randn(R, H, device="cuda").to(BF16))
        want = both()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals():
    g = torch.randn(4, 64, device="cuda").to(BF16)
    kept = moe.checkpoint_swiglu(g, g)
    for bad in (lambda: moe.checkpoint_swiglu(g, g[:3]), lambda: moe.checkpoint_swiglu(g, g.float()), lambda: moe.checkpoint_swiglu(g[0], g[0]),
                lambda: moe.checkpoint_swiglu(g.cpu(), g.cpu()), lambda: moe.swiglu_checkpoint_bwd(kept, g[:3]),
                lambda: moe.swiglu_checkpoint_bwd(kept, g.float()), lambda: moe.swiglu_checkpoint_bwd(kept, g, torch.ones(3, device="cuda")),
                lambda: moe.read_checkpoint(kept._replace(cols=70)), lambda: moe.read_checkpoint(kept._replace(e=kept.e[:, :, :1]))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(NotImplementedError):
        moe.checkpoint_swiglu(g.half(), g.half())
    with pytest.raises(RuntimeError, match="forward-only"):
        moe.checkpoint_swiglu(g.clone().requires_grad_(True), g)
    r, p = block(8, 4, 2, 64, 64, BF16, False)
    with pytest.raises(ValueError, match="None or 8"):
        moe.fused_jagged_bmm_swiglu_combine(r["offsets"], r["index"], p["x"], p["w"], None, p["wp"], None, p["wo"], None, 2, checkpoint_bits=4)


def test_block_without_tokens():
    D, H, E, K = 64, 96, 4, 2
    rnd = lambda *s: torch.randn(*s, device="cuda").to(BF16)
    p = {"x": rnd(0, D), "w": rnd(E, H, D).permute(0, 2, 1), "b": None, "wp": rnd(E, H, D).permute(0, 2, 1), "bp": None, "wo": rnd(E, D, H).permute(0, 2, 1),
         "bo": rnd(E, D), "gates": rnd(0, K)}
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    r = {"offsets": torch.zeros(E + 1, dtype=torch.int64, device="cuda"), "index": none.view(0, K), "gate_index": none}
    y, grads = run_block(r, p, K, 8, rnd(0, D))
    assert y.shape == (0, D) and len(grads) == 6
    for n, g in grads.items():
        assert g.shape == p[n].shape and not g.any()
