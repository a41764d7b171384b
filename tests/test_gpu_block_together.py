"""The operators around an expert block as a layer uses them one after another, against the layer's definition in 64 bits: a decode step (norm, few
tokens, residual and next norm) and a training step (norm, routing, the block with its activations in 8 bits, merge with residual and norms)."""
import pytest
import torch

from fast_moe_amd.kernels import moe
from tests.helpers import make_routing

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
EPS = 1e-6


def rms(v, w):
    return v / torch.sqrt((v * v).mean(dim=1, keepdim=True) + EPS) * w


def layer(T, E, D, H, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s, scale=1.0: (torch.randn(*s, generator=g) * scale).to(dtype).cuda()
    p = {"x": rnd(T, D), "router": rnd(E, D, scale=2 * D ** -0.5), "w": rnd(E, H, D, scale=D ** -0.5).permute(0, 2, 1),
         "wp": rnd(E, H, D, scale=D ** -0.5).permute(0, 2, 1), "wo": rnd(E, D, H, scale=H ** -0.5).permute(0, 2, 1), "token_gate": rnd(T, 1)}
    for n in ("before", "after", "next"):
        p[n] = 1 + rnd(D, scale=0.2)
    p["scale"] = rnd(D, scale=0.5)
    return p


def decode(p, k, mask=None):
    n = moe.block_norm(p["x"], p["before"])
    y = moe.fused_moe_few_tokens(n, p["router"], None, p["w"], None, p["wp"], None, p["wo"], None, k, token_mask=mask)
    return moe.block_norm_add(y, p["x"], weight=p["after"], gate=p["token_gate"], gate_sigmoid=True, scale=p["scale"], next_weight=p["next"])


@pytest.mark.parametrize("T,E,k,D,H", [(1, 8, 2, 128, 96), (16, 16, 4, 256, 64), (37, 12, 3, 200, 104), (64, 8, 2, 64, 48)])
def test_a_decode_step(T, E, k, D, H):
    p = layer(T, E, D, H, F32, seed=T)
    out, nxt = decode(p, k)
    v = {n: t.double().cpu() for n, t in p.items()}
    n = rms(v["x"], v["before"])
    logits = n @ v["router"].T
    best = logits.sort(dim=1, descending=True)
    # (fp32 logits are off by 2^-24 times 64 at most, of the sum of magnitudes: the choice is the same one where the gaps are far wider)
    assert k == E or (best.values[:, k - 1] - best.values[:, k]).min() > 1e-4
    prob = torch.softmax(best.values[:, :k], dim=1)
    y = torch.zeros(T, D, dtype=torch.float64)
    for t in range(T):
        for j in range(k):
            e = best.indices[t, j]
            a = n[t] @ v["w"][e]
            y[t] += prob[t, j] * ((a * torch.sigmoid(a) * (n[t] @ v["wp"][e])) @ v["wo"][e])
    want = v["x"] + v["scale"] * torch.sigmoid(v["token_gate"]) * rms(y, v["after"])
    # sums of at most 256 products in fp32, five of them in a row and three norms, each within 2^-24 * 16 in norm: 2^-16 covers them twice over
    for a, b in ((out, want), (nxt, rms(want, v["next"]))):
        assert ((a.double().cpu() - b).norm(dim=1) <= 2.0 ** -16 * b.norm(dim=1)).all()


def test_a_decode_step_replayed_for_a_padded_batch():
    p, k = layer(24, 16, 256, 128, BF16, seed=5), 4
    mask = torch.ones(24, dtype=torch.bool, device="cuda")
    decode(p, k, mask)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = decode(p, k, mask)
    for live in (24, 1, 0, 17):
        p["x"].copy_(torch.randn(24, 256, device="cuda").to(BF16))
        mask.copy_(torch.arange(24, device="cuda") < live)
        want = decode(p, k, mask)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        alone = decode({n: t[:live] if n in ("x", "token_gate") else t for n, t in p.items()}, k) if live else None
        if live and (live + 31) // 32 == 1 and live > 16:       # (the same tiles as the padded batch: the same bits)
            assert torch.equal(alone[0], want[0][:live])
        assert torch.equal(want[0][live:], p["x"][live:])       # a masked row adds nothing


def code(v):
    """What a block's 8 bits stand for, straight through for the gradient."""
    H = v.shape[1]
    blocks = torch.nn.functional.pad(v.detach(), (0, -H % 32)).view(v.shape[0], -1, 32)
    top = blocks.abs().amax(dim=2, keepdim=True)
    e = torch.where(top > 0, (torch.frexp(top)[1] - 1), torch.zeros_like(top, dtype=torch.int32))
    q = torch.ldexp(torch.round(torch.ldexp(blocks, 6 - e)).clamp(-127, 127), e - 6).view(v.shape[0], -1)[:, :H]
    return v + (q - v.detach())


@pytest.mark.parametrize("merged", [False, True])
def test_a_training_step(merged):
    T, E, k, D, H = 96, 6, 2, 128, 96
    p, r = layer(T, E, D, H, F32, seed=7), make_routing(T, E, k, seed=7)
    p["share"] = (torch.rand(T, k, generator=torch.Generator().manual_seed(1)) + 0.2).cuda()
    d = [torch.randn(T, D, generator=torch.Generator().manual_seed(s)).cuda() for s in (2, 3)]
    c = {n: t.cuda() for n, t in r.items()}
    leaves = {n: t.detach().requires_grad_(True) for n, t in p.items() if n != "router"}
    q = leaves.__getitem__
    around = dict(weight=q("after"), gate=q("token_gate"), gate_sigmoid=True, scale=q("scale"), next_weight=q("next"))
    n = moe.block_norm(q("x"), q("before"))
    if merged:          # the expert rows go to the norms without being merged first (nothing in 8 bits)
        hidden = moe.index_select_jagged_bmm_swiglu(0, c["offsets"], c["index"], n, q("w"), None, q("wp"), None)
        rows = moe.index_select_jagged_bmm(0, c["offsets"], torch.arange(T * k, device="cuda").view(-1, 1), hidden, q("wo"), None)
        out, nxt = moe.mul_merge_k_norm_add(c["token_index"], c["reverse_index"], rows, q("x"), q("share"), c["gate_index"], **around)
    else:
        y = moe.fused_jagged_bmm_swiglu_combine(c["offsets"], c["index"], n, q("w"), None, q("wp"), None, q("wo"), None, k, q("share"), c["gate_index"],
                                                checkpoint_bits=8)
        out, nxt = moe.block_norm_add(y, q("x"), **around)
    torch.autograd.backward((out, nxt), d)

    v = {m: t.detach().double().cpu().requires_grad_(True) for m, t in leaves.items()}
    off, tok, gi = r["offsets"], r["token_index"], r["gate_index"]
    x = rms(v["x"], v["before"])
    rows, exact = [], []
    for e in range(E):
        part = x[tok[off[e]:off[e + 1]]]
        a, u = part @ v["w"][e], part @ v["wp"][e]
        exact.append((a * torch.sigmoid(a) * u) @ v["wo"][e])
        if not merged:
            a, u = code(a), code(u)
        rows.append((a * torch.sigmoid(a) * u) @ v["wo"][e])
    merge = lambda rows: torch.zeros(T, D, dtype=torch.float64).index_add(0, tok, torch.cat(rows) * v["share"].flatten()[gi][:, None])
    y = merge(rows)
    y = y + (merge(exact) - y).detach()         # (the forward pass has the values, the backward pass their codes, the shares' gradient with it)
    want = v["x"] + v["scale"] * torch.sigmoid(v["token_gate"]) * rms(y, v["after"])
    want_next = rms(want, v["next"])
    torch.autograd.backward((want, want_next), [t.double().cpu() for t in d])
    for a, b in ((out, want), (nxt, want_next)):
        assert ((a.detach().double().cpu() - b.detach()).norm() <= 2.0 ** -16 * b.detach().norm())
    for m, t in leaves.items():
        # in norm: fp32 sums, and with 8 bits the few codes that lie next to a border and fall the other way (of 18432, by one step of 64)
        rel = ((t.grad.double().cpu() - v[m].grad).norm() / v[m].grad.norm()).item()
        assert rel <= (2.0 ** -15 if merged else 2e-3), (m, rel)
