"""kernels.moe.fused_moe_few_tokens and its e4m3 form against the definition in 64 bits."""
import pytest
import torch

from fast_moe_amd.kernels import moe, moe_fp8
from fast_moe_amd.kernels.hip import ops

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def make(T, E, D, H, O, dtype, swiglu=True, biases=False, seed=0):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s, scale=1.0: (torch.randn(*s, generator=g) * scale).to(dtype).cuda()
    p = {"x": rnd(T, D), "gate_weight": rnd(E, D, scale=D ** -0.5), "weight": rnd(E, H, D, scale=D ** -0.5).permute(0, 2, 1),
         "weight_out": rnd(E, O, H, scale=H ** -0.5).permute(0, 2, 1)}
    p["weight_p"] = rnd(E, H, D, scale=D ** -0.5).permute(0, 2, 1) if swiglu else None
    for n, shape in (("gate_bias", (E,)), ("bias", (E, H)), ("bias_p", (E, H)), ("bias_out", (E, O))):
        p[n] = rnd(*shape, scale=0.2) if biases and (n != "bias_p" or swiglu) else None
    return p


def reference(p, k, renorm=True, mask=None):
    """The definition in 64 bits on the CPU, token by token.  -> (y, what the roundings of h may move y by)"""
    d = {n: None if t is None else t.detach().double().cpu() for n, t in p.items()}
    # (products and a sum of its own for every logit: equal experts get equal ones, which a library's matrix product does not promise)
    logits = (d["x"][:, None, :] * d["gate_weight"]).sum(dim=2) + (0 if d["gate_bias"] is None else d["gate_bias"])
    prob = torch.softmax(logits, dim=1)
    T, O = d["x"].shape[0], d["weight_out"].shape[2]
    y, slack = torch.zeros(T, O, dtype=torch.float64), torch.zeros(T, O, dtype=torch.float64)
    for t in range(T):
        if mask is not None and not mask[t]:
            continue
        chosen = torch.sort(logits[t], descending=True, stable=True).indices[:k].tolist()
        total = prob[t, chosen].sum() if renorm else 1.0
        for e in chosen:
            bias = lambda n: 0 if d[n] is None else d[n][e]
            a = d["x"][t] @ d["weight"][e] + bias("bias")
            h = a * torch.sigmoid(a)
            if d["weight_p"] is not None:
                h = h * (d["x"][t] @ d["weight_p"][e] + bias("bias_p"))
            gate = prob[t, e] / total
            y[t] += gate * (h @ d["weight_out"][e] + bias("bias_out"))
            slack[t] += gate * (h.abs() @ d["weight_out"][e].abs())
    return y, slack


def check(got, p, k, renorm=True, mask=None, fp8=False):
    want, slack = reference(p, k, renorm, mask)
    # bf16: h and y are rounded once each, by 2^-8 of the value at most; fp32 sums of up to 2^12 products in any order are
    # off by at most their count times 2^-24 of the sum of magnitudes (2^-12: an eighth of one bf16 rounding of h), in both products and the router
    eps = 2.0 ** -8 if got.dtype == BF16 else 0.0
    bound = eps * want.abs() + (eps + 2.0 ** -11) * slack + 1e-30
    if got.dtype == F32:
        bound = 2.0 ** -14 * (slack + want.abs()) + 1e-30
    err = (got.double().cpu() - want).abs()
    assert got.shape == want.shape and (err <= bound).all(), f"{int((err > bound).sum())} of {err.numel()} off, worst {(err / bound).max():.3g} of the bound"


CASES = [
    # T, E, k, D, H, O
    (1, 8, 2, 128, 256, 128), (1, 64, 8, 256, 176, 256), (2, 1, 1, 64, 64, 64), (3, 5, 5, 40, 24, 56), (16, 16, 4, 512, 96, 80),
    (17, 12, 3, 200, 104, 72), (32, 4, 2, 136, 48, 40), (33, 8, 2, 96, 80, 64), (64, 4, 2, 64, 128, 64), (64, 2, 2, 64, 40, 48), (64, 130, 8, 64, 32, 48),
    (5, 256, 16, 64, 32, 32), (7, 20, 6, 1, 1, 1), (9, 9, 3, 33, 17, 31), (40, 6, 2, 1023, 31, 15), (64, 256, 16, 24, 8, 24),
]


@pytest.mark.parametrize("T,E,k,D,H,O", CASES)
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("swiglu,biases", [(True, False), (False, True), (True, True)])
def test_against_the_definition(T, E, k, D, H, O, dtype, swiglu, biases):
    p = make(T, E, D, H, O, dtype, swiglu, biases, seed=T * 1000 + E)
    check(moe.fused_moe_few_tokens(k=k, **p), p, k)


@pytest.mark.parametrize("T,E,k,D,H,O", [c for c in CASES if c[3] > 1])
@pytest.mark.parametrize("swiglu,biases", [(True, False), (False, True)])
@pytest.mark.parametrize("pow2", [True, False])
def test_e4m3_weights_against_the_definition(T, E, k, D, H, O, swiglu, biases, pow2):
    p = make(T, E, D, H, O, BF16, swiglu, biases, seed=T * 1000 + E + 1)
    pairs, plain = {}, dict(p)
    for n in ("weight", "weight_p", "weight_out"):
        if p[n] is None:
            pairs[n] = None
            continue
        q, s = moe_fp8.quantize_expert_weights(p[n])
        if not pow2:        # another quantisation's scales
            s = s * (1 + torch.rand(s.shape, generator=torch.Generator().manual_seed(5)).cuda())
        pairs[n], plain[n] = (q, s), q.float().double() / s.double()[:, None, :]
    got = moe_fp8.fused_moe_few_tokens(p["x"], p["gate_weight"], p["gate_bias"], pairs["weight"], p["bias"], pairs["weight_p"], p["bias_p"],
                                       pairs["weight_out"], p["bias_out"], k)
    check(got, plain, k)


@pytest.mark.parametrize("T", [1, 16, 30, 64])
def test_renorm_off_and_masked_rows(T):
    p = make(T, 16, 64, 48, 64, BF16, True, True, seed=T)
    check(moe.fused_moe_few_tokens(k=3, renorm=False, **p), p, 3, renorm=False)
    mask = (torch.arange(T) % 3 != 1)
    p["x"][1::3] = float("nan")             # what a padded row holds does not matter
    got = moe.fused_moe_few_tokens(k=3, token_mask=mask.cuda(), **p)
    p["x"] = torch.where(mask.cuda()[:, None], p["x"], torch.zeros_like(p["x"]))
    check(got, p, 3, mask=mask)
    assert not got[1::3].any()
    none = moe.fused_moe_few_tokens(k=3, token_mask=torch.zeros(T, dtype=torch.bool, device="cuda"), **p)
    assert not none.any()


def test_ties_take_the_lowest_expert_and_nan_stays_in_its_row():
    p = make(4, 9, 64, 32, 64, F32, seed=3)
    p["gate_weight"][:] = p["gate_weight"][0].clone()            # every logit equal
    check(moe.fused_moe_few_tokens(k=4, **p), p, 4)              # the stable order: experts 0 .. 3
    p = make(20, 9, 64, 32, 64, BF16, seed=4)
    clean = moe.fused_moe_few_tokens(k=2, **p)
    p["x"][7, 3] = float("nan")
    got = moe.fused_moe_few_tokens(k=2, **p)
    rest = torch.arange(20) != 7
    assert got[7].isnan().all() and torch.equal(got[rest], clean[rest])


def test_infinite_weights_reach_only_the_tokens_of_their_expert():
    p = make(6, 4, 64, 32, 64, BF16, seed=5)
    p["gate_bias"] = torch.tensor([0.0, 0.0, 0.0, -60000.0], dtype=BF16, device="cuda")     # nobody asks expert 3 ...
    clean = moe.fused_moe_few_tokens(k=2, **p)
    p["weight_out"][3] = float("inf")
    p["weight"][3] = float("nan")
    assert torch.equal(moe.fused_moe_few_tokens(k=2, **p), clean)
    p = make(6, 4, 64, 32, 64, BF16, seed=5)
    logits = p["x"].float() @ p["gate_weight"].float().T
    hit = (logits.topk(2, dim=1).indices == 2).any(dim=1)
    assert hit.any() and not hit.all()                                                      # ... some ask expert 2
    clean = moe.fused_moe_few_tokens(k=2, **p)
    p["weight_out"][2] = float("inf")
    got = moe.fused_moe_few_tokens(k=2, **p)
    assert torch.equal(got[~hit], clean[~hit]) and not got[hit].isfinite().any()


def test_strided_operands_give_the_same_bits():
    p = make(5, 8, 64, 48, 64, BF16, True, True, seed=6)
    want = moe.fused_moe_few_tokens(k=2, **p)
    wide = torch.zeros(5, 200, dtype=BF16, device="cuda")
    wide[:, 8:72] = p["x"]
    storage = torch.zeros(8, 2, 48, 80, dtype=BF16, device="cuda")           # gate and up interleaved by expert, rows with a gap
    storage[:, 0, :, :64], storage[:, 1, :, :64] = p["weight"].permute(0, 2, 1), p["weight_p"].permute(0, 2, 1)
    q = dict(p, x=wide[:, 8:72], weight=storage[:, 0, :, :64].permute(0, 2, 1), weight_p=storage[:, 1, :, :64].permute(0, 2, 1))
    assert torch.equal(moe.fused_moe_few_tokens(k=2, **q), want)
    odd = torch.zeros(5, 67, dtype=BF16, device="cuda")                      # rows at odd addresses: the element loads
    odd[:, 1:65] = p["x"]
    q = dict(p, x=odd[:, 1:65])
    check(moe.fused_moe_few_tokens(k=2, **q), p, 2)


def test_same_bits_each_time_on_two_streams_and_from_a_graph():
    p, other = make(12, 16, 256, 128, 256, BF16, seed=7), make(12, 16, 256, 128, 256, BF16, seed=8)
    want, want2 = moe.fused_moe_few_tokens(k=4, **p), moe.fused_moe_few_tokens(k=4, **other)
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(8):
        with torch.cuda.stream(a):
            got.append((moe.fused_moe_few_tokens(k=4, **p), want))
        with torch.cuda.stream(b):
            got.append((moe.fused_moe_few_tokens(k=4, **other), want2))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in got)
    graphs, outs = [], []
    for q in (p, other):                    # two graphs with a workspace each
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(moe.fused_moe_few_tokens(k=4, **q))
        graphs.append(graph)
    for seed in (9, 10, 11):
        p["x"].copy_(make(12, 16, 256, 128, 256, BF16, seed=seed)["x"])
        want = moe.fused_moe_few_tokens(k=4, **p)
        torch.cuda.synchronize()
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want2)


def test_no_tokens_and_the_layer_beside_it():
    p = make(0, 8, 64, 48, 64, BF16, seed=1)
    assert moe.fused_moe_few_tokens(k=2, **p).shape == (0, 64)
    from fast_moe_amd import FastMoELayer
    torch.manual_seed(0)
    layer = FastMoELayer(128, 256, 128, 8).to(BF16).cuda()
    x = torch.randn(1, 6, 128, device="cuda").to(BF16)
    with torch.no_grad():
        want = layer(x, 2)[0].float()
        got = moe.fused_moe_few_tokens(x[0], layer.gate.gate.weight, layer.gate.gate.bias, layer._experts_hidden_w.permute(0, 2, 1),
                                       layer._experts_hidden_bias, None, None, layer._experts_w.permute(0, 2, 1), layer._experts_bias, 2).float()
    # the layer rounds logits, gates, hidden rows (twice) and expert rows to bf16: a few steps of 2^-8
    assert (got - want).abs().max() <= 0.05 * want.abs().max()


def test_refusals():
    p = make(4, 8, 64, 48, 64, BF16, True, True, seed=1)
    call = lambda k=2, **kw: moe.fused_moe_few_tokens(k=k, **dict(p, **kw))
    big = torch.zeros(65, 64, dtype=BF16, device="cuda")
    for bad, match in ((dict(x=big), "up to 64 tokens"), (dict(k=9), "1 <= k <= E"), (dict(k=0), "1 <= k <= E"),
                       (dict(x=p["x"][:, :32]), "do not fit"), (dict(weight=p["weight"].contiguous()), "contraction contiguous"),
                       (dict(weight_p=p["weight_p"].permute(0, 2, 1).contiguous()[:, :, :].permute(0, 2, 1)[:, :, :47]), "do not fit"),
                       (dict(gate_weight=p["gate_weight"].float()), "must be torch.bfloat16"), (dict(bias=p["bias"][:, :40]), "bias must be"),
                       (dict(weight_p=None), "goes with weight_p"), (dict(token_mask=torch.ones(4, dtype=torch.uint8, device="cuda")), "must be bool"),
                       (dict(x=p["x"].cpu()), "GPU")):
        with pytest.raises(ValueError, match=match):
            call(**bad)
    with pytest.raises(NotImplementedError, match="bf16 or fp32"):
        call(x=p["x"].half())
    with pytest.raises(RuntimeError, match="forward-only"):
        call(x=p["x"].clone().requires_grad_(True))
    with pytest.raises(NotImplementedError, match="not available"):
        call(kernel=moe.KernelType.PYTORCH)
    (q, s), (qo, so) = moe_fp8.quantize_expert_weights(p["weight"]), moe_fp8.quantize_expert_weights(p["weight_out"])
    with pytest.raises(ValueError, match="scales of weight "):
        ops.few_tokens(p["x"], p["gate_weight"], None, q, None, None, None, qo, None, 2, scales=(s[:, :4], None, so))


def test_single_rows_of_any_stride_and_rows_far_apart():
    p = make(1, 4, 64, 1, 1, BF16, seed=2)
    want = moe.fused_moe_few_tokens(k=2, **p)
    far = torch.zeros(2, (1 << 20) + 64, dtype=BF16, device="cuda")
    far[0, :64] = p["x"][0]
    q = dict(p, x=far[:1, :64], weight=p["weight"].contiguous(), weight_p=p["weight_p"].contiguous(), weight_out=p["weight_out"].contiguous())
    assert torch.equal(moe.fused_moe_few_tokens(k=2, **q), want)
    far[1, :64] = 2 * p["x"][0]
    two = moe.fused_moe_few_tokens(k=2, **dict(p, x=far[:, :64]))
    assert torch.equal(two, moe.fused_moe_few_tokens(k=2, **dict(p, x=far[:, :64].contiguous())))
    p = make(2, 2, 1, 8, 4, BF16, seed=3)
    same = p["weight"][:, :, :1].expand(2, 1, 8)                # every hidden column the same storage
    with pytest.raises(ValueError, match="contraction contiguous"):
        moe.fused_moe_few_tokens(k=1, **dict(p, weight=same, weight_p=None))


@pytest.mark.parametrize("T,E,k,D,H,O", [(1, 8, 2, 128, 256, 128), (4, 16, 4, 256, 176, 256), (16, 8, 2, 512, 96, 80), (33, 8, 2, 96, 80, 64), (9, 9, 3, 33, 17, 31)])
@pytest.mark.parametrize("fp8", [False, True])
def test_bf16_rounds_the_output_and_hardly_anything_else(T, E, k, D, H, O, fp8):
    p = make(T, E, D, H, O, BF16, True, False, seed=T + 17)
    plain, pairs = dict(p), {}
    if fp8:
        for n in ("weight", "weight_p", "weight_out"):
            pairs[n] = moe_fp8.quantize_expert_weights(p[n])
            plain[n] = pairs[n][0].float().double() / pairs[n][1].double()[:, None, :]
        got = moe_fp8.fused_moe_few_tokens(p["x"], p["gate_weight"], None, pairs["weight"], None, pairs["weight_p"], None, pairs["weight_out"], None, k)
    else:
        got = moe.fused_moe_few_tokens(k=k, **p)
    want, slack = reference(plain, k)
    # Hidden rows of 16 bits (2^-17 of the value, 2^-16 with room), fp32 sums of up to 512 products and the router's: 2^-14 of the sum of magnitudes holds
    # them all; then the output's own rounding.  A hidden row's second half has a column that its expert's tokens leave free: an expert with more tokens than
    # half of them has its hidden rows rounded to bf16, 2^-8 of the value.  Columns: 16, of which narrow outputs of few tokens use a half or a quarter.
    columns = 16 if T > 8 or O >= 4096 else 8 if T > 4 or O >= 2048 else 4
    logits = (plain["x"].double().cpu()[:, None, :] * plain["gate_weight"].double().cpu()).sum(dim=2)
    chosen = torch.zeros(T, E).scatter_(1, torch.sort(logits, descending=True, stable=True, dim=1).indices[:, :k], 1.0)
    crowded = (chosen * (2 * chosen.sum(dim=0) > columns)).amax(dim=1, keepdim=True).double()
    bound = 2.0 ** -8 * want.abs() + (2.0 ** -14 + 2.0 ** -8 * crowded) * slack + 1e-30
    assert ((got.double().cpu() - want).abs() <= bound).all()
