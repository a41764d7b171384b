"""bf16 operator API of the MoE forward -- the drop-in boundary.

Function names, positional order, keyword names and argument meaning are those
of /root/reference/kernels/moe.py:39-292.  Differences, all on purpose:

* ``kernel`` defaults to ``KernelType.HIP`` (the reference defaults to its
  PyTorch path, which this package does not contain); ``KernelType.TRITON`` is
  accepted and runs the same HIP kernels; any other value raises.
* every operator here has a backward (kernels/hip/autograd.py), the 3D and the two-input
  gating variants included; of the fp8 operators, silu_jagged_bmm_fp8 and silu_jagged_fp8 are
  forward only (as in the reference) and raise when an input requires grad under grad mode.
* ``max_seq_len`` is accepted and ignored: tile scheduling reads ``offsets`` on
  the device, so no host synchronisation is needed to obtain it.
* operands must be bf16 or fp32 CUDA tensors (fp32 runs true-fp32 MFMA, no tf32).
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Tuple, Union

import torch

from .hip import autograd as _ag
from .hip import ops
from .hip._lib import EPI_GATED, EPI_NONE, EPI_SWIGLU
from .utils import KernelType, require_hip_kernel


@dataclass
class IndexSelectJaggedBmmOption:
    """kernels/triton/triton_moe.py:36-43: backward-tuning knobs, accepted and unused."""
    d_jagged_use_grouped_gemm: bool = True
    d_jagged_use_wrap_specialization: bool = True
    d_jagged_gemm_out_type: torch.dtype = torch.float32
    d_weight_optimization: bool = True
    d_weight_split_k_kernel: bool = True
    d_weight_split_k_kernel_tma: bool = False


@dataclass
class SiluJaggedBmmCombineOption:
    """kernels/triton/triton_moe.py:3562-3567: accepted and unused (backward only)."""
    activation_checkpointing: bool = False
    d_weight_optimization: bool = True
    d_weight_split_k_kernel: bool = True
    d_weight_split_k_kernel_tma: bool = False


def _check_gather_args(name, index, jagged, weight):
    assert index.ndim == 2 and index.shape[0] == jagged.shape[0], (
        f"{name}: index must be [L, A] with L = jagged.shape[0]")
    assert weight.ndim == 3, f"{name}: weight must be [E, K, N]"


def index_select_jagged_bmm(
    max_seq_len: int,
    offsets: torch.Tensor,
    index: torch.Tensor,
    jagged: torch.Tensor,
    weight: torch.Tensor,
    bias: Optional[torch.Tensor],
    kernel: KernelType = KernelType.HIP,
    triton_option: Optional[IndexSelectJaggedBmmOption] = None,
) -> torch.Tensor:
    """kernels/moe.py:39-68.  ``out[off_e:off_e+1] = jagged[index[...] // A] @ weight[e] + bias[e]``."""
    require_hip_kernel(kernel, "index_select_jagged_bmm")
    _check_gather_args("index_select_jagged_bmm", index, jagged, weight)
    if _ag.needs_grad(jagged, weight, bias):
        return _ag.IndexSelectJaggedBmm.apply(offsets, index, jagged, weight, bias, None, None)
    return ops.grouped_gemm(offsets, jagged, weight, total_rows=index.numel(), row_index=index,
                            index_div=index.shape[-1], bias=bias, epilogue=EPI_NONE)


def mul_merge_k_add(
    index: torch.Tensor,
    reverse_index: torch.Tensor,
    value: torch.Tensor,
    stable_sorting: bool = False,
    weight: Optional[torch.Tensor] = None,
    weight_index: Optional[torch.Tensor] = None,
    kernel: KernelType = KernelType.HIP,
    triton_cc_version: str = "",
) -> torch.Tensor:
    """kernels/moe.py:71-115.  ``out[n] = sum of value[r] * weight_flat[weight_index[r]]`` over the
    K rows r = reverse_index[n, :], added in ascending r."""
    require_hip_kernel(kernel, "mul_merge_k_add")
    N = index.shape[0]
    L, K = reverse_index.shape
    assert index.ndim == 1 and reverse_index.ndim == 2
    assert N == L * K and N == value.shape[0]
    if weight is not None:
        assert weight_index is not None
        assert weight.numel() == weight_index.numel() == value.shape[0], (
            f"{weight.shape=}, {weight_index.shape=}, {value.shape=}")
    if _ag.needs_grad(value, weight):
        return _ag.MulMergeKAdd.apply(index, reverse_index, value, weight, weight_index)
    return ops.combine(value, reverse_index, weight, weight_index)


def index_select_jagged_bmm_3D(
    max_seq_len: int,
    offsets: torch.Tensor,
    index: torch.Tensor,
    jagged: torch.Tensor,
    weight: torch.Tensor,
    bias: torch.Tensor,
    kernel: KernelType = KernelType.HIP,
) -> torch.Tensor:
    """kernels/moe.py:118-153.  jagged [L, E, D_in]: expert e reads slice ``[:, e, :]``."""
    require_hip_kernel(kernel, "index_select_jagged_bmm_3D")
    assert index.ndim == 2 and index.shape[0] == jagged.shape[0]
    assert jagged.ndim == 3 and jagged.shape[1] == weight.shape[0]
    if _ag.needs_grad(jagged, weight, bias):
        return _ag.IndexSelectJaggedBmm3D.apply(offsets, index, jagged, weight, bias)
    jagged = ops._rows_contiguous(jagged)
    return ops.grouped_gemm(offsets, jagged, weight, total_rows=index.numel(), row_index=index,
                            index_div=index.shape[-1], bias=bias, epilogue=EPI_NONE,
                            a_expert_stride=jagged.stride(1))


def index_select_jagged_bmm_swiglu(
    max_seq_len: int,
    offsets: torch.Tensor,
    index: torch.Tensor,
    jagged: torch.Tensor,
    weight: torch.Tensor,
    bias: Optional[torch.Tensor],
    weight_p: torch.Tensor,
    bias_p: Optional[torch.Tensor],
    kernel: KernelType = KernelType.HIP,
) -> torch.Tensor:
    """kernels/moe.py:156-189.  ``silu(x W + b) * (x Wp + bp)`` in one kernel."""
    require_hip_kernel(kernel, "index_select_jagged_bmm_swiglu")
    _check_gather_args("index_select_jagged_bmm_swiglu", index, jagged, weight)
    assert weight.shape == weight_p.shape
    if weight_p.stride() != weight.stride():
        weight_p = weight_p.contiguous()
        weight = weight.contiguous()
    if _ag.needs_grad(jagged, weight, bias, weight_p, bias_p):
        return _ag.IndexSelectJaggedBmm.apply(offsets, index, jagged, weight, bias, weight_p, bias_p)
    return ops.grouped_gemm(offsets, jagged, weight, total_rows=index.numel(), row_index=index,
                            index_div=index.shape[-1], bias=bias, b2=weight_p, bias2=bias_p,
                            epilogue=EPI_SWIGLU)


def index_select_jagged_gating_bmm(
    max_seq_len: int,
    offsets: torch.Tensor,
    index: torch.Tensor,
    jagged_a: torch.Tensor,
    jagged_b: torch.Tensor,
    weight_a: torch.Tensor,
    bias_a: Optional[torch.Tensor],
    weight_b: torch.Tensor,
    bias_b: Optional[torch.Tensor],
    kernel: KernelType = KernelType.HIP,
) -> torch.Tensor:
    """kernels/moe.py:192-233.  ``silu(A Wa + ba) * (B Wb + bb)``; one fused kernel when A is B,
    otherwise two GEMMs, the second of which multiplies by the SiLU of the first one's result in
    its epilogue (bf16; fp32: two GEMMs and an element-wise kernel)."""
    require_hip_kernel(kernel, "index_select_jagged_gating_bmm")
    assert (index.ndim == 2 and index.shape[0] == jagged_a.shape[0] == jagged_b.shape[0]
            and jagged_a.shape == jagged_b.shape and weight_a.shape == weight_b.shape)
    if jagged_a is jagged_b:
        return index_select_jagged_bmm_swiglu(max_seq_len, offsets, index, jagged_a, weight_a, bias_a,
                                              weight_b, bias_b, kernel)
    if _ag.needs_grad(jagged_a, jagged_b, weight_a, weight_b, bias_a, bias_b):
        return _ag.IndexSelectJaggedGatingBmm.apply(offsets, index, jagged_a, jagged_b, weight_a, weight_b,
                                                    bias_a, bias_b)
    alpha = ops.grouped_gemm(offsets, jagged_a, weight_a, total_rows=index.numel(), row_index=index,
                             index_div=index.shape[-1], bias=bias_a)
    if jagged_a.dtype == torch.bfloat16 and index.numel() > 0:
        return ops.grouped_gemm(offsets, jagged_b, weight_b, total_rows=index.numel(), row_index=index,
                                index_div=index.shape[-1], bias=bias_b, epilogue=EPI_GATED, gate=alpha)
    beta = ops.grouped_gemm(offsets, jagged_b, weight_b, total_rows=index.numel(), row_index=index,
                            index_div=index.shape[-1], bias=bias_b)
    return ops.silu_mul(alpha, beta)


def silu_jagged_bmm_combine(
    max_seq_len: int,
    offsets: torch.Tensor,
    jagged: torch.Tensor,
    weight: torch.Tensor,
    bias: Optional[torch.Tensor],
    index: torch.Tensor,
    reverse_index: torch.Tensor,
    gating_scores: Optional[torch.Tensor] = None,
    gates_index: Optional[torch.Tensor] = None,
    has_silu: bool = True,
    kernel: KernelType = KernelType.HIP,
    triton_option: Optional[SiluJaggedBmmCombineOption] = None,
) -> torch.Tensor:
    """kernels/moe.py:236-292.  ``silu(jagged) @ weight[e] + bias[e]`` on expert-sorted rows, then
    the weighted merge of the K rows of each token."""
    if kernel == KernelType.TRITON_CC:
        raise NotImplementedError("TRITON_CC is not supported for silu_jagged_bmm_combine")
    require_hip_kernel(kernel, "silu_jagged_bmm_combine")
    N = index.shape[0]
    L, K = reverse_index.shape
    assert index.ndim == 1 and reverse_index.ndim == 2
    assert N == L * K and N == jagged.shape[0], f"{N=}, {L=}, {K=}, {jagged.shape=}"
    if _ag.needs_grad(jagged, weight, bias, gating_scores):
        return _ag.SiluJaggedBmmCombine.apply(offsets, jagged, weight, bias, index, reverse_index,
                                              gating_scores, gates_index, has_silu)
    bmm_out = ops.grouped_gemm(offsets, jagged, weight, total_rows=N, bias=bias, epilogue=EPI_NONE,
                               a_silu=has_silu)
    return ops.combine(bmm_out, reverse_index, gating_scores, gates_index)


def fused_jagged_bmm_swiglu_combine(
    offsets: torch.Tensor,
    index: torch.Tensor,
    jagged: torch.Tensor,
    weight: torch.Tensor,
    bias: Optional[torch.Tensor],
    weight_p: torch.Tensor,
    bias_p: Optional[torch.Tensor],
    weight_out: torch.Tensor,
    bias_out: Optional[torch.Tensor],
    k: int,
    gates: Optional[torch.Tensor] = None,
    gates_index: Optional[torch.Tensor] = None,
    kernel: KernelType = KernelType.HIP,
    *,
    checkpoint_bits: Optional[int] = None,
) -> torch.Tensor:
    """kernels/pytorch/moe.py:306-391 (pytorch_fused_jagged_bmm_swiglu_combine): the whole expert
    block of a SwiGLU MoE, ``merge_k(gates * ((silu(x W + b) * (x Wp + bp)) W_out + b_out))`` ->
    [L, D].  Three launches (gather + SwiGLU GEMM, down GEMM, merge); differentiable through the
    two operators it is made of.  ``checkpoint_bits=8``: the same values, but only the two pre-activations
    are kept for the backward pass, in 8 bits (``checkpoint_swiglu``), and the gradients are those of what the codes
    stand for: a third to a quarter of the memory, at errors of up to 1 / 128 of the largest of 32 neighbours."""
    require_hip_kernel(kernel, "fused_jagged_bmm_swiglu_combine")
    assert index.ndim == 2 and index.shape[1] == k, f"{index.shape=}, {k=}"
    if checkpoint_bits not in (None, 8):
        raise ValueError(f"fused_jagged_bmm_swiglu_combine: checkpoint_bits must be None or 8, got {checkpoint_bits}")
    if checkpoint_bits and _ag.needs_grad(jagged, weight, bias, weight_p, bias_p, weight_out, bias_out, gates):
        _check_gather_args("fused_jagged_bmm_swiglu_combine", index, jagged, weight)
        if weight_p.stride() != weight.stride():
            weight, weight_p = weight.contiguous(), weight_p.contiguous()
        return _ag.SwigluBlockCheckpoint8.apply(offsets, index, jagged, weight, bias, weight_p, bias_p, weight_out, bias_out, gates, gates_index,
                                                ops.invert_index(index))
    hidden = index_select_jagged_bmm_swiglu(0, offsets, index, jagged, weight, bias, weight_p, bias_p, kernel)
    token_index = torch.div(index.reshape(-1), k, rounding_mode="floor")
    reverse_index = ops.invert_index(index)
    return silu_jagged_bmm_combine(0, offsets, hidden, weight_out, bias_out, token_index, reverse_index,
                                   gates, gates_index, has_silu=False, kernel=kernel)


def fused_moe_few_tokens(
    x: torch.Tensor,
    gate_weight: torch.Tensor,
    gate_bias: Optional[torch.Tensor],
    weight: torch.Tensor,
    bias: Optional[torch.Tensor],
    weight_p: Optional[torch.Tensor],
    bias_p: Optional[torch.Tensor],
    weight_out: torch.Tensor,
    bias_out: Optional[torch.Tensor],
    k: int,
    renorm: bool = True,
    token_mask: Optional[torch.Tensor] = None,
    kernel: KernelType = KernelType.HIP,
) -> torch.Tensor:
    """A whole MoE layer for up to 64 tokens (a decode step) in two or three launches, [T, D] -> [T, O]: router
    ``softmax(x gate_weight^T + gate_bias)``, the ``k`` largest of every token (``renorm``: divided by their sum), and
    ``sum_j g_j * (act(x W[e_j] + bias[e_j]) W_out[e_j] + bias_out[e_j])`` with ``act(a) = silu(a)``, or
    ``silu(a) * (x W_p[e_j] + bias_p[e_j])`` when ``weight_p`` is given.

    No counterpart in the reference.  What FastMoELayer.forward and fused_jagged_bmm_swiglu_combine compute, for the batch
    sizes where the time is that of the launches and of reading the chosen experts' weights; logits are not rounded to
    the tokens' type here, so that a near tie may fall the other way.  gate_weight is [E, D] (``nn.Linear.weight``), the expert weights
    [E, D_in, D_out] views of [E, D_out, D_in] storage, everything in x's dtype (bf16 or fp32).  ``token_mask`` (bool [T]):
    rows where it is False read no expert and come out as zeros (the padding of a captured decode batch).  Forward only."""
    require_hip_kernel(kernel, "fused_moe_few_tokens")
    ops._forward_only("fused_moe_few_tokens", x, gate_weight, gate_bias, weight, bias, weight_p, bias_p, weight_out, bias_out)
    return ops.few_tokens(x, gate_weight, gate_bias, weight, bias, weight_p, bias_p, weight_out, bias_out, k, renorm, token_mask)


# ------------------------------------------------------------ around the expert block
def _norm_call(index, reverse_index, merge_index, merge, y, residual, args: ops.NormArgs):
    tensors = [merge, y, residual, *args[:3], args.scale if isinstance(args.scale, torch.Tensor) else None, args.next_weight, args.next_bias]
    if _ag.needs_grad(*tensors):
        return _ag.NormAdd.apply(index, reverse_index, merge_index, merge, y, residual, args.weight, args.bias, args.gate, args.scale,
                                 args.next_weight, args.next_bias, args.gate_sigmoid, args.eps, args.norm)
    return ops.norm_add(y, residual, args, reverse_index, merge, merge_index)[:2]


def block_norm(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *, eps: float = 1e-6, norm: str = "rms",
               kernel: KernelType = KernelType.HIP) -> torch.Tensor:
    """The norm before the first block: ``norm(x) * weight + bias`` over the last dimension of x [T, D] (bf16 or fp32, up to 8192
    columns), ``norm`` = "rms" or "layer"; fp32 inside, rounded once.  Differentiable.  No counterpart in the reference."""
    require_hip_kernel(kernel, "block_norm")
    return _norm_call(None, None, None, None, None, x, ops.NormArgs(next_weight=weight, next_bias=bias, eps=eps, norm=norm))[1]


def block_norm_add(y: torch.Tensor, residual: torch.Tensor, *, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                   gate: Optional[torch.Tensor] = None, gate_sigmoid: bool = False, scale: Union[torch.Tensor, float, None] = None,
                   next_weight: Optional[torch.Tensor] = None, next_bias: Optional[torch.Tensor] = None, eps: float = 1e-6, norm: str = "rms",
                   kernel: KernelType = KernelType.HIP) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Between two blocks: ``out = residual + scale * gate * (norm(y) * weight + bias)`` and ``next = norm(out) * next_weight + next_bias``,
    in one pass; returns (out, next), next None without ``next_weight``.  y, residual [T, D] of one dtype (bf16 or fp32, up to 8192
    columns).  Without ``weight`` y is not normed.  ``gate``: [T] or [T, 1] (a gate per token) or [T, D], in their dtype, behind a sigmoid
    with ``gate_sigmoid``.  ``scale``: [D] or a number.  scale, weights and biases share one dtype, bf16 or fp32.  fp32 inside, each output
    rounded once, ``next`` from the unrounded out.  Differentiable in every tensor.  No counterpart in the reference."""
    require_hip_kernel(kernel, "block_norm_add")
    return _norm_call(None, None, None, None, y, residual,
                      ops.NormArgs(weight, bias, gate, gate_sigmoid, scale, next_weight, next_bias, eps, norm))


def mul_merge_k_norm_add(index: torch.Tensor, reverse_index: torch.Tensor, value: torch.Tensor, residual: torch.Tensor,
                         merge_weight: Optional[torch.Tensor] = None, weight_index: Optional[torch.Tensor] = None, *,
                         weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
                         gate_sigmoid: bool = False, scale: Union[torch.Tensor, float, None] = None,
                         next_weight: Optional[torch.Tensor] = None, next_bias: Optional[torch.Tensor] = None, eps: float = 1e-6,
                         norm: str = "rms", kernel: KernelType = KernelType.HIP) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """``block_norm_add`` of the merge of an expert block's rows, without the merged rows' round trip: y is
    ``mul_merge_k_add(index, reverse_index, value, weight=merge_weight, weight_index=weight_index)`` (index: the token of every row),
    summed in fp32 and not rounded.  For the backward pass the merged rows are kept in fp32."""
    require_hip_kernel(kernel, "mul_merge_k_norm_add")
    N = index.shape[0]
    L, K = reverse_index.shape
    assert index.ndim == 1 and N == L * K and N == value.shape[0] and L == residual.shape[0], (
        f"mul_merge_k_norm_add: {index.shape=}, {reverse_index.shape=}, {value.shape=}, {residual.shape=}")
    assert merge_weight is None or (weight_index is not None and merge_weight.numel() == weight_index.numel() == N), (
        "mul_merge_k_norm_add: merge_weight and weight_index need an entry per row")
    return _norm_call(index, reverse_index, weight_index, merge_weight, value, residual,
                      ops.NormArgs(weight, bias, gate, gate_sigmoid, scale, next_weight, next_bias, eps, norm))


# ------------------------------------------------------- activation checkpoints in 8 bits
SwigluCheckpoint = ops.SwigluCheckpoint


def checkpoint_swiglu(gate: torch.Tensor, up: torch.Tensor, kernel: KernelType = KernelType.HIP) -> SwigluCheckpoint:
    """The two pre-activations [R, H] of a SwiGLU expert block (bf16 or fp32) in 8 bits: blocks of 32 neighbours under a shared power of
    two (MXINT8), 33 / 32 bytes a value.  A block holding an infinity or NaN reads as NaN.  Forward only (what it keeps stands in for the
    saved tensors of a backward pass).  No counterpart in the reference, which keeps both in their own dtype."""
    require_hip_kernel(kernel, "checkpoint_swiglu")
    ops._forward_only("checkpoint_swiglu", gate, up)
    return ops.swiglu_checkpoint(gate, up)


def read_checkpoint(kept: SwigluCheckpoint, kernel: KernelType = KernelType.HIP) -> Tuple[torch.Tensor, torch.Tensor]:
    """(gate, up) that the codes stand for, in the dtype they had; exact in bf16."""
    require_hip_kernel(kernel, "read_checkpoint")
    return ops.swiglu_checkpoint_read(kept)


def swiglu_checkpoint_bwd(kept: SwigluCheckpoint, d_hidden: torch.Tensor, row_weight: Optional[torch.Tensor] = None,
                          kernel: KernelType = KernelType.HIP) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Backward of ``w * silu(gate) * up`` from the checkpoint, in one pass: d_hidden [R, H] is the gradient of the hidden rows behind the
    rows' weights w ([R], bf16 or fp32; None: 1).  -> (d_gate, d_up, w * hidden, d_w fp32 [R])."""
    require_hip_kernel(kernel, "swiglu_checkpoint_bwd")
    ops._forward_only("swiglu_checkpoint_bwd", d_hidden, row_weight)
    return ops.swiglu_checkpoint_bwd(kept, d_hidden, row_weight)
