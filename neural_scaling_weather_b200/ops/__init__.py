"""Fused operators of the weather transformer.

Each public function takes PyTorch tensors and returns PyTorch tensors with autograd.
CPU tensors run the plain-PyTorch oracle in :mod:`.reference`.  CUDA tensors run the
hand-written sm_100a kernels of the ``_C`` extension (tcgen05/TMEM GEMMs with fused
epilogues, windowed attention with fused QK-norm, shift and mask, fused norms, loss and
optimizer kernels); a CUDA call without the extension raises.

Compute precision on CUDA follows ``torch.autocast``: inside an autocast region (the
trainer uses one, as the reference does) activations are bf16 (or fp16); parameters stay
fp32 masters and are cast once per optimizer step into a cached low-precision copy.  The
kernels compute in 16 bits, so fp32 CUDA inputs outside autocast are also computed in bf16;
for fp32 arithmetic on the GPU (fp32 inference, as the reference runs it) wrap the call in
:func:`reference_ops`, which sends CUDA tensors through the plain-PyTorch oracle too.
"""

from __future__ import annotations

import contextlib
import threading
from typing import Optional, Sequence, Union

import torch

from . import fused, reference
from ._ext import available as extension_available
from ._ext import require as require_extension
from .geometry import WindowGeometry

TensorOrParts = Union[torch.Tensor, Sequence[torch.Tensor]]


def compute_dtype(t: torch.Tensor) -> torch.dtype:
    """Activation dtype of a CUDA op: the autocast dtype if active, else the input dtype."""
    if t.is_cuda and torch.is_autocast_enabled("cuda"):
        return torch.get_autocast_dtype("cuda")
    return t.dtype


_mode = threading.local()


@contextlib.contextmanager
def reference_ops():
    """Within this context every operator runs the plain-PyTorch oracle (:mod:`.reference`),
    on CUDA tensors too, in the tensors' own precision (fp32 math for fp32 inputs)."""
    prev = getattr(_mode, "reference", False)
    _mode.reference = True
    try:
        yield
    finally:
        _mode.reference = prev


def _use_cuda(t: torch.Tensor) -> bool:
    if not t.is_cuda or getattr(_mode, "reference", False):
        return False
    require_extension()
    return True


def _cat(parts):
    if isinstance(parts, torch.Tensor) or parts is None:
        return parts
    parts = list(parts)
    return parts[0] if len(parts) == 1 else torch.cat(parts, dim=0)


def rms_norm(x: torch.Tensor, w: torch.Tensor, eps: Optional[float] = None) -> torch.Tensor:
    if not _use_cuda(x):
        return reference.rms_norm(x, w, eps)
    from .fused import rms_norm_cuda

    return rms_norm_cuda(x, w, eps)


def rms_norm_with_skip(x: torch.Tensor, w: torch.Tensor, eps: Optional[float] = None):
    """``(rms_norm(x, w), x)``: the pre-norm block input and its skip connection from one
    autograd node, so their gradients are summed inside the RMSNorm backward on CUDA."""
    if not _use_cuda(x):
        return reference.rms_norm(x, w, eps), x
    from .fused import rms_norm_skip_cuda

    return rms_norm_skip_cuda(x, w, eps)


def linear_allreduce(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                     residual: Optional[torch.Tensor] = None, group: str = "tp") -> torch.Tensor:
    """Row-parallel linear: ``all_reduce_group(x W^T) + bias + residual``.  On CUDA with a
    symmetric-memory group of 2..8 GPUs the all-reduce runs inside the GEMM's epilogue over
    NVLink peer memory; otherwise GEMM, then the NCCL all-reduce mapping, then the adds."""
    from ..parallel import symm
    from ..parallel.mappings import allreduce_forward_identity_backward

    if _use_cuda(x) and symm.available(group):
        from .fused import linear_allreduce_cuda

        return linear_allreduce_cuda(x, weight, bias, residual, group)
    y = linear(x, weight)
    y = allreduce_forward_identity_backward(y, group)
    if bias is not None:
        y = y + bias.to(y.dtype)
    return y if residual is None else y + residual


def linear_colparallel(x: torch.Tensor, weight: TensorOrParts, bias: Optional[TensorOrParts] = None,
                       activation: Optional[str] = None, group: str = "tp") -> torch.Tensor:
    """Column-parallel linear of a replicated input: ``act(x W_local^T + b_local)``, whose input
    gradient is all-reduced over ``group`` (the reference's ``copy_to_parallel_region`` followed by
    the linear).  On CUDA with a symmetric-memory group of 2..8 GPUs the all-reduce runs inside the
    data-gradient GEMM's epilogue over NVLink; otherwise the NCCL mapping wraps the linear."""
    from ..parallel import comm, symm
    from ..parallel.mappings import identity_forward_allreduce_backward

    if comm.get_size(group) > 1 and _use_cuda(x) and symm.available(group):
        from .fused import linear_cuda

        return linear_cuda(x, weight, bias, None, activation, allreduce_group=group)
    x = identity_forward_allreduce_backward(x, group)
    return linear(x, weight, bias, activation=activation)


def linear(x: torch.Tensor, weight: TensorOrParts, bias: Optional[TensorOrParts] = None,
           residual: Optional[torch.Tensor] = None, activation: Optional[str] = None):
    """``act(x W^T + b) + residual``; ``weight``/``bias`` may be lists concatenated on N."""
    if not _use_cuda(x):
        return reference.linear(x, _cat(weight), _cat(bias), residual, activation)
    from .fused import linear_cuda

    return linear_cuda(x, weight, bias, residual, activation)


def mlp(x: torch.Tensor, w1: torch.Tensor, b1: torch.Tensor, w2: torch.Tensor, b2: torch.Tensor,
        residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``fc2(GELU(fc1(x))) + residual`` with biases (fused backward on CUDA)."""
    if not _use_cuda(x):
        h = reference.linear(x, w1, b1, activation="gelu")
        return reference.linear(h, w2, b2, residual=residual)
    from .fused import mlp_cuda

    return mlp_cuda(x, w1, b1, w2, b2, residual)


GATED_ACTIVATIONS = ("silu", "gelu")


def gated_mlp(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor,
              b_gate: Optional[torch.Tensor] = None, b_up: Optional[torch.Tensor] = None,
              b_down: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
              activation: str = "silu") -> torch.Tensor:
    """Gated feed-forward network ``(act(x Wg^T + bg) * (x Wu^T + bu)) Wd^T + bd + residual``.

    ``x`` (..., K); ``w_gate`` and ``w_up`` (H, K), ``w_down`` (N, H); biases (H,), (H,), (N,) or None;
    ``residual`` (..., N).  ``activation``: ``"silu"`` or ``"gelu"`` (exact).  Any sizes and strides; rows whose
    strides are not multiples of 16 bytes cost one copy of the operand.  On CUDA the hidden values are 16-bit (in fp16
    they overflow past 65504), and the gate's and the up projection's biases share a type.  On CUDA both projections, the
    activation and the product are one kernel; the backward's data gradients read the weights as they are
    stored.  Calls without gradients of at most 16 rows take kernels that stream the weights once."""
    if activation not in GATED_ACTIVATIONS:
        raise ValueError(f"gated_mlp: activation {activation!r} is not one of {GATED_ACTIVATIONS}")
    if _use_cuda(x):  # checks the shapes itself
        return fused.gated_mlp_cuda(x, w_gate, w_up, w_down, b_gate, b_up, b_down, residual, activation)
    fused.check_gated_shapes(x, w_gate, w_up, w_down, residual)
    return reference.gated_mlp(x, w_gate, w_up, w_down, b_gate, b_up, b_down, residual, activation)


def route_tokens(logits: torch.Tensor, top_k: int, normalize: bool = True):
    """The router of a block with routed experts: ``(weights, experts, balance)`` from ``logits`` (..., E).

    ``experts`` (..., top_k, int64) are the indices of each token's largest logits, in falling order, of equal ones the
    lower index first.  ``weights`` (..., top_k, fp32) are a softmax over the chosen logits, or with ``normalize=False``
    their values in the softmax over all.  ``balance`` (a scalar) is ``E sum_e f_e P_e``, the share of the choices that
    fell on an expert times its mean probability: 1 where both are even; its gradient is that of the probabilities.
    A masked expert has the logit -inf; a token whose logits are all -inf has weights of zero.  On CUDA bf16, fp16 or
    fp32 logits, at most 512 experts and 16 choices.  First derivatives in reverse mode."""
    if logits.dim() < 1 or not 1 <= top_k <= logits.shape[-1]:
        raise ValueError(f"route_tokens: top_k {top_k} of logits {tuple(logits.shape)}")
    if _use_cuda(logits):
        if logits.dtype not in fused.DT:
            raise TypeError(f"route_tokens: logits of {logits.dtype} on CUDA (bf16, fp16 or fp32)")
        return require_extension().route_tokens(logits, top_k, normalize)
    return reference.route_tokens(logits, top_k, normalize)


def expert_mlp(x: torch.Tensor, weights: torch.Tensor, experts: torch.Tensor, w_gate: torch.Tensor,
               w_up: torch.Tensor, w_down: torch.Tensor, residual: Optional[torch.Tensor] = None,
               activation: str = "silu") -> torch.Tensor:
    """Routed gated feed-forward networks: ``y_t = sum_j weights[t, j] MLP_experts[t, j](x_t) + residual_t`` with
    ``MLP_e(x) = (act(x Wg_e^T) * (x Wu_e^T)) Wd_e^T``.

    ``x`` (..., K); ``weights`` and ``experts`` (..., k) as :func:`route_tokens` returns them (any integer and floating
    types; an index outside ``0 .. E - 1`` leaves its assignment out, an index that is there twice counts twice);
    ``w_gate`` and ``w_up`` (E, H, K), ``w_down`` (E, N, H); ``residual`` (..., N).  ``activation``: ``"silu"`` or
    ``"gelu"`` (exact).  Gradients of everything but the indices, each in its tensor's type; first derivatives in
    reverse mode.  Any sizes and strides on CUDA (weights whose rows are not multiples of 16 bytes are copied once a
    call), at most 512 experts, 16 a token.  The hidden values, the experts' outputs and, in the backward, the weighted
    gradients of the output and those of the hidden values are 16-bit there (in fp16 they overflow past 65504 and lose
    bits below 6e-5: scale the loss).  The rows are sorted by expert on the device (nothing waits for it) and the products
    run grouped by expert; calls without gradients have forms of their own for a few assignments and for few rows an
    expert."""
    if activation not in GATED_ACTIVATIONS:
        raise ValueError(f"expert_mlp: activation {activation!r} is not one of {GATED_ACTIVATIONS}")
    if _use_cuda(x):
        return fused.expert_mlp_cuda(x, weights, experts, w_gate, w_up, w_down, residual, activation)
    fused.check_expert_ids(experts)
    fused.check_expert_shapes(x, weights, experts, w_gate, w_up, w_down, residual)
    return reference.expert_mlp(x, weights, experts, w_gate, w_up, w_down, residual, activation)


def norm_gate_residual(y: torch.Tensor, skip: torch.Tensor, w_post: torch.Tensor,
                       gate: Optional[torch.Tensor] = None, w_next: Optional[torch.Tensor] = None,
                       skip_scale: float = 1.0, eps: Optional[float] = None):
    """The norms around a residual connection in one pass: ``(s, n)`` with
    ``s = skip_scale skip + gate * rms_norm(y, w_post)`` and ``n = rms_norm(s, w_next)``.

    ``y`` (a branch's output) and ``skip`` (..., D); ``w_post``, ``w_next`` (D,); ``gate`` (D,), or one row for
    each index of the first dimension (samples, D; at most 65535 on CUDA, made for a batch's few: the backward takes
    1.3 us a sample), or None for ones.  D is at most 16384 on CUDA.  ``n`` is None without ``w_next`` (the last branch
    of a network)."""
    if _use_cuda(y):  # checks the shapes itself
        return fused.norm_gate_residual_cuda(y, skip, w_post, gate, w_next, skip_scale, eps)
    D = y.shape[-1]
    if y.dim() < 2 or skip.shape != y.shape:
        raise ValueError(f"norm_gate_residual: y {tuple(y.shape)} and skip {tuple(skip.shape)} must be of one shape "
                         "(..., D)")
    if w_post.shape != (D,) or (w_next is not None and w_next.shape != (D,)):
        raise ValueError(f"norm_gate_residual: w_post and w_next must be ({D},)")
    if gate is not None and gate.shape not in ((D,), (y.shape[0], D)):
        raise ValueError(f"norm_gate_residual: gate {tuple(gate.shape)} is neither ({D},) nor ({y.shape[0]}, {D})")
    return reference.norm_gate_residual(y, skip, w_post, gate, w_next, skip_scale, eps)


def clip_grad_norm(grads: Sequence[torch.Tensor], max_norm: float,
                   out: Optional[Sequence[torch.Tensor]] = None) -> torch.Tensor:
    """Scale ``grads`` (separate tensors, fp32 / bf16 / fp16 mixed freely) to a global L2 norm of at most
    ``max_norm``, in place or into ``out``; returns the norm before clipping (an fp32 scalar tensor; nothing
    waits for the device).  On CUDA the tensors are contiguous, and none overlaps what another one writes.  The factor is the trainer's: ``max_norm / (norm + 1e-6)`` where the norm exceeds
    ``max_norm``, else 1 (also for a NaN norm: non-finite gradients stay visible)."""
    if isinstance(grads, torch.Tensor):
        grads = [grads]
    if len(grads) == 0:
        raise ValueError("clip_grad_norm: no tensors")
    if not max_norm > 0:
        raise ValueError(f"clip_grad_norm: max_norm must be positive, got {max_norm}")
    if out is not None and len(out) != len(grads):
        raise ValueError(f"clip_grad_norm: {len(out)} outputs for {len(grads)} tensors")
    if not _use_cuda(grads[0]):
        with torch.no_grad():
            return reference.clip_grad_norm(grads, max_norm, out)
    return require_extension().clip_grads(grads, max_norm, [] if out is None else out)


def window_attention(qkv: torch.Tensor, q_norm_w: torch.Tensor, k_norm_w: torch.Tensor,
                     num_heads: int, head_dim: int, geom: WindowGeometry, scale: float,
                     rel_bias: Optional[torch.Tensor] = None):
    """Shifted-window attention over (B, T, H, W, 3*nh*hd) -> (B, T, H, W, nh*hd).

    ``rel_bias`` (nh, ``geom.num_buckets(T)``), of any float type and strides: a learned bias that is added to the logits by
    head and displacement of query and key, entry ``geom.relative_buckets(T)[i, j]``; with its gradient.  Entries of -inf
    mask displacements; a query that has none left is zero."""
    if not _use_cuda(qkv):
        fused.check_rel_bias(rel_bias, num_heads, geom, qkv.shape[1])
        return reference.window_attention(qkv, q_norm_w, k_norm_w, num_heads, head_dim, geom, scale, rel_bias)
    return fused.window_attention_cuda(qkv, q_norm_w, k_norm_w, num_heads, head_dim, geom, scale, rel_bias)


def patch_embed(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor],
                patch_size: int, add: Optional[torch.Tensor] = None):
    """(N, C, H, W) -> (N, h, w, E); ``add`` (P, h, w, E) is broadcast over N // P."""
    if not _use_cuda(x):
        return reference.patch_embed(x, weight, bias, patch_size, add)
    from .fused import patch_embed_cuda

    return patch_embed_cuda(x, weight, bias, patch_size, add)


def coord_pos_embed(coords: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor],
                    patch_size: int) -> torch.Tensor:
    """Patch projection of a constant coordinate field (T, 4, H, W) -> (T, h, w, E): on CUDA computed
    once per weight version and reused by every forward until the next optimizer step."""
    if not _use_cuda(coords):
        return reference.patch_embed(coords, weight, bias, patch_size)
    from .fused import coord_pos_embed_cuda

    return coord_pos_embed_cuda(coords, weight, bias, patch_size)


def head_unpatchify(x: torch.Tensor, weight: torch.Tensor, patch_size: int, out_chans: int):
    """(B, T, h, w, E) -> (B, T, C, h*p, w*p)."""
    if not _use_cuda(x):
        return reference.head_unpatchify(x, weight, patch_size, out_chans)
    from .fused import head_unpatchify_cuda

    return head_unpatchify_cuda(x, weight, patch_size, out_chans)


def weighted_sse(x: torch.Tensor, y: torch.Tensor, area_w: Optional[torch.Tensor] = None,
                 ch_w: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Scalar sum of ``(x-y)^2 * area_w[h,1] * ch_w[c,1,1]`` (fp32)."""
    if not _use_cuda(x):
        return reference.weighted_sse(x, y, area_w, ch_w)
    from .fused import weighted_sse_cuda

    return weighted_sse_cuda(x, y, area_w, ch_w)


def weighted_se_per_channel(x: torch.Tensor, y: torch.Tensor, area_w: torch.Tensor):
    """``sum_{h,w} area_w * (x-y)^2`` keeping the leading dims (fp32)."""
    if not _use_cuda(x):
        return reference.weighted_se_per_channel(x, y, area_w)
    from .fused import weighted_se_per_channel_cuda

    return weighted_se_per_channel_cuda(x, y, area_w)


__all__ = [
    "WindowGeometry",
    "clip_grad_norm",
    "compute_dtype",
    "expert_mlp",
    "extension_available",
    "gated_mlp",
    "head_unpatchify",
    "linear",
    "mlp",
    "norm_gate_residual",
    "patch_embed",
    "reference",
    "rms_norm",
    "route_tokens",
    "weighted_se_per_channel",
    "weighted_sse",
    "window_attention",
]
