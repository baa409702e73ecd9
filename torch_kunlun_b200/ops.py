"""Fused operators of the kunlun backend that have no single aten name.

* ``linear(x, w, b, act)`` -- act(x @ w^T + b) in one quantised GEMM launch;
  the activation is applied to the rounded, bias-added output, i.e. the same
  values the reference produces with linear followed by a separate
  relu / gelu / silu launch (csrc/ops.cpp:480-495, :151-160,
  csrc/ops_nn.cpp:132-147, csrc/ops_extra.cpp:71).
* ``silu_mul(gate, up)`` -- T(silu(gate)) * up, the gated-MLP product, in one
  elementwise pass.
* ``dropout``, ``residual_norm`` -- differentiable training operators: dropout
  whose mask is a function of (seed, offset, element index) and is never
  stored, and the norms behind and before a transformer block with the block's
  dropout, gate and residual scale in one pass.
* ``linear_cross_entropy`` -- the loss of a vocabulary projection and its
  gradients without the logits.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _C

ACT = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4, "silu_gate": 5}


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
           act: str = "none", residual: Optional[torch.Tensor] = None,
           amax_x: Optional[torch.Tensor] = None,
           amax_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """act(x @ w^T + b) [+ residual]: with a residual the epilogue adds it
    after the bias (rounded to T), giving the values of linear followed by a
    separate add (csrc/ops.cpp:480-495 then csrc/ops.cpp:117-149).

    amax_x (1-element fp32) is x's per-tensor scale when the caller already
    has it (skips the pass over x); amax_out (1-element fp32, written)
    receives max |y| — folded into the fp16 epilogue where it applies, one
    pass over y otherwise — so the GEMM that consumes y skips its own pass.
    """
    return _C.linear_act(x, weight, bias, ACT[act], residual, amax_x, amax_out)


def silu_mul(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    return _C.silu_mul(gate, up)


def amax(x: torch.Tensor) -> torch.Tensor:
    """max |x| as a 1-element fp32 tensor on x's device (the per-tensor scale)."""
    return _C.amax(x)


def linear_scaled(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                  act: str = "none", amax_x: Optional[torch.Tensor] = None,
                  amax_w: Optional[torch.Tensor] = None,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``linear`` with given per-tensor scales; row blocks of x with the whole
    x's amax reproduce one unsplit call exactly."""
    return _C.linear_scaled(x, weight, bias, ACT[act], amax_x, amax_w, out)


def silu_mul_amax(gate: torch.Tensor, up: torch.Tensor):
    """(T(silu(gate)) * up, its max |value| as a 1-element fp32 tensor) in
    one pass: the gated activation and the scale the next GEMM quantises it
    with."""
    return _C.silu_mul_amax(gate, up)


def quantize_limbs(x: torch.Tensor, amax: torch.Tensor) -> torch.Tensor:
    """The int16 codes of a 2-D tensor under a given per-tensor scale, as two
    int8 limb planes [2, rows, round_up(cols, 16)] (hi signed, lo unsigned):
    an operand several GEMMs share is quantised once."""
    return _C.quantize_limbs(x, amax)


def linear_from_limbs(a_limbs: torch.Tensor, b_limbs: torch.Tensor, k: int, amax_a: torch.Tensor,
                      amax_b: torch.Tensor, bias: Optional[torch.Tensor] = None, act: str = "none",
                      out: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.float16,
                      gate: Optional[torch.Tensor] = None,
                      amax_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """act(a b^T + bias) on operands from quantize_limbs: the values of
    linear_scaled(a, b, amax_x=amax_a, amax_w=amax_b) (K <= 32768).

    act="silu_gate" with `gate` [M, N]: T(silu(gate)) * (a b^T + bias), each
    product rounded once -- silu_mul(gate, up) fused into the up projection.
    amax_out (1-element fp32, written) receives max |y| from the epilogue
    (fp16 outputs on the vector path)."""
    return _C.linear_from_limbs(a_limbs, b_limbs, k, amax_a, amax_b, bias, ACT[act], out, dtype, gate, amax_out)


def _u64(value: int, name: str) -> int:
    value = int(value)
    if not 0 <= value < 1 << 64:
        raise ValueError(f"{name} must be in [0, 2**64), got {value}")
    return value


def dropout(x: torch.Tensor, p: float, seed: int, offset: int = 0) -> torch.Tensor:
    """x / (1 - p) where the element is kept, 0 elsewhere (also for inf and
    NaN).  Element i, in row-major order, is kept when word i % 4 of the
    Philox4x32-10 block with counter (i // 4, offset) and key seed is at least
    round(p * 2**32).  The same (seed, offset) gives the same mask on every call
    and in the backward pass, so give each call of a step an offset of its
    own.  0 <= p <= 1; float16 and float32."""
    return _C.dropout(x, float(p), _u64(seed, "seed"), _u64(offset, "offset"))


def residual_norm(x: torch.Tensor, f: torch.Tensor, weight: Optional[torch.Tensor] = None,
                  bias: Optional[torch.Tensor] = None, *, norm: str = "layer", post_norm: bool = False,
                  post_weight: Optional[torch.Tensor] = None, post_bias: Optional[torch.Tensor] = None,
                  gate: Optional[torch.Tensor] = None, residual_scale: float = 1.0, eps: float = 1e-5,
                  p: float = 0.0, seed: int = 0, offset: int = 0):
    """(x_new, h) for a residual stream x and a block's output f [..., D]:

        u     = Norm(f) * post_weight + post_bias if post_norm else f
        x_new = residual_scale * x + gate * dropout(u, p, seed, offset)
        h     = Norm(x_new) * weight + bias

    Norm is "layer" (mean and variance) or "rms" (mean square), with eps under
    the root.  h is the next block's input; a post-LayerNorm block takes h alone.
    gate is [D], or x's shape with 1 in place of some last dimensions before D
    ([B, 1, D] gates each sample).  All tensors share one dtype, float16 or
    float32; sums are fp32 (of the unrounded x_new for h) and each output is
    rounded once.  D is at most 32768.  Differentiable in every tensor; the
    backward pass forms the mask and the unrounded x_new again from x and f."""
    if norm not in ("layer", "rms"):
        raise ValueError(f"norm must be 'layer' or 'rms', got {norm!r}")
    return _C.residual_norm(x, f, weight, bias, norm == "rms", bool(post_norm), post_weight, post_bias, gate,
                            float(residual_scale), float(eps), float(p), _u64(seed, "seed"),
                            _u64(offset, "offset"))


REDUCTION = {"none": 0, "mean": 1, "sum": 2}


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor,
                         bias: Optional[torch.Tensor] = None, ignore_index: int = -100,
                         reduction: str = "mean") -> torch.Tensor:
    """cross_entropy(x @ weight^T + bias, target) without the logits, in fp32.

    x [..., D], weight [V, D] and bias [V] share one dtype, float16 or float32;
    target [...] is int64.  Rows whose target is ignore_index take no part (loss
    and gradient 0, whatever x holds there) and cost nothing; any other target
    outside [0, V) makes its loss NaN.  reduction is "mean" (over the rows with a
    target), "sum" or "none" (target's shape); a row's loss and its row of x's
    gradient depend on that row alone.  Products are those of the tensors' own
    values (float32 to 22 bits) summed in fp32, not the int16-quantised ones of
    ``linear``.  In the backward pass softmax - onehot is held to 11 bits for
    float16 and 22 for float32, and an entry of any size may be 2**-39 off.
    Differentiable in x, weight and bias."""
    if reduction not in REDUCTION:
        raise ValueError(f"reduction must be one of {sorted(REDUCTION)}, got {reduction!r}")
    return _C.linear_cross_entropy(x, weight, target, bias, int(ignore_index), REDUCTION[reduction])


__all__ = ["linear", "dropout", "residual_norm", "linear_cross_entropy", "silu_mul", "silu_mul_amax", "amax", "linear_scaled", "quantize_limbs",
           "linear_from_limbs", "ACT"]
