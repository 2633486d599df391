"""SwiGLU experts for the few tokens of a decoding step (no reference
counterpart: there the pieces are permute, two grouped GEMMs, the activation and
unpermute, which is also the way to go here for many tokens)."""

from __future__ import annotations

from typing import Optional

import torch

from primus_turbo.pytorch.kernels.moe.moe_decode_impl import moe_decode_impl

__all__ = ["moe_decode"]


@torch._dynamo.disable
def moe_decode(
    x: torch.Tensor,
    w_gate_up: torch.Tensor,
    w_down: torch.Tensor,
    topk_idx: torch.Tensor,
    topk_probs: torch.Tensor,
    gate_up_scale_inv: Optional[torch.Tensor] = None,
    down_scale_inv: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """y[t] = sum_j topk_probs[t, j] * Wd_e (silu(Wg_e x[t]) * (Wu_e x[t])), e = topk_idx[t, j].

    ``x``: [T, H] bfloat16 / float16.  ``w_gate_up``: [E, 2 I, H], the gate's
    rows, then the up projection's; ``w_down``: [E, H, I] (the layouts of
    ``grouped_gemm_fp8`` with ``trans_b=True``).  Both are one of

    - QuantizedTensors as ``create_quantized_weight`` makes them (TENSORWISE,
      ROWWISE along the last axis, or BLOCKWISE 128 x 128);
    - fp8 tensors with ``gate_up_scale_inv`` / ``down_scale_inv`` in the same
      layouts: one value, [E, rows, 1], or [E, ceil(rows / 128), ceil(columns / 128)];
    - tensors of x's type.

    ``topk_idx``: [T, k] int32 / int64 as for ``moe_permute``; entries outside
    [0, E) (another rank's experts) add nothing.  ``topk_probs``: [T, k] float32.

    H and I are multiples of 16, E <= 1024, k <= 32.  The tokens are not
    quantized; silu(gate) * up * prob is rounded to x's type between the two
    products, everything else is summed in fp32.  Each reached expert's weights
    are read once for every 64 tokens, which makes this the path for small T;
    for many tokens use moe_permute and grouped_gemm_fp8.  Inference only: a
    tensor that needs gradients, a weight too, is refused outside torch.no_grad().
    Under torch.compile the call runs between its graphs.
    """
    return moe_decode_impl(x, w_gate_up, w_down, topk_idx, topk_probs, gate_up_scale_inv, down_scale_inv)
