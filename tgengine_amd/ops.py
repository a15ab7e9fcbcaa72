"""Operators of a temporal attention model on prepared batches, as HIP kernels.

What a model does with the neighbours that ``DataPipeline.prepare`` gathers:

* ``embed``: rows of a learned node table for ``NeighborData.neighbor_ids``,
  scaled; the gradient is summed by sorted ids.
* ``layer_norm``: over the tokens' channels, with the gradients of tokens,
  weight and bias.
* ``cross_attention``: query tokens to the states of another sequence under
  ``NeighborData.mask``, from one query per node to long sequences on both sides.
* ``clip_grad_norm_``: the global norm of all gradients, and clipping by it.

Tensors are float32 or bfloat16 on the GPU; sums and statistics are held in 32
bits.  Every call launches on the caller's current stream and does not wait for
the device; the same inputs give the same bits.  The first three take part in
autograd (once: their backward passes leave no graph; forward-mode derivatives and
tracing are refused).  There is no CPU path.
"""
from __future__ import annotations

from typing import Iterable, Optional, Sequence, Tuple, Union

import torch
from torch import Tensor

from tgengine_amd.core.temporal_graph import _host


def embed(table: Tensor, ids: Tensor, scale: float = 1.0) -> Tensor:
    """``scale * table[ids]``: (*ids.shape, dim) in the table's dtype.

    ids are int32 or int64 of any shape; one outside [0, rows), such as the -1 of a
    padded neighbour slot, gives zeros and takes no gradient.  The table's gradient
    is dense, (rows, dim).
    """
    return _host().embed(table, ids, scale)


def layer_norm(x: Tensor, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None,
               eps: float = 1e-5) -> Tensor:
    """Layer norm over the last dimension (1 to 16,384 values) of x.

    weight and bias are (dim,), both of one dtype, which may be float32 beside
    bfloat16 tokens; either may be left out.
    """
    return _host().layer_norm(x, weight, bias, eps)


def cross_attention(q: Tensor, k: Tensor, v: Tensor, mask: Optional[Tensor] = None,
                    scale: Optional[float] = None) -> Tensor:
    """softmax(scale * q k^T) v over the keys that ``mask`` keeps: (B, Lq, H, D).

    q is (B, Lq, H, D), k and v are (B, Lk, Hkv, D) with H a multiple of Hkv (query
    head h reads head h // (H // Hkv)) and D up to 256; any strides with a dense last
    dimension are read in place, broadcast ones too.  mask is (B, Lk), True where a
    key takes part: the k and v of the others are not used, whatever they hold, and a
    row that keeps no key gives zeros and takes no gradient.  scale defaults to
    D ** -0.5.
    """
    return _host().cross_attention(q, k, v, mask, scale)


def gated_scan(x: Tensor, gate: Tensor, mask: Optional[Tensor] = None,
               state: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
    """A gated recurrence along the tokens: h = a h + (1 - a) x with a = sigmoid(gate).

    x and gate are (B, L, D) of one dtype, in any strides with a dense last dimension.
    Returns every state, (B, L, D) in x's dtype, and the last one, (B, D) in float32.
    state, (B, D) in float32, is the one before the first token (zeros without it): the
    last state of a call is the next call's, down to one token at a time.  mask is
    (B, L), True where a token takes part: the others leave the state as it is, and
    their x and gate are not used, whatever they hold.
    """
    return _host().gated_scan(x, gate, mask, state)


def residual_norm(x: Tensor, residual: Tensor, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None, *,
                  gate: Optional[Tensor] = None, scale: Optional[Tensor] = None, post_weight: Optional[Tensor] = None,
                  center: bool = True, eps: float = 1e-5) -> Tuple[Tensor, Tensor]:
    """The residual sum after a block and the norm before the next one, in one pass.

    x is the block's output and residual what ran past it, of one shape and dtype.
    Returns (y, sum) with sum = residual + scale * sigmoid(gate) * n and
    y = norm(sum) * weight + bias.  n is x, or norm(x) * post_weight where the block
    ends with a norm of its own; gate has x's shape and scale, like weight, bias and
    post_weight, is (dim,); what is left out is not there.  norm is over the last
    dimension (1 to 16,384 values): with ``center`` as in ``layer_norm``, without it by
    the root of the mean square alone.  The four vectors are of one dtype, which may be
    float32 beside bfloat16 tokens.
    """
    return _host().residual_norm(x, residual, weight, bias, gate, scale, post_weight, center, eps)


def clip_grad_norm_(grads: Union[Tensor, Iterable[Tensor]], max_norm: float,
                    out: Optional[Sequence[Tensor]] = None) -> Tensor:
    """Scales gradients by min(1, max_norm / (norm + 1e-6)) and returns ``norm``, the
    2-norm over all of them together, as a float32 scalar on the device.

    grads are contiguous tensors, or parameters and other leaves that require a
    gradient, whose ``.grad`` is taken (those without one are left out).  With ``out``, one tensor per gradient in either dtype,
    the clipped gradients are written there and the gradients stay as they are.  What is
    written may share no memory with another gradient or output, so that a parameter
    that two modules share is given once.
    """
    if isinstance(grads, Tensor):
        grads = [grads]
    # a Parameter's isinstance check runs Python code: plain tensors skip it
    grads = [g if type(g) is Tensor or not isinstance(g, torch.nn.Parameter) else g.grad for g in grads]
    if out is None:
        grads = [g for g in grads if g is not None]
        if not grads:
            raise ValueError("clip_grad_norm_: no gradients")
    elif any(g is None for g in grads):
        raise ValueError("clip_grad_norm_: out needs a gradient for each of its tensors")
    return _host().clip_grad_norm(grads, max_norm, [] if out is None else list(out))
