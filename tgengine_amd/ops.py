"""Operators of a temporal attention model on prepared batches, as HIP kernels.

What a model does with the neighbours that ``DataPipeline.prepare`` gathers:

* ``embed``: rows of a learned node table for ``NeighborData.neighbor_ids``,
  scaled; the gradient is summed by sorted ids.
* ``layer_norm``: over the tokens' channels, with the gradients of tokens,
  weight and bias.
* ``cross_attention``: query tokens to the states of another sequence under
  ``NeighborData.mask``, from one query per node to long sequences on both sides.
* ``gated_scan``: a gated recurrence along the same tokens under the same mask, from a
  node's state and to it, from one new token to long histories.
* ``residual_norm``: the residual sum after a block, with the block's own norm, gate and
  scale, and the norm before the next one.
* ``clip_grad_norm_``: the global norm of all gradients, and clipping by it.
* ``adamw_`` and ``AdamW``: a step over all parameters, averages in 32 bits or 8.

Tensors are float32 or bfloat16 on the GPU; sums and statistics are held in 32
bits.  Every call launches on the caller's current stream and does not wait for
the device; the same inputs give the same bits.  The first five take part in
autograd (once: their backward passes leave no graph; forward-mode derivatives and
tracing are refused).  There is no CPU path.
"""
from __future__ import annotations

import copy
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


def adamw_(params: Sequence[Tensor], grads: Sequence[Tensor], exp_avg: Sequence[Tensor], exp_avg_sq: Sequence[Tensor],
           steps: Sequence[Tensor], *, lr: Union[float, Tensor] = 1e-3, betas: Tuple[float, float] = (0.9, 0.999),
           eps: float = 1e-8, weight_decay: float = 1e-2, scales: Optional[Sequence[Optional[Tensor]]] = None,
           grad_norm: Optional[Tensor] = None, max_norm: Optional[float] = None) -> None:
    """One AdamW step over all tensors together, in place.

    Every list has one contiguous tensor per parameter; ``AdamW`` keeps them.  exp_avg and
    exp_avg_sq are both float32 and hold the averages of the gradients and of their
    squares, or both float8_e4m3fn and hold the first and the square root of the second
    in units of ``scales``: float32 (2, blocks), a power of two for every 256 values.
    All of them are zeros before the first step.  steps are int64 of one value and
    counted on the device, so that a step captured in a graph counts at every replay; lr
    may be a float32 tensor on the device for the same reason.

    With ``grad_norm``, the float32 scalar that ``clip_grad_norm_`` returns, the gradients
    are scaled by min(1, max_norm / (grad_norm + 1e-6)) as they are read:
    ``clip_grad_norm_(grads, float("inf"))`` takes the norm and writes nothing else if it
    is finite (otherwise the gradients become NaN, as inf / inf is).
    """
    if (grad_norm is None) != (max_norm is None):
        raise ValueError("adamw_: grad_norm and max_norm come together")
    rate = lr if isinstance(lr, Tensor) and lr.is_cuda else None
    _host().adamw(list(params), list(grads), list(exp_avg), list(exp_avg_sq), list(steps),
                  [] if scales is None else list(scales), 0.0 if rate is not None else float(lr), rate, betas[0], betas[1],
                  eps, weight_decay, grad_norm, 0.0 if max_norm is None else max_norm)


def _kept(state, device: torch.device):
    """A copy of an optimizer's state for one parameter, its tensors on ``device`` in their own types."""
    if isinstance(state, Tensor):
        return state.to(device, copy=True)
    if isinstance(state, dict):
        return {k: _kept(v, device) for k, v in state.items()}
    if type(state) in (list, tuple):
        return type(state)(_kept(v, device) for v in state)
    return copy.deepcopy(state)


class AdamW(torch.optim.Optimizer):
    """AdamW over all parameters of a group in one step of kernels (``adamw_``).

    ``bits=8`` keeps both averages in 8 bits a value (and a scale for every 256), for
    tensors of 4,096 values or more; smaller ones stay in 32 bits, which cost nothing.
    ``step`` takes the norm of ``clip_grad_norm_`` and a max_norm, to clip without writing
    the gradients.  A step can be captured in a graph once every parameter has taken one
    outside.  Parameters without a gradient are left out of a step.
    """

    def __init__(self, params, lr: Union[float, Tensor] = 1e-3, betas: Tuple[float, float] = (0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float = 1e-2, bits: int = 32):
        if not (float(lr) >= 0.0 and eps >= 0.0 and weight_decay >= 0.0 and all(0.0 <= b < 1.0 for b in betas)):
            raise ValueError(f"AdamW: lr={float(lr)} betas={betas} eps={eps} weight_decay={weight_decay}")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, bits=bits))

    def add_param_group(self, param_group: dict) -> None:
        if param_group.get("bits", self.defaults["bits"]) not in (8, 32):
            raise ValueError("AdamW: bits must be 8 or 32")
        super().add_param_group(param_group)

    def _new(self, p: Tensor, bits: int) -> dict:
        if p.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW: a parameter's first step cannot be captured: its averages would start again at every replay")
        held = bits == 8 and p.numel() >= 4096
        kind = dict(dtype=torch.float8_e4m3fn if held else torch.float32, device=p.device)
        out = {"step": torch.zeros((), dtype=torch.int64, device=p.device),
               "exp_avg": torch.zeros(p.shape, **kind), "exp_avg_sq": torch.zeros(p.shape, **kind)}
        if held:
            out["scales"] = torch.zeros(2, -(-p.numel() // 256), device=p.device)
        return out

    @torch.no_grad()
    def step(self, closure=None, *, grad_norm: Optional[Tensor] = None, max_norm: Optional[float] = None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            params = [p for p in group["params"] if p.grad is not None]
            if not params:
                continue
            for p in params:
                if p.grad.layout is not torch.strided:
                    raise RuntimeError("AdamW: sparse gradients are not supported")
                if not self.state[p]:
                    self.state[p].update(self._new(p, group["bits"]))
            states = [self.state[p] for p in params]
            adamw_(params, [p.grad if p.grad.is_contiguous() else p.grad.contiguous() for p in params],
                   [s["exp_avg"] for s in states], [s["exp_avg_sq"] for s in states], [s["step"] for s in states],
                   lr=group["lr"], betas=group["betas"], eps=group["eps"], weight_decay=group["weight_decay"],
                   scales=[s.get("scales") for s in states], grad_norm=grad_norm, max_norm=max_norm)
        return loss

    def load_state_dict(self, state_dict) -> None:
        given = {}

        def own_types(_) -> None:
            # the base class casts state to its parameter's type; the averages, scales and steps keep theirs
            ids = [i for g in given["param_groups"] for i in g["params"]]
            params = [p for g in self.param_groups for p in g["params"]]
            for i, p in zip(ids, params):
                if i in given["state"]:
                    self.state[p] = _kept(given["state"][i], p.device)

        # behind the caller's hooks that change what is loaded, before those that see it loaded
        hooks = [self.register_load_state_dict_pre_hook(lambda _, state: given.update(state)),
                 self.register_load_state_dict_post_hook(own_types, prepend=True)]
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()
