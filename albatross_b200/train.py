"""Operators with gradients: what turns sampled tokens into updates of a model of this family.

    RWKV7_TRAIN_OP   the WKV-7 recurrence of `RWKV7_BATCH_OP` over whole sequences, out of place and differentiable
    layer_norm       a block's norms, also in groups of a head (the norm behind the recurrence), differentiable
    token_logp       log-probabilities of given ids under logits, differentiable: what the policy or a reference model gave the tokens
    policy_loss      clipped ratios against the policy that sampled, with a penalty for leaving a reference; differentiable
    policy_loss_grad the same, loss and gradient by the logits in one pass over them
    preference_loss  pairs of a better and a worse answer; differentiable

They run on the current stream of their tensors' device and take strided inputs: the last dimension dense and, but for the recurrence,
one stride between rows (logits[:, :-1] of several sequences has two). Others are copied, once for both passes. Gradients are those of
the formulas in include/albatross_b200.h; they cannot be differentiated again, and there are no forward-mode derivatives: a tensor with a
tangent is refused. Neither can they be traced (torch.compile, torch.export, make_fx: call them from a function under
torch.compiler.disable) or transformed by torch.func.grad; torch.vmap calls them slice by slice. The reference only generates: none of
these has a counterpart there.

Arguments are checked, memory is taken and gradients are tied to autograd in csrc/train_op.cpp (`torch.ops.albatross_b200`), which
calls the C entries of the kernel library; what does not fit raises RuntimeError.
"""
from __future__ import annotations

import ctypes as C
import os
from typing import Optional, Sequence, Tuple

import torch

from . import _lib
from . import build as _build


def _load():
    if not os.path.exists(_build.TRAIN_OP_LIB):
        raise ImportError(f"{_build.TRAIN_OP_LIB} is missing: build it with `python -m albatross_b200.build`")
    torch.ops.load_library(_build.TRAIN_OP_LIB)
    missing = C.c_char_p()
    bind = C.CDLL(_build.TRAIN_OP_LIB).albatross_b200_train_bind
    bind.argtypes = [C.c_char_p, C.POINTER(C.c_char_p)]
    if bind(_lib.LIB_PATH.encode(), C.byref(missing)):
        raise ImportError(f"{_lib.LIB_PATH} does not have {missing.value.decode()}: build both again with `python -m albatross_b200.build`")
    ops = torch.ops.albatross_b200
    return {n: getattr(ops, n).default for n in ("wkv7", "layer_norm", "token_logp", "policy_loss", "policy_loss_grad", "preference_loss")}


_ops = _load()
_wkv7, _layer_norm, _token_logp, _policy_loss, _policy_loss_grad, _preference_loss = _ops.values()


def RWKV7_TRAIN_OP(state: Optional[torch.Tensor], r, w, k, v, a, b, lengths: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """WKV-7 over r, w, k, v, a, b [B, T, C] (all fp16 or all bf16; `w` before exp(-exp(w))), starting from `state` [B, H, 64, 64] fp32
    (None: zeros), which is left as it is. Returns y [B, T, C] and the state after the last step. `lengths`, int32 [B] on the device:
    sequence b ends after lengths[b] steps; what the inputs hold behind its end is not used, y and all gradients are zero there.
    Training keeps 16 KB per head and 16 steps between the passes. A NaN or an infinity in a step's inputs may show in the outputs of up to
    15 steps before it.

    Decays: as long as none of a chunk of 16 steps' channels shrinks below 2^-16 over it (0.5 a step; a model's own, exp(-exp(w)) with w below
    -0.5, stays above 0.545) a chunk is taken at once. Beyond that it is taken in pieces, down to single steps: up to 60 times as long forward and
    250 times backward for decays below 2^-16 in a step.
    Precision: states and sums are 32-bit; gradients that end in 16 bits are summed over a state's rows with 16-bit factors, and in bf16 what v and
    the gradient of y hold below 2^-27 of a chunk's largest value loses bits."""
    return _wkv7(state, r, w, k, v, a, b, lengths)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, eps: float = 1e-5,
               groups: int = 1) -> torch.Tensor:
    """Layer norm over the last dimension of x (fp16, bf16 or fp32), or over each of its `groups` equal parts: `groups=H, eps=64e-5` is the norm
    of the heads behind the recurrence (ln_x). `weight`, `bias` [C]: of x's type or fp32."""
    return _layer_norm(x, weight, bias, eps, groups)


def token_logp(logits: torch.Tensor, ids: torch.Tensor, mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """log softmax(logits)[..., ids] in fp32, for logits [..., V] (fp16, bf16 or fp32) and ids [...] (the token that position predicts). Where `mask`
    (bool) is False the result and the gradient are 0, whatever logits and ids hold there."""
    return _token_logp(logits, ids, mask)


def _denom(denom: Optional[float]) -> float:
    if denom is not None and not denom > 0.0:
        raise RuntimeError("policy_loss: the denominator must be positive")
    return 0.0 if denom is None else denom


def policy_loss(logits: torch.Tensor, ids: torch.Tensor, old_logp: Optional[torch.Tensor], advantages: torch.Tensor,
                mask: Optional[torch.Tensor] = None, ref_logp: Optional[torch.Tensor] = None, clip: Sequence[float] = (0.2, 0.2), kl: float = 0.0,
                denom: Optional[float] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The clipped policy loss of sampled tokens, and their log-probabilities (without gradient; 0 where masked).

    Per token, with ratio = exp(logp - old_logp): -min(ratio A, clamp(ratio, 1 - clip[0], 1 + clip[1]) A) + kl (exp(ref_logp - logp) - (ref_logp - logp) - 1);
    their sum where `mask` (bool [...]) is True, divided by `denom` or else by the number of such tokens (at least 1). logits [..., V], ids [...];
    old_logp, advantages and ref_logp broadcast to the ids' shape and get no gradient; with kl 0 ref_logp does not count, and an advantage of 0
    makes nothing of any ratio. old_logp None: the ratio is 1, as on the first step after sampling. At a border of the clip range the unclipped
    side's gradient counts.

    old_logp are log-probabilities under the distribution that the tokens were drawn from. token_logp gives those of softmax(logits);
    `sampler_simple_batch` of this package draws from another one (the argmax of logits plus uniform noise), and ratios against token_logp of its
    logits carry the difference."""
    return _policy_loss(logits, ids, old_logp, advantages, mask, ref_logp, clip[0], clip[1], kl, _denom(denom))


def policy_loss_grad(logits: torch.Tensor, ids: torch.Tensor, old_logp: Optional[torch.Tensor], advantages: torch.Tensor,
                     mask: Optional[torch.Tensor] = None, ref_logp: Optional[torch.Tensor] = None, clip: Sequence[float] = (0.2, 0.2), kl: float = 0.0,
                     denom: Optional[float] = None, scale: float = 1.0, out: Optional[torch.Tensor] = None):
    """`policy_loss` and `scale` times its gradient by the logits, which are read once: (loss, logp, dlogits). `out`: where the gradient goes, dense
    and like the logits; it may be the logits themselves, but, where gradients are recorded, no leaf that requires one. (For `logits.backward(dlogits)`; no autograd graph is made here.)"""
    return _policy_loss_grad(logits, ids, old_logp, advantages, mask, ref_logp, clip[0], clip[1], kl, _denom(denom), scale, out)


def preference_loss(logits: torch.Tensor, ids: torch.Tensor, ref_logp: torch.Tensor, mask: Optional[torch.Tensor] = None, beta: float = 0.1,
                    label_smoothing: float = 0.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """The preference loss of P pairs of answers: logits [2P, T, V], ids [2P, T], the better answers first, then the worse ones in the same order.
    With s the sums of an answer's log-probabilities where `mask` (bool [2P, T]) is True and m = beta ((s_better - ref_better) - (s_worse - ref_worse)):
    the mean of -(1 - label_smoothing) log sigmoid(m) - label_smoothing log sigmoid(-m). `ref_logp` [2P]: the sums under the reference model (no
    gradient). Returns the loss and the sums s (without gradient)."""
    return _preference_loss(logits, ids, ref_logp, mask, beta, label_smoothing)
