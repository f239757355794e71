"""Operators with gradients: what turns sampled tokens into updates of a model of this family.

    RWKV7_TRAIN_OP   the WKV-7 recurrence of `RWKV7_BATCH_OP` over whole sequences, out of place and differentiable
    layer_norm       a block's norms, also in groups of a head (the norm behind the recurrence), differentiable
    token_logp       log-probabilities of given ids under logits, differentiable: what the policy, the sampler or a reference
                     model gave the tokens
    policy_loss      clipped ratios against the policy that sampled, with a penalty for leaving a reference; differentiable
    policy_loss_grad the same, loss and gradient by the logits in one pass over them
    preference_loss  pairs of a better and a worse answer; differentiable

They run on the current stream of their tensors' device and take strided inputs (the last dimension dense; others are
copied). Gradients are those of the formulas in include/albatross_b200.h; they cannot be differentiated again. The reference
only generates: none of these has a counterpart there.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib

HEAD_SIZE = 64
_DT = {torch.float16: _lib.DT_F16, torch.bfloat16: _lib.DT_BF16, torch.float32: _lib.DT_F32}


def _run(name: str, device: torch.device, *args) -> None:
    """Calls the C entry on the current stream of `device`."""
    fn, stream = getattr(_lib.lib, name), torch.cuda.current_stream(device).cuda_stream
    if device.index == torch.cuda.current_device():
        status = fn(*args, stream)
    else:
        with torch.cuda.device(device):
            status = fn(*args, stream)
    if status:
        _lib.check(status, name)


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _dense_last(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def _steps(t: torch.Tensor) -> torch.Tensor:
    """[B, T, C] with a dense last dimension and every step on a 16-byte boundary."""
    if t.stride(2) == 1 and not (t.stride(0) | t.stride(1)) & 7 and not t.data_ptr() & 15:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _needs_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# --------------------------------------------------------------------------------------------
# The recurrence
# --------------------------------------------------------------------------------------------
def _wkv_seq(B, T, H, xs, state, lengths, checkpoints) -> _lib.Wkv7Seq:
    s = _lib.Wkv7Seq(_DT[xs[0].dtype], B, T, H)
    for i, x in enumerate(xs):
        s.x[i], s.batch_stride[i], s.step_stride[i] = x.data_ptr(), x.stride(0), x.stride(1)
    s.state, s.lengths, s.checkpoints = _ptr(state), _ptr(lengths), _ptr(checkpoints)
    return s


def _wkv_forward(state, xs, lengths, keep: bool):
    B, T, C_ = xs[0].shape
    H, device = C_ // HEAD_SIZE, xs[0].device
    checkpoints = torch.empty((B, H, -(-T // _lib.WKV_CHUNK), HEAD_SIZE, HEAD_SIZE), dtype=torch.float32, device=device) if keep else None
    y = torch.empty((B, T, C_), dtype=xs[0].dtype, device=device)
    out = torch.empty((B, H, HEAD_SIZE, HEAD_SIZE), dtype=torch.float32, device=device)
    s = _wkv_seq(B, T, H, xs, state, lengths, checkpoints)
    _run("ab_wkv7_seq_fwd", device, C.byref(s), y.data_ptr(), out.data_ptr())
    return y, out, checkpoints


class _Wkv7(torch.autograd.Function):
    @staticmethod
    def forward(ctx, state, lengths, *xs):
        y, out, checkpoints = _wkv_forward(state, xs, lengths, True)
        ctx.save_for_backward(state, lengths, checkpoints, *xs)
        ctx.set_materialize_grads(False)
        return y, out

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dout):
        state, lengths, checkpoints, *xs = ctx.saved_tensors
        B, T, C_ = xs[0].shape
        device = xs[0].device
        dy = None if dy is None else _steps(dy)
        dout = None if dout is None else dout.contiguous()
        need = ctx.needs_input_grad
        dxs = [torch.empty((B, T, C_), dtype=xs[0].dtype, device=device) if n else None for n in need[2:]]
        dstate = torch.empty((B, C_ // HEAD_SIZE, HEAD_SIZE, HEAD_SIZE), dtype=torch.float32, device=device) if need[0] else None
        s = _wkv_seq(B, T, C_ // HEAD_SIZE, xs, state, lengths, checkpoints)
        _run("ab_wkv7_seq_bwd", device, C.byref(s), _ptr(dy), 0 if dy is None else dy.stride(0), 0 if dy is None else dy.stride(1), _ptr(dout),
             (C.c_void_p * 6)(*(_ptr(d) for d in dxs)), _ptr(dstate))
        return (dstate, None, *dxs)


def RWKV7_TRAIN_OP(state: Optional[torch.Tensor], r, w, k, v, a, b, lengths: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """WKV-7 over r, w, k, v, a, b [B, T, C] (all fp16 or all bf16; `w` before exp(-exp(w))), starting from `state` [B, H, 64, 64] fp32
    (None: zeros), which is left as it is. Returns y [B, T, C] and the state after the last step. `lengths`, int32 [B] on the device:
    sequence b ends after lengths[b] steps; what the inputs hold behind its end is not used, y and all gradients are zero there.
    Training keeps 16 KB per head and 16 steps between the passes. A NaN or an infinity in a step's inputs may show in the outputs of up to
    15 steps before it."""
    xs = (r, w, k, v, a, b)
    assert r.dim() == 3 and r.is_cuda and r.dtype in (torch.float16, torch.bfloat16)
    B, T, C_ = r.shape
    H = C_ // HEAD_SIZE
    assert B > 0 and H > 0 and C_ == H * HEAD_SIZE
    assert all(x.shape == r.shape and x.dtype == r.dtype and x.device == r.device for x in xs)
    if state is not None:
        assert state.shape == (B, H, HEAD_SIZE, HEAD_SIZE) and state.dtype == torch.float32 and state.device == r.device
        state = state.contiguous()
    if lengths is not None:
        assert lengths.shape == (B,) and lengths.dtype == torch.int32 and lengths.device == r.device
        lengths = lengths.contiguous()
    xs = tuple(_steps(x) for x in xs)
    if _needs_grad(state, *xs):
        return _Wkv7.apply(state, lengths, *xs)
    return _wkv_forward(state, xs, lengths, False)[:2]


# --------------------------------------------------------------------------------------------
# The norms
# --------------------------------------------------------------------------------------------
def _as_rows(x: torch.Tensor) -> torch.Tensor:
    """[..., C] as rows [n, C] with a dense last dimension; a view where the strides allow one."""
    return _dense_last(x.reshape(-1, x.shape[-1]))


def _wtype(x, weight, bias):
    return _DT[(weight if weight is not None else bias if bias is not None else x).dtype]


def _norm_forward(x, weight, bias, eps, groups, keep):
    rows = _as_rows(x)
    n, C_ = rows.shape
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    stats = torch.empty((2, n, groups), dtype=torch.float32, device=x.device) if keep else None
    at = stats.data_ptr() if keep else None
    _run("ab_layer_norm_fwd", x.device, _DT[x.dtype], _wtype(x, weight, bias), n, C_, groups, rows.data_ptr(), rows.stride(0), _ptr(weight), _ptr(bias),
         eps, y.data_ptr(), at, at + 4 * n * groups if keep else None)
    return y, stats


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, groups):
        y, stats = _norm_forward(x, weight, bias, eps, groups, True)
        ctx.save_for_backward(x, weight, bias, stats)
        ctx.groups = groups
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, bias, stats = ctx.saved_tensors
        rows, drows = _as_rows(x), _as_rows(dy)
        n, C_ = rows.shape
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if ctx.needs_input_grad[0] else None
        dw = torch.empty_like(weight) if ctx.needs_input_grad[1] else None
        db = torch.empty_like(bias) if ctx.needs_input_grad[2] else None
        scratch = torch.empty(_lib.lib.ab_layer_norm_scratch_bytes(n, C_), dtype=torch.uint8, device=x.device) if dw is not None or db is not None else None
        _run("ab_layer_norm_bwd", x.device, _DT[x.dtype], _wtype(x, weight, bias), n, C_, ctx.groups, rows.data_ptr(), rows.stride(0), _ptr(weight),
             stats.data_ptr(), stats.data_ptr() + 4 * n * ctx.groups, drows.data_ptr(), drows.stride(0), _ptr(dx), _ptr(dw), _ptr(db), _ptr(scratch))
        return dx, dw, db, None, None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, eps: float = 1e-5,
               groups: int = 1) -> torch.Tensor:
    """Layer norm over the last dimension of x (fp16, bf16 or fp32), or over each of its `groups` equal parts: `groups=H, eps=64e-5` is the norm
    of the heads behind the recurrence (ln_x). `weight`, `bias` [C]: of x's type or fp32."""
    assert x.is_cuda and x.dtype in _DT and x.dim() >= 1
    C_ = x.shape[-1]
    assert C_ > 0 and groups > 0 and C_ % groups == 0
    if weight is not None and bias is not None:
        assert weight.dtype == bias.dtype
    for p in (weight, bias):
        assert p is None or (p.shape == (C_,) and p.dtype in (x.dtype, torch.float32) and p.device == x.device)
    weight, bias = (None if p is None else p.contiguous() for p in (weight, bias))
    if _needs_grad(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, float(eps), groups)
    return _norm_forward(x, weight, bias, float(eps), groups, False)[0]


# --------------------------------------------------------------------------------------------
# Losses on logits
# --------------------------------------------------------------------------------------------
def _check_rows(logits, ids, mask):
    assert logits.is_cuda and logits.dtype in _DT and logits.dim() >= 1 and logits.shape[-1] > 0
    assert ids.shape == logits.shape[:-1] and ids.dtype in (torch.int64, torch.int32) and ids.device == logits.device
    assert mask is None or (mask.shape == ids.shape and mask.dtype == torch.bool and mask.device == logits.device)
    return ids.long().contiguous(), None if mask is None else mask.contiguous()


def _rows_of(rows, ids, mask) -> _lib.LogitRows:
    return _lib.LogitRows(_DT[rows.dtype], rows.shape[1], rows.shape[0], rows.stride(0), rows.data_ptr(), ids.data_ptr(), _ptr(mask))


def _dlogits(logits, ids, mask, stats, g, rows_per_g, scale):
    out = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    t = _rows_of(_as_rows(logits), ids, mask)
    _run("ab_token_logp_bwd", logits.device, C.byref(t), stats.data_ptr(), g.data_ptr(), rows_per_g, _ptr(scale), out.data_ptr())
    return out


def _f32(n, like, *more):
    return torch.empty((n, *more), dtype=torch.float32, device=like.device)


def _logp_forward(logits, ids, mask, keep):
    rows = _as_rows(logits)
    logp = torch.empty(ids.shape, dtype=torch.float32, device=logits.device)
    stats = _f32(rows.shape[0], logits, 2) if keep else None
    t = _rows_of(rows, ids, mask)
    _run("ab_token_logp_fwd", logits.device, C.byref(t), None, logp.data_ptr(), _ptr(stats))
    return logp, stats


class _TokenLogp(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, mask):
        logp, stats = _logp_forward(logits, ids, mask, True)
        ctx.save_for_backward(logits, ids, mask, stats)
        return logp

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        logits, ids, mask, stats = ctx.saved_tensors
        return _dlogits(logits, ids, mask, stats, g.contiguous(), 1, None), None, None


def token_logp(logits: torch.Tensor, ids: torch.Tensor, mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """log softmax(logits)[..., ids] in fp32, for logits [..., V] (fp16, bf16 or fp32) and ids [...] (the token that position predicts). Where `mask`
    (bool) is False the result and the gradient are 0, whatever logits and ids hold there."""
    ids, mask = _check_rows(logits, ids, mask)
    if _needs_grad(logits):
        return _TokenLogp.apply(logits, ids, mask)
    return _logp_forward(logits, ids, mask, False)[0]


def _policy_args(logits, ids, old_logp, advantages, mask, ref_logp, clip, kl, denom):
    ids, mask = _check_rows(logits, ids, mask)

    def rows(t):
        assert t is None or t.device == logits.device
        return None if t is None else t.detach().to(torch.float32).broadcast_to(ids.shape).contiguous()
    old_logp, advantages, ref_logp = rows(old_logp), rows(advantages), rows(ref_logp)
    low, high = clip
    assert 0.0 <= low <= 1.0 and high >= 0.0 and (denom is None or denom > 0.0)
    return ids, mask, (old_logp, advantages, ref_logp), (float(low), float(high), float(kl), float(denom or 0.0))


def _policy_struct(tensors, numbers) -> _lib.Policy:
    return _lib.Policy(*(_ptr(t) for t in tensors), *numbers)


def _policy_forward(logits, ids, mask, tensors, numbers, keep):
    rows = _as_rows(logits)
    n = rows.shape[0]
    logp = torch.empty(ids.shape, dtype=torch.float32, device=logits.device)
    loss = torch.empty((), dtype=torch.float32, device=logits.device)
    stats, g = (_f32(n, logits, 2), _f32(n, logits)) if keep else (None, None)
    scratch = torch.empty(2 * n + 2, dtype=torch.float64, device=logits.device)
    t, p = _rows_of(rows, ids, mask), _policy_struct(tensors, numbers)
    _run("ab_policy_loss_fwd", logits.device, C.byref(t), C.byref(p), loss.data_ptr(), logp.data_ptr(), _ptr(stats), _ptr(g), scratch.data_ptr())
    return loss, logp, stats, g


class _PolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, mask, tensors, numbers):
        loss, logp, stats, g = _policy_forward(logits, ids, mask, tensors, numbers, True)
        ctx.save_for_backward(logits, ids, mask, stats, g)
        ctx.mark_non_differentiable(logp)
        return loss, logp

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss, _):
        logits, ids, mask, stats, g = ctx.saved_tensors
        return _dlogits(logits, ids, mask, stats, g, 1, dloss.contiguous()), None, None, None, None


def policy_loss(logits: torch.Tensor, ids: torch.Tensor, old_logp: Optional[torch.Tensor], advantages: torch.Tensor,
                mask: Optional[torch.Tensor] = None, ref_logp: Optional[torch.Tensor] = None, clip: Sequence[float] = (0.2, 0.2), kl: float = 0.0,
                denom: Optional[float] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The clipped policy loss of sampled tokens, and their log-probabilities (without gradient; 0 where masked).

    Per token, with ratio = exp(logp - old_logp): -min(ratio A, clamp(ratio, 1 - clip[0], 1 + clip[1]) A) + kl (exp(ref_logp - logp) - (ref_logp - logp) - 1);
    their sum where `mask` (bool [...]) is True, divided by `denom` or else by the number of such tokens (at least 1). logits [..., V], ids [...];
    old_logp, advantages and ref_logp broadcast to the ids' shape and get no gradient; old_logp None: the ratio is 1, as on the first step after
    sampling. At a border of the clip range the unclipped side's gradient counts."""
    ids, mask, tensors, numbers = _policy_args(logits, ids, old_logp, advantages, mask, ref_logp, clip, kl, denom)
    if _needs_grad(logits):
        return _PolicyLoss.apply(logits, ids, mask, tensors, numbers)
    return _policy_forward(logits, ids, mask, tensors, numbers, False)[:2]


def policy_loss_grad(logits: torch.Tensor, ids: torch.Tensor, old_logp: Optional[torch.Tensor], advantages: torch.Tensor,
                     mask: Optional[torch.Tensor] = None, ref_logp: Optional[torch.Tensor] = None, clip: Sequence[float] = (0.2, 0.2), kl: float = 0.0,
                     denom: Optional[float] = None, scale: float = 1.0, out: Optional[torch.Tensor] = None):
    """`policy_loss` and `scale` times its gradient by the logits, which are read once: (loss, logp, dlogits). `out`: where the gradient goes, dense
    and like the logits; it may be the logits themselves. (For `logits.backward(dlogits)`; no autograd graph is made here.)"""
    ids, mask, tensors, numbers = _policy_args(logits, ids, old_logp, advantages, mask, ref_logp, clip, kl, denom)
    logits = logits.detach()
    rows = _as_rows(logits)
    n = rows.shape[0]
    if out is None:
        out = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    assert out.shape == logits.shape and out.dtype == logits.dtype and out.device == logits.device and out.is_contiguous()
    logp = torch.empty(ids.shape, dtype=torch.float32, device=logits.device)
    loss = torch.empty((), dtype=torch.float32, device=logits.device)
    scratch = torch.empty(2 * n + 2, dtype=torch.float64, device=logits.device)
    t, p = _rows_of(rows, ids, mask), _policy_struct(tensors, numbers)
    _run("ab_policy_loss_grad", logits.device, C.byref(t), C.byref(p), float(scale), loss.data_ptr(), logp.data_ptr(), out.data_ptr(), scratch.data_ptr())
    return loss, logp, out


def _preference_forward(logits, ids, mask, ref_logp, beta, smoothing, keep):
    n, T = ids.shape
    rows = _as_rows(logits)
    loss = torch.empty((), dtype=torch.float32, device=logits.device)
    logp = _f32(n, logits)
    stats, g = (_f32(n * T, logits, 2), _f32(n, logits)) if keep else (None, None)
    scratch = torch.empty(n * T, dtype=torch.float64, device=logits.device)
    t = _rows_of(rows, ids, mask)
    _run("ab_preference_loss_fwd", logits.device, C.byref(t), n // 2, T, ref_logp.data_ptr(), beta, smoothing, loss.data_ptr(), logp.data_ptr(), _ptr(stats),
         _ptr(g), scratch.data_ptr())
    return loss, logp, stats, g


class _PreferenceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, mask, ref_logp, beta, smoothing):
        loss, logp, stats, g = _preference_forward(logits, ids, mask, ref_logp, beta, smoothing, True)
        ctx.save_for_backward(logits, ids, mask, stats, g)
        ctx.mark_non_differentiable(logp)
        return loss, logp

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss, _):
        logits, ids, mask, stats, g = ctx.saved_tensors
        return _dlogits(logits, ids, mask, stats, g, max(1, ids.shape[1]), dloss.contiguous()), None, None, None, None, None


def preference_loss(logits: torch.Tensor, ids: torch.Tensor, ref_logp: torch.Tensor, mask: Optional[torch.Tensor] = None, beta: float = 0.1,
                    label_smoothing: float = 0.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """The preference loss of P pairs of answers: logits [2P, T, V], ids [2P, T], the better answers first, then the worse ones in the same order.
    With s the sums of an answer's log-probabilities where `mask` (bool [2P, T]) is True and m = beta ((s_better - ref_better) - (s_worse - ref_worse)):
    the mean of -(1 - label_smoothing) log sigmoid(m) - label_smoothing log sigmoid(-m). `ref_logp` [2P]: the sums under the reference model (no
    gradient). Returns the loss and the sums s (without gradient)."""
    assert logits.dim() == 3 and logits.shape[0] % 2 == 0 and logits.shape[0] > 0
    ids, mask = _check_rows(logits, ids, mask)
    assert ref_logp.shape == (logits.shape[0],) and ref_logp.device == logits.device and 0.0 <= label_smoothing <= 1.0
    ref_logp = ref_logp.detach().to(torch.float32).contiguous()
    if _needs_grad(logits):
        return _PreferenceLoss.apply(logits, ids, mask, ref_logp, float(beta), float(label_smoothing))
    return _preference_forward(logits, ids, mask, ref_logp, float(beta), float(label_smoothing), False)[:2]
