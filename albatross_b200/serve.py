"""Operators that serve a token: the draw of an id under filters, and products with 4-bit weights in groups.

    sampler_batch    one id per row of logits under a temperature, top-k, top-p and min-p, from given uniform numbers, with its log-probability
    linear_int4      a few rows of activations by 4-bit codes with a scale, and perhaps a zero point, for each group of inputs
    quantize_int4    a matrix in that form

They run on the current stream of their tensors' device, need no memory of their own between calls and can be captured into CUDA graphs. Arguments are
checked in csrc/serve_op.cpp (`torch.ops.albatross_b200`), which calls the C entries of the kernel library; what does not fit raises RuntimeError. Neither
has a counterpart in the reference.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple, Union

import torch

from . import _shim
from . import build as _build

_sample, _linear_int4 = _shim.load(_build.SERVE_OP_LIB, "albatross_b200_serve_bind", ("sample", "linear_int4"))

Number = Union[float, torch.Tensor]


def sampler_batch(logits: torch.Tensor, uniform: torch.Tensor, temperature: Number = 1.0, top_k: Union[int, torch.Tensor] = 0, top_p: Number = 1.0,
                  min_p: Number = 0.0, out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Draws one id per row of logits [..., V] (fp16, bf16 or fp32; V up to 2^18) by `uniform`, fp32 numbers in [0, 1), one per row: ids [..., 1] (int64)
    and their log-probabilities [..., 1] (fp32) under the distribution they were drawn from, which is what policy_loss wants for old_logp.

    With w = exp((logit - largest) / temperature) and the values in order, larger ones first, equals by id, the front part is kept in which
    each value but the first has a rank below top_k, a sum of w in front of it below top_p * (the sum over the first top_k), and w >= min_p.
    The id is the first one whose sum of w up to and with it exceeds uniform * (the sum that is kept). It is the one that 64 bits give, unless
    uniform or top_p meets a border within some 1e-9 of the sum. temperature 0 or top_k 1: the first largest value. top_k <= 0, top_p >= 1 and
    min_p <= 0 filter nothing. Each of the four is a number, or a tensor of one per row on the device of logits, read as fp32 (top_k: int32),
    in which a NaN filters nothing; as a temperature it is 0. -inf is never drawn; a row with a NaN, or of -inf alone, gives -1 and NaN.

    There are no gradients: the log-probabilities carry none, whatever the logits require (they are an old_logp; token_logp of the ids has one).

    `out`: a dense int64 tensor of one id per row to write into, on the device, apart from the inputs, or in pinned host memory (read it
    after synchronising the stream)."""
    T, k, p, m = temperature, top_k, top_p, min_p
    t = torch.is_tensor
    return _sample(logits, uniform, T if t(T) else None, k if t(k) else None, p if t(p) else None, m if t(m) else None, 1.0 if t(T) else T, 0 if t(k) else k,
                   1.0 if t(p) else p, 0.0 if t(m) else m, out)


class Int4Matrix(NamedTuple):
    """A matrix [N, K] as `linear_int4` takes it: linear_int4(x, *matrix)."""
    w: torch.Tensor                 # uint8 [N, K / 2]: codes 0 .. 15, even inputs in the low nibble
    scale: torch.Tensor             # fp16 or bf16 [N, K / group]
    zero: Optional[torch.Tensor]    # uint8 [N, K / group], or None: 8 everywhere

    def dequantize(self) -> torch.Tensor:
        """fp32 [N, K]"""
        N, groups = self.scale.shape
        q = torch.stack([self.w & 15, self.w >> 4], -1).view(N, groups, -1).float()
        return ((q - (8.0 if self.zero is None else self.zero.float()[..., None])) * self.scale.float()[..., None]).view(N, -1)


@torch.no_grad()
def quantize_int4(w: torch.Tensor, group: int = 128, zeros: bool = False, dtype: torch.dtype = torch.float16) -> Int4Matrix:
    """w [N, K] (any float type), in groups of 32, 64 or a multiple of 128 inputs: s = max |w| / 7 and q = rint(w / s) + 8, or with `zeros`
    s = (max - min) / 15 over the group's values and 0, z = rint(-min / s), q = rint(w / s) + z. `dtype`: of the scales, and so of the activations.
    w may be a parameter: the result has no part in its gradients."""
    N, K = w.shape
    if K % group or not (group in (32, 64) or group % 128 == 0):
        raise ValueError(f"groups of {group} inputs (32, 64 or a multiple of 128, which divides {K})")
    g = w.float().view(N, K // group, group)
    if zeros:
        low, high = g.amin(-1).clamp(max=0.0), g.amax(-1).clamp(min=0.0)
        scale = ((high - low) / 15.0).to(dtype)
    else:
        scale = (g.abs().amax(-1) / 7.0).to(dtype)
    s = torch.where(scale > 0, scale, torch.ones_like(scale)).float()
    zero = torch.round(-low / s).clamp_(0, 15) if zeros else torch.full_like(s, 8.0)
    q = (torch.round(g / s[..., None]) + zero[..., None]).clamp_(0, 15).to(torch.uint8).view(N, K)
    return Int4Matrix((q[:, 0::2] | (q[:, 1::2] << 4)).contiguous(), scale, zero.to(torch.uint8) if zeros else None)


def linear_int4(x: torch.Tensor, w: torch.Tensor, scale: torch.Tensor, zero: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x [..., K] (fp16 or bf16) by a matrix of 4-bit codes: y[..., n] = sum_k x[..., k] (q[n, k] - zero[n, k / group]) scale[n, k / group], in the type of x.

    w: uint8 [N, K / 2], even k in the low nibble; scale [N, K / group] of the type of x; zero: uint8 [N, K / group], codes 0 .. 15, or None:
    8. group is 32, 64 or a multiple of 128. Codes times activations are exact, sums and scales 32-bit; y is rounded once. For few rows, whose
    time is that of reading the codes: they are taken in once for up to 8 rows, and for up to 16 where groups are not of 32 and the matrix is
    small; again for more, up to 65535. (16384 x 4096 in groups of 64, and torch's product with the dequantised fp16 matrix: 8 rows 22 and 28
    us, 16 rows 54 and 28, 64 rows 185 and 28, 320 rows 990 and 41.) No gradients."""
    return _linear_int4(x, w, scale, zero)
