"""GPU: clipping of gradients where outputs have another type on the same memory, and at the ends of the numbers' range."""
import pytest
import torch

import albatross_b200 as ab

pytestmark = pytest.mark.gpu


def normal(*shape, dtype, seed=0):
    return torch.randn(shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("dtype,to", [(torch.float16, torch.bfloat16), (torch.bfloat16, torch.float16)])
@pytest.mark.parametrize("limit", [1e6, 0.5])
def test_outputs_of_another_type_on_the_gradients_memory(dtype, to, limit):
    """Values are converted, whether the norm is above its limit or not; a tensor that keeps its type does not change that."""
    for shapes in ([(1000, 77)], [(5,), (4097,), (3, 64)]):
        grads = [normal(*s, dtype=dtype, seed=i) for i, s in enumerate(shapes)] + [normal(300, dtype=torch.float32, seed=9)]
        before = [g.double() for g in grads]
        norm = ab.clip_grad_norm(grads, limit, out=[g.view(to) for g in grads[:-1]] + grads[-1:])
        want = sum(float(b.square().sum()) for b in before) ** 0.5
        assert abs(float(norm) - want) <= 2.0 ** -21 * want
        f = min(1.0, limit / want)
        for g, b, t in zip(grads, before, [to] * len(shapes) + [torch.float32]):
            # an output is rounded to its type (half a step); the factor and the product to 32 bits (2^-21 with the norm's own error)
            half = torch.finfo(t).eps / 2
            tiny = torch.finfo(t).smallest_normal * torch.finfo(t).eps
            assert bool(((g.view(t).double() - b * f).abs() <= (half + 2.0 ** -21) * b.abs() * f + tiny).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_norm_beyond_32_bits_clips_nothing(dtype):
    """What is returned is not finite, so the gradients stay as they are, and go into other tensors times the scale alone."""
    g = torch.full((64,), 3e38, device="cuda").to(dtype)
    keep = g.clone()
    assert bool(ab.clip_grad_norm([g], 1.0).isinf()) and torch.equal(g, keep)
    out = torch.zeros(64, device="cuda")
    assert bool(ab.clip_grad_norm([g], 1.0, scale=0.125, out=[out]).isfinite()) and not torch.equal(out, 0.125 * keep.float())
    assert bool(ab.clip_grad_norm([g], 1.0, scale=0.5, out=[out]).isinf()) and torch.equal(out, 0.5 * keep.float())
