"""GPU: clipping of gradients where outputs have another type on the same memory, at the ends of the numbers' range, and without memory."""
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


@pytest.mark.parametrize("dtype,to", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float32, torch.float16)])
@pytest.mark.parametrize("value,limit,scale", [(1e38, 1.0, 1.0), (1e38, 1e-6, 1.0), (3e38, 1.0, 2.0 ** -10), (1e30, 1e-15, 1.0), (1e10, 1e-28, 1.0), (1.0, 1e-20, 1e-25)])
def test_factors_below_32_bits_normal_numbers(dtype, to, value, limit, scale):
    """limit / norm under 2^-126, where a 32-bit number has few places left: the outputs have all of theirs."""
    g = (value * (0.1 + 0.9 * torch.rand(3, 67, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)))).to(dtype)
    g[0, 0] = 0.0
    g *= 8.0 ** -1
    keep = g.double()
    out = torch.full(g.shape, torch.nan, device="cuda", dtype=to)
    norm = ab.clip_grad_norm([g], limit, scale=scale, out=[out])
    want = scale * float(keep.square().sum()) ** 0.5
    assert abs(float(norm) - want) <= 2.0 ** -21 * want + 2.0 ** -149
    f = scale * min(1.0, limit / want)
    # rounded to 32 bits and to the output's type; products below 2^-126 have steps of 2^-149, and the factor and its product are rounded there
    tiny = torch.finfo(to).smallest_normal * torch.finfo(to).eps + 2.0 ** -148
    assert bool(((out.double() - keep * f).abs() <= (torch.finfo(to).eps / 2 + 2.0 ** -21) * keep.abs() * f + tiny).all())
    assert float(out[0, 0]) == 0.0


def test_memory_that_runs_out_is_told_as_torch_tells_it():
    """A gradient without memory of its own for each value is copied: more than this process is allowed."""
    g = torch.ones(1, device="cuda").expand(1 << 34)
    torch.cuda.empty_cache()
    torch.cuda.set_per_process_memory_fraction(0.05)
    try:
        with pytest.raises(torch.OutOfMemoryError):
            ab.grad_norm([g])
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    assert float(ab.grad_norm([g[:9]])) == 3.0
