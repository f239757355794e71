"""GPU: the norm over all gradients, and clipping, against 64 bits.

Tolerances. A unit's eight squares are added up in 32 bits (8 * 2^-24 relative at most, half of that in a root), the rest in 64, and the norm is
rounded to 32: NORM = 2^-22 + 2^-24. An output is g times a factor that is rounded to 32 bits, the product rounded to 32 and then to its type: eps / 2 and 3 * 2^-24,
beside NORM for the factor's own error."""
import ctypes as C

import pytest
import torch

import albatross_b200 as ab
from albatross_b200 import _lib

pytestmark = pytest.mark.gpu

DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
NORM = 2.0 ** -22 + 2.0 ** -24


def exact_norm(grads, scale=1.0):
    return scale * sum(float(g.double().square().sum()) for g in grads) ** 0.5


def check(grads, limit, scale=1.0, out=None):
    before = [g.clone() for g in grads]
    norm = ab.clip_grad_norm(grads, limit, scale=scale, out=out)
    want = exact_norm(before, scale)
    assert norm.shape == () and norm.dtype == torch.float32
    assert abs(float(norm) - want) <= NORM * want, (float(norm), want)
    f = scale * (min(1.0, limit / want) if want > limit else 1.0)
    for g, b, o in zip(grads, before, grads if out is None else out):
        if out is not None and o.data_ptr() != g.data_ptr():
            assert torch.equal(g, b)
        half = torch.finfo(o.dtype).eps / 2
        tiny = torch.finfo(o.dtype).smallest_normal * half * 2
        d = (o.double() - b.double() * f).abs()
        assert bool((d <= (half + NORM + 3 * 2.0 ** -24) * b.double().abs() * f + tiny).all())
    return norm


def some(shapes, dtype, seed=0, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(s, device="cuda", generator=g) * std).to(DT[d]) for s, d in zip(shapes, [dtype] * len(shapes) if isinstance(dtype, str) else dtype)]


SHAPES = [(1,), (7,), (8,), (9,), (768,), (12, 64), (33, 31), (1000, 1001), (0,), (5, 0), (2, 3, 4), (), (300, 4096)]


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("limit", [0.5, 1e6])
def test_many_shapes_in_place(dtype, limit):
    check(some(SHAPES, dtype), limit)


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("to", ["fp16", "bf16", "fp32"])
def test_into_other_tensors_and_types(dtype, to):
    grads = some(SHAPES, dtype, seed=1)
    out = [torch.full_like(g, torch.nan, dtype=DT[to]) for g in grads]
    check(grads, 3.0, scale=0.25, out=out)
    check(grads, float("inf"), scale=0.25, out=out)


def test_mixed_types_in_one_list():
    kinds = ["fp16", "bf16", "fp32"] * 5
    grads = some(SHAPES, kinds, seed=2)
    check(grads, 2.0)
    check(some(SHAPES, kinds, seed=3), 2.0, scale=3.0, out=[torch.empty_like(g, dtype=torch.float32) for g in grads])


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("to", ["fp16", "fp32"])
@pytest.mark.parametrize("shift", range(9))
def test_any_address(dtype, to, shift):
    """Views that start anywhere in a larger tensor; outputs on other addresses than the gradients'. What lies around them stays."""
    for n in (1, 3, 8, 13, 777, 20001):
        base = some([(n + 40,)], dtype, seed=n)[0]
        out = torch.full((n + 40,), 99.0, device="cuda", dtype=DT[to])
        for gap in (shift, 0, 5):
            out.fill_(99.0)
            check([base[shift:shift + n]], 0.1, out=[out[gap:gap + n]])
            assert bool((out[:gap] == 99).all()) and bool((out[gap + n:] == 99).all())
        whole = base.clone()
        check([base[shift:shift + n]], 0.1)
        assert torch.equal(base[:shift], whole[:shift]) and torch.equal(base[shift + n:], whole[shift + n:])


def test_a_bucket_with_a_single_value_in_front():
    shapes = [(1,), (768, 3), (2,), (5000,), (1,), (64, 64)]
    n = sum(torch.Size(s).numel() for s in shapes)
    flat, out = some([(n,)], "bf16", seed=4)[0], torch.empty(n, device="cuda")
    grads, outs, at = [], [], 0
    for s in shapes:
        k = torch.Size(s).numel()
        grads.append(flat[at:at + k].view(s)), outs.append(out[at:at + k].view(s))
        at += k
    check(grads, 0.3, out=outs)
    check(grads, 0.3)


@pytest.mark.parametrize("count", [60, 119, 120, 121, 999, 1000, 1001, 2500])
def test_number_of_tensors(count):
    shapes = [(1 + (37 * i) % 300,) for i in range(count)]
    check(some(shapes, "bf16", seed=count), 1.0)
    check(some(shapes, "fp16", seed=count), 1.0, scale=0.5, out=[torch.empty(s, device="cuda") for s in shapes])
    assert abs(float(ab.grad_norm(some(shapes, "fp32", seed=count))) / exact_norm(some(shapes, "fp32", seed=count)) - 1) <= NORM


def test_values_at_the_ends_of_the_range():
    for dtype, v in (("fp32", 1e30), ("fp32", 1e-30), ("fp32", 1e-44), ("bf16", 1e30), ("bf16", 1e-30), ("fp16", 65504.0), ("fp16", 2.0 ** -24), ("fp32", 0.0)):
        g = torch.full((3, 5001), v, device="cuda", dtype=DT[dtype])
        norm = ab.grad_norm([g])
        want = exact_norm([g])
        # (below 2^-126 a result has steps of 2^-149)
        assert abs(float(norm) - want) <= NORM * want + 2.0 ** -149, (dtype, v)
    mixed = some([(4000,)], "fp32", seed=6)[0]
    mixed[::3] = 1e25
    mixed[1::3] = 1e-25
    check([mixed], 1.0)
    zero = [torch.zeros(4096, device="cuda")]
    assert float(ab.clip_grad_norm(zero, 0.0)) == 0.0 and bool((zero[0] == 0).all())
    g = some([(100,)], "fp32")
    ab.clip_grad_norm(g, 0.0)
    assert bool((g[0] == 0).all())


def test_a_norm_that_is_not_finite_clips_nothing():
    for bad in (torch.inf, -torch.inf, torch.nan):
        grads = some([(1000,), (77,)], "fp16", seed=7)
        grads[1][5] = bad
        keep = [g.clone() for g in grads]
        norm = ab.clip_grad_norm(grads, 0.1)
        assert not bool(norm.isfinite()) and torch.equal(grads[0], keep[0])
        out = [torch.empty_like(g, dtype=torch.float32) for g in grads]
        ab.clip_grad_norm(grads, 0.1, scale=0.5, out=out)
        assert torch.equal(out[0], keep[0].float() * 0.5) and not bool(out[1][5].isfinite()) and torch.equal(out[1][:5], keep[1][:5].float() * 0.5)
    big = [torch.full((16,), 3e38, device="cuda")]            # the sum of squares is fine in 64 bits, the norm is not in 32
    assert bool(ab.grad_norm(big).isinf())
    check([torch.full((16,), 1e37, device="cuda")], 1.0)


def test_a_norm_below_the_limit_leaves_every_bit():
    grads = some(SHAPES, "bf16", seed=8)
    keep = [g.clone() for g in grads]
    ab.clip_grad_norm(grads, exact_norm(grads) * 1.001)
    assert all(torch.equal(a, b) for a, b in zip(grads, keep))


def test_tensors_in_other_orders_and_with_gaps():
    for make in (lambda t: t.t(), lambda t: t[:, ::2], lambda t: t[::2], lambda t: t[3:50, 5:40], lambda t: t[:, 0], lambda t: t.view(10, 10, 80).permute(2, 0, 1)):
        base = some([(100, 80)], "fp32", seed=9)[0]
        keep, g = base.clone(), make(base)
        touched = torch.zeros_like(base)
        make(touched).fill_(1)
        check([g, some([(50,)], "fp16")[0]], 0.7)
        assert torch.equal(base[touched == 0], keep[touched == 0])
        other = make(some([(100, 80)], "fp32", seed=9)[0])
        check([other], 0.7, out=[torch.empty(other.shape, device="cuda", dtype=torch.bfloat16)])
        wide = torch.empty(*other.shape, 3, device="cuda")
        check([other.contiguous()], 0.7, out=[wide[..., 1]])
    assert abs(float(ab.grad_norm([torch.ones(5, device="cuda").expand(7, 5)])) - 35 ** 0.5) < 1e-5


def test_large_tensors_repeat_bit_for_bit_and_in_graphs():
    grads = some([(3000, 4096), (65536, 300), (77,), (20000, 1001)], "bf16", seed=10, std=0.01)
    out = [torch.empty_like(g) for g in grads]
    norm = check(grads, 1.0, out=out)
    first = [o.clone() for o in out]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = ab.clip_grad_norm(grads, 1.0, out=out)
    for _ in range(3):
        [o.zero_() for o in out]
        graph.replay()
        assert torch.equal(again, norm) and all(torch.equal(a, b) for a, b in zip(out, first))
    s = torch.cuda.Stream()
    other = some([(1000, 1000)] * 3, "fp32", seed=11)
    want = ab.grad_norm(other)
    torch.cuda.synchronize()
    for _ in range(5):
        with torch.cuda.stream(s):
            b = ab.grad_norm(other)
        a = ab.clip_grad_norm(grads, 1.0, out=out)
        torch.cuda.synchronize()
        assert torch.equal(a, norm) and torch.equal(b, want) and all(torch.equal(x, y) for x, y in zip(out, first))


def test_offsets_beyond_32_bits():
    n = (1 << 31) + 4099
    g = torch.zeros(n, device="cuda", dtype=torch.bfloat16)
    g[::1 << 20] = 2.0
    g[-1] = 3.0
    g[1 << 31] = 5.0
    want = float(g[::1 << 20].double().square().sum() + 9.0) ** 0.5
    norm = ab.clip_grad_norm([g], 1.0)
    assert abs(float(norm) - want) <= NORM * want
    assert abs(float(g[-1]) - 3 / want) <= 2.0 ** -8 * 3 / want and abs(float(g[1 << 31]) - 5 / want) <= 2.0 ** -8 * 5 / want
    assert float(g.sum(dtype=torch.float64)) > 0


def test_what_does_not_fit_is_refused():
    g = some([(100,), (50,)], "fp16")
    flat = torch.zeros(300, device="cuda", dtype=torch.float16)
    leaf = torch.zeros(100, device="cuda", requires_grad=True)
    bad = [dict(grads=[]), dict(grads=[g[0].int()]), dict(grads=[g[0].cpu()]), dict(grads=[g[0].double()]), dict(max_norm=-1.0), dict(max_norm=float("nan")), dict(scale=0.0), dict(scale=-1.0),
           dict(scale=float("inf")), dict(scale=float("nan")), dict(out=[g[0].clone()]), dict(out=[g[0].clone(), g[0].clone()]), dict(out=[g[0].cpu(), g[1].clone()]),
           dict(grads=[g[0], g[0]]), dict(grads=[flat[:100], flat[50:150]]), dict(grads=[flat[:100], flat[200:]], out=[flat[100:200], flat[150:250]]),
           dict(grads=[flat[:100], flat[100:200]], out=[flat[100:200], flat[200:]]), dict(grads=[flat[:100]], out=[flat[1:101]]), dict(grads=[flat[:1].expand(50)]),
           dict(grads=[flat[:100]], out=[flat.view(torch.float32)[:100]]), dict(grads=[g[0]], out=[leaf]), dict(grads=[g[0].to_sparse()]),
           # not dense, and among each other's values
           dict(grads=[flat[:100:2], flat[1:100:2]]), dict(grads=[flat.view(30, 10)[:, :3], flat.view(30, 10)[:, 2:5]]), dict(grads=[flat.view(30, 10)[:20, :3], flat[50:60]])]
    for b in bad:
        args = {"grads": g, "max_norm": 1.0, **b}
        with pytest.raises(RuntimeError):
            ab.clip_grad_norm(args.pop("grads"), args.pop("max_norm"), **args)
    ab.clip_grad_norm([flat[:100], flat[100:200]], 1.0, out=[flat[:100], torch.empty(100, device="cuda")])
    assert float(ab.grad_norm([g[0], g[0]])) == pytest.approx(exact_norm([g[0], g[0]]), rel=1e-6)
    version = flat._version
    ab.clip_grad_norm([flat], 1.0)
    assert flat._version > version
    assert _lib.device_status() == 0


def test_a_step_of_learning_from_drawn_tokens():
    """A 4-bit policy's logits, ids and log-probabilities drawn from them, loss and gradients of an adapter beside it, clipped: as a user puts them together."""
    g = torch.Generator(device="cuda").manual_seed(20)
    V, D, rows = 2000, 256, 24
    head = ab.quantize_int4(0.1 * torch.randn(V, D, device="cuda", generator=g), 64)
    hidden = torch.randn(rows, D, device="cuda", generator=g).half()
    frozen = ab.linear_int4(hidden, *head)
    ids, old = ab.sampler_batch(frozen, torch.rand(rows, device="cuda", generator=g))
    assert torch.allclose(old[:, 0], ab.token_logp(frozen, ids[:, 0]), atol=1e-5)
    adapter = torch.zeros(V, D, device="cuda", dtype=torch.float16, requires_grad=True)
    weight = torch.ones(D, device="cuda", dtype=torch.float16, requires_grad=True)
    advantages = torch.randn(rows, device="cuda", generator=g)
    logits = frozen + ab.layer_norm(hidden, weight) @ adapter.t()
    loss, logp = ab.policy_loss(logits, ids[:, 0], old[:, 0], advantages)
    (loss * 65536.0).backward()
    grads = [adapter.grad, weight.grad]
    out = [torch.empty_like(t, dtype=torch.float32) for t in grads]
    norm = ab.clip_grad_norm(grads, 0.5, scale=1 / 65536.0, out=out)
    # the same in 64 bits: at ratio 1 the loss falls by -A d logp
    x = torch.nn.functional.layer_norm(hidden.double(), (D,)).half().double()
    z = frozen.double()
    d = (torch.softmax(z, -1) - torch.nn.functional.one_hot(ids[:, 0], V)) * (advantages.double() / rows)[:, None]
    want = d.t() @ x
    f = min(1.0, 0.5 / float(want.norm()))
    assert abs(float(norm) - float(want.norm())) <= 2e-3 * float(want.norm())          # (fp16 gradients of logits, fp16 products)
    assert float((out[0].double() - want * f).norm()) <= 3e-3 * float(want.norm()) * f
    assert float(out[0].double().square().sum() + out[1].double().square().sum()) ** 0.5 <= 0.5 * (1 + 1e-5)
