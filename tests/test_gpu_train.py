"""GPU: the operators with gradients against plain implementations in 64 bits.

Tolerances. A result in a 16-bit type is rounded once: at most eps / 2 of each value. What is computed before that is held in 32 bits
(u = 2^-24): a sum of 64 products is off by at most 64 u of the sum of their sizes, some 6 times the sum itself for random signs, and
typically by a tenth of that; a chain of steps with decays below 0.98 adds up to a few such errors. F32 = 2e-5 (about 330 u) covers
that relative to the 2-norm of a tensor; for single values against its largest one, 4 times as much."""
import ctypes as C

import pytest
import torch

import albatross_b200 as ab
from albatross_b200 import _lib

pytestmark = pytest.mark.gpu

F32 = 2e-5
DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def close(got, want, what="", more=0.0, size=0.0):
    """`more`: rounding of intermediate values that the operator is documented to make, relative. `size`: of the terms that a result is the
    difference of, where they cancel."""
    half = torch.finfo(got.dtype).eps / 2
    got, want = got.detach().double(), want.detach().double()
    assert got.shape == want.shape, what
    assert torch.isfinite(got).all() == torch.isfinite(want).all(), what
    d, norm, top = (got - want).abs(), float(want.norm()), float(want.abs().max()) if want.numel() else 0.0
    if norm == 0 and not size:
        assert float(got.abs().sum()) == 0, what
        return
    least = 2.0 ** -25 + F32 * size             # half the smallest fp16 step
    assert float(d.norm()) <= (half + F32 + more) * norm + least * want.numel() ** 0.5, (what, float(d.norm()), norm)
    assert bool((d <= (half + more) * want.abs() + 4 * F32 * top + least).all()), (what, float(d.max()), top)


# ------------------------------------------------------------------------------------------------------------------
# the recurrence
# ------------------------------------------------------------------------------------------------------------------
def wkv_inputs(B, T, H, dtype, seed=0, lo=None, hi=None, lengths=None):
    g = torch.Generator(device="cuda").manual_seed(1000 * seed + 17 * B + 3 * T + H)
    n = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    Cw = H * 64
    r, k, v = (0.7 * n(B, T, Cw) for _ in range(3))
    w = -torch.nn.functional.softplus(-n(B, T, Cw)) - 0.5 if lo is None else lo + (hi - lo) * torch.rand(B, T, Cw, device="cuda", generator=g)
    kk = torch.nn.functional.normalize(n(B, T, H, 64), dim=-1).view(B, T, Cw)
    a, b = -kk, kk * torch.sigmoid(n(B, T, Cw))
    xs = [t.to(DT[dtype]) for t in (r, w, k, v, a, b)]
    return 0.3 * n(B, H, 64, 64), xs, (0.1 * n(B, T, Cw)).to(DT[dtype]), 0.1 * n(B, H, 64, 64)


def wkv_exact(state, xs, lengths=None):
    """The definition, step by step, in the inputs' type."""
    r, w, k, v, a, b = xs
    B, T, Cw = r.shape
    S, ys = state, []
    head = lambda z, t: z[:, t].reshape(B, Cw // 64, 64)  # noqa: E731
    for t in range(T):
        d = torch.exp(-torch.exp(head(w, t)))
        u = torch.einsum("bhij,bhj->bhi", S, head(a, t))
        N = S * d[:, :, None] + torch.einsum("bhi,bhj->bhij", u, head(b, t)) + torch.einsum("bhi,bhj->bhij", head(v, t), head(k, t))
        y = torch.einsum("bhij,bhj->bhi", N, head(r, t))
        if lengths is not None:
            on = (lengths > t)[:, None, None]
            N, y = torch.where(on[..., None], N, S), torch.where(on, y, torch.zeros_like(y))
        S = N
        ys.append(y.reshape(B, Cw))
    return (torch.stack(ys, 1) if ys else r * 0), S


NAMES = ("state", "r", "w", "k", "v", "a", "b")


def wkv_check(state, xs, dy, dout, lengths=None, more=0.0):
    leaves = [t.detach().requires_grad_() for t in (state, *xs)]
    y, out = ab.RWKV7_TRAIN_OP(*leaves, lengths=lengths)
    got = torch.autograd.grad((y, out), leaves, (dy, dout))
    exact = [t.detach().double().requires_grad_() for t in (state, *xs)]
    ye, oute = wkv_exact(exact[0], exact[1:], lengths)
    want = torch.autograd.grad((ye, oute), exact, (dy.double(), dout.double()))
    close(y, ye.detach(), "y", more)
    close(out, oute.detach(), "state", more)
    for n, p, q in zip(NAMES, got, want):
        assert p.dtype == (torch.float32 if n == "state" else xs[0].dtype)
        close(p, q, "d" + n, more)
    return y, out, got


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("B,T,H", [(1, 1, 1), (2, 2, 3), (1, 15, 2), (3, 16, 1), (1, 17, 2), (2, 31, 1), (1, 32, 1), (1, 33, 3), (2, 100, 2), (1, 257, 1)])
def test_recurrence_and_its_gradients(B, T, H, dtype):
    wkv_check(*wkv_inputs(B, T, H, dtype))


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("lo,hi", [(-8.0, -0.5), (-9.0, 1.0), (-2.0, 3.0), (-1.0, 5.0), (4.0, 6.0), (-20.0, -15.0)])
def test_recurrence_with_any_decay(lo, hi, dtype):
    """Decays from none at all to exp(-400), far outside of what the model makes, in one chunk."""
    wkv_check(*wkv_inputs(2, 53, 2, dtype, seed=3, lo=lo, hi=hi))


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("bits", [0.99, 1.01, 1.9, 2.1, 3.9, 4.1, 7.9, 8.1, 15.0, 17.0])
def test_recurrence_around_the_sizes_of_a_steep_chunks_pieces(bits, dtype):
    """Decays of 2^-bits per step, some channels of less: chunks of 16, 8, 4, 2 and 1 steps at once; 37 steps end inside a piece."""
    state, xs, dy, dout = wkv_inputs(2, 37, 2, dtype, seed=31)
    xs[1][:] = torch.log(torch.tensor(bits * 0.6931, dtype=torch.float64)).item()
    xs[1][:, :, ::7] = -1.0
    wkv_check(state, xs, dy, dout)


def test_recurrence_with_a_few_steep_steps():
    """Chunks of ordinary decays beside chunks of steep ones, and single steep channels."""
    state, xs, dy, dout = wkv_inputs(1, 90, 2, "bf16", seed=5)
    xs[1][:, 20] = 4.0
    xs[1][:, 40:44, ::3] = 2.5
    xs[1][:, 70, 5] = 6.0
    wkv_check(state, xs, dy, dout)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("lengths", [(40, 0, 1, 16, 17), (7, 40, 39, 32, 33)])
def test_recurrence_of_unequal_lengths(lengths, dtype):
    """What stands behind a sequence's end is not used, and comes back as zeros."""
    state, xs, dy, dout = wkv_inputs(5, 40, 2, dtype, seed=7)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    clean = [x.clone() for x in xs]
    behind = torch.arange(40, device="cuda")[None] >= n[:, None]
    for i, x in enumerate(xs + [dy]):
        x[behind] = float("nan") if i % 2 else float("inf")
    leaves = [t.detach().requires_grad_() for t in (state, *xs)]
    y, out = ab.RWKV7_TRAIN_OP(*leaves, lengths=n)
    got = torch.autograd.grad((y, out), leaves, (dy, dout))
    exact = [t.double().requires_grad_() for t in (state, *clean)]
    ye, oute = wkv_exact(exact[0], exact[1:], n)
    want = torch.autograd.grad((ye, oute), exact, (dy.masked_fill(behind[..., None], 0).double(), dout.double()))
    close(y, ye.detach(), "y")
    close(out, oute.detach(), "state")
    for name, p, q in zip(NAMES, got, want):
        close(p, q, "d" + name)
        if name != "state":
            assert bool((p[behind] == 0).all())
    assert bool((y[behind] == 0).all())
    assert torch.equal(out[lengths.index(0)] if 0 in lengths else out[:0], state[lengths.index(0)] if 0 in lengths else state[:0])


def test_recurrence_takes_lengths_into_their_range():
    state, xs, dy, dout = wkv_inputs(2, 20, 1, "fp16")
    y, out = ab.RWKV7_TRAIN_OP(state, *xs, lengths=torch.tensor([-3, 99], dtype=torch.int32, device="cuda"))
    want, wout = ab.RWKV7_TRAIN_OP(state, *xs)
    assert torch.equal(y[1], want[1]) and torch.equal(out[1], wout[1]) and bool((y[0] == 0).all()) and torch.equal(out[0], state[0])


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_recurrence_of_strided_inputs(dtype):
    """Slices of one projection, steps before sequences, odd addresses and an upstream gradient without strides."""
    B, T, H = 2, 35, 2
    state, xs, dy, dout = wkv_inputs(B, T, H, dtype, seed=9)
    want, wout = ab.RWKV7_TRAIN_OP(state, *xs)
    packed = torch.cat(xs, -1)                                          # [B, T, 6 C]
    slices = packed.split(H * 64, -1)
    turned = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in xs]   # [T, B, C] in memory
    odd = [torch.cat([x.new_zeros(1), x.reshape(-1)])[1:].view(x.shape) for x in xs]
    backwards = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in xs]   # the last dimension is not dense
    for other in (slices, turned, odd, backwards):
        leaves = [t.detach().requires_grad_() for t in (state, *other)]
        y, out = ab.RWKV7_TRAIN_OP(*leaves)
        assert torch.equal(y, want) and torch.equal(out, wout)
        one = torch.ones((), device="cuda", dtype=y.dtype)
        g1 = torch.autograd.grad((y, out), leaves, (one.expand(y.shape), dout), retain_graph=True)
        g2 = torch.autograd.grad((y, out), leaves, (torch.ones_like(y), dout))
        assert all(torch.equal(p, q) for p, q in zip(g1, g2))
    wkv_check(state, odd, torch.cat([dy.new_zeros(3), dy.reshape(-1)])[3:].view(dy.shape), dout)


def test_recurrence_of_states_inside_larger_tensors():
    """A state and its gradient that start 4 bytes behind a 16-byte boundary, as narrowing a larger tensor leaves them."""
    state, xs, dy, dout = wkv_inputs(1, 20, 2, "fp16")
    inside = lambda t: torch.cat([t.new_zeros(1), t.flatten()])[1:].view(t.shape)  # noqa: E731
    leaves = [state.clone().requires_grad_()] + [x.clone().requires_grad_() for x in xs]
    want = ab.RWKV7_TRAIN_OP(*leaves)
    want_g = torch.autograd.grad(want, leaves, (dy, dout))
    y, out = ab.RWKV7_TRAIN_OP(inside(leaves[0]), *leaves[1:])
    joined = torch.cat([out.new_zeros(1), out.flatten()])
    got_g = torch.autograd.grad((y, joined), leaves, (dy, torch.cat([dout.new_zeros(1), dout.flatten()])))
    assert torch.equal(y, want[0]) and torch.equal(out, want[1])
    assert all(torch.equal(a, b) for a, b in zip(got_g, want_g))


def test_recurrence_without_a_state_and_with_some_gradients():
    state, xs, dy, dout = wkv_inputs(2, 21, 2, "bf16", seed=11)
    leaves = [t.detach().requires_grad_() for t in xs]
    y, out = ab.RWKV7_TRAIN_OP(None, *leaves)
    got = torch.autograd.grad(y, leaves, dy)                            # nothing comes from the state
    exact = [t.double().requires_grad_() for t in xs]
    ye, oute = wkv_exact(torch.zeros_like(state).double(), exact)
    for p, q in zip(got, torch.autograd.grad(ye, exact, dy.double())):
        close(p, q)
    # the state alone (what tuning a state asks for), from the last state alone
    s = state.clone().requires_grad_()
    y, out = ab.RWKV7_TRAIN_OP(s, *xs)
    g, = torch.autograd.grad(out, s, dout)
    se = state.double().requires_grad_()
    close(g, torch.autograd.grad(wkv_exact(se, [x.double() for x in xs])[1], se, dout.double())[0])
    with torch.no_grad():
        assert not ab.RWKV7_TRAIN_OP(s, *leaves)[0].requires_grad


def test_recurrence_of_no_steps():
    state, xs, _, dout = wkv_inputs(2, 0, 1, "fp16")
    s = state.clone().requires_grad_()
    y, out = ab.RWKV7_TRAIN_OP(s, *xs)
    assert y.shape == (2, 0, 64) and torch.equal(out, state)
    assert torch.equal(torch.autograd.grad(out, s, dout)[0], dout)


def test_recurrence_gives_the_same_every_time_and_in_every_batch():
    state, xs, dy, dout = wkv_inputs(3, 50, 2, "fp16", seed=13)

    def run(at):
        leaves = [t[at].detach().clone().requires_grad_() for t in (state, *xs)]
        y, out = ab.RWKV7_TRAIN_OP(*leaves)
        return (y, out) + torch.autograd.grad((y, out), leaves, (dy[at], dout[at]))
    whole = run(slice(None))
    assert all(torch.equal(p, q) for p, q in zip(whole, run(slice(None))))
    assert all(torch.equal(p[1:2], q) for p, q in zip(whole, run(slice(1, 2))))


def test_recurrence_agrees_with_the_inference_operator():
    state, xs, _, _ = wkv_inputs(2, 45, 3, "fp16", seed=15)
    mine, y = state.clone(), None
    y = ab.RWKV7_BATCH_OP(mine, *xs)
    got, out = ab.RWKV7_TRAIN_OP(state, *xs)
    close(got, y.double(), more=2.0 ** -11)     # both are rounded
    close(out, mine.double())


def test_recurrence_in_pieces_equals_the_whole():
    state, xs, _, _ = wkv_inputs(1, 64, 2, "bf16", seed=17)
    y, out = ab.RWKV7_TRAIN_OP(state, *xs)
    y1, s = ab.RWKV7_TRAIN_OP(state, *(x[:, :32] for x in xs))
    y2, s = ab.RWKV7_TRAIN_OP(s, *(x[:, 32:] for x in xs))
    assert torch.equal(torch.cat([y1, y2], 1), y) and torch.equal(s, out)


def test_recurrence_against_differences():
    """Along a direction, the gradient is what the 64-bit formula's outputs change by."""
    state, xs, dy, dout = wkv_inputs(1, 20, 1, "bf16", seed=19)
    leaves = [t.detach().requires_grad_() for t in (state, *xs)]
    y, out = ab.RWKV7_TRAIN_OP(*leaves)
    grads = torch.autograd.grad((y, out), leaves, (dy, dout))
    base = [t.detach().double() for t in leaves]
    for i, (g, name) in enumerate(zip(grads, NAMES)):
        step = 1e-4 * torch.randn(base[i].shape, device="cuda", dtype=torch.float64, generator=torch.Generator(device="cuda").manual_seed(i))
        side = []
        for sign in (1, -1):
            moved = [b + sign * step if j == i else b for j, b in enumerate(base)]
            ye, oute = wkv_exact(moved[0], moved[1:])
            side.append(float((ye * dy).sum() + (oute * dout).sum()))
        # rounding to bf16: 2^-8 of each value at most, of random sign, so that the errors add up as their 2-norm (twice it is 7 deviations);
        # the difference's own error is of third order, 1e-8 of it
        want, got = (side[0] - side[1]) / 2, float((g.double() * step).sum())
        assert abs(got - want) <= (2.0 ** -8 + 1e-4) * float((g.double() * step).norm()) * 2, name


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("B,T,H", [(150, 20, 1), (37, 35, 5), (1, 700, 1), (2, 129, 75)])
def test_recurrence_of_more_heads_than_sms_and_of_long_sequences(B, T, H, dtype):
    wkv_check(*wkv_inputs(B, T, H, dtype, seed=21))


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_recurrence_of_unequal_lengths_with_steep_steps(dtype):
    """Chunks that end inside, in pieces: their rows behind the end come back as zeros all the same."""
    state, xs, dy, dout = wkv_inputs(4, 45, 2, dtype, seed=23, lo=-2.0, hi=3.0)
    n = torch.tensor([45, 33, 17, 5], dtype=torch.int32, device="cuda")
    behind = torch.arange(45, device="cuda")[None] >= n[:, None]
    clean = [x.clone() for x in xs]
    for x in xs + [dy]:
        x[behind] = float("nan")
    leaves = [t.detach().requires_grad_() for t in (state, *xs)]
    y, out = ab.RWKV7_TRAIN_OP(*leaves, lengths=n)
    got = torch.autograd.grad((y, out), leaves, (dy, dout))
    exact = [t.double().requires_grad_() for t in (state, *clean)]
    ye, oute = wkv_exact(exact[0], exact[1:], n)
    want = torch.autograd.grad((ye, oute), exact, (dy.masked_fill(behind[..., None], 0).double(), dout.double()))
    close(y, ye.detach(), "y")
    close(out, oute.detach(), "state")
    for name, p, q in zip(NAMES, got, want):
        close(p, q, "d" + name)
        assert name == "state" or bool((p[behind] == 0).all())


def test_recurrence_of_small_and_large_values():
    """Scales far from 1: gradients as small as those of a mean over many tokens, keys and states in the thousands. Everything is linear in v and the state together, and
    in dy and the state's gradient together: exact powers of two change nothing but the exponent."""
    state, xs, dy, dout = wkv_inputs(1, 40, 2, "bf16", seed=25)

    def run(scale, gscale):
        leaves = [t.detach().requires_grad_() for t in (state * scale, *xs[:3], xs[3] * scale, *xs[4:])]
        y, out = ab.RWKV7_TRAIN_OP(*leaves)
        return y, out, torch.autograd.grad((y, out), leaves, (dy * gscale, dout * gscale))
    y, out, g = run(1.0, 1.0)
    for scale, gscale in ((2.0 ** 12, 2.0 ** -30), (2.0 ** -20, 2.0 ** 10)):
        y2, out2, g2 = run(scale, gscale)
        assert torch.equal(y2, y * scale) and torch.equal(out2, out * scale)
        for name, p, q in zip(NAMES, g2, g):
            assert torch.equal(p, q * (gscale if name in ("state", "v") else scale * gscale)), name


def test_recurrence_keeps_a_nan_in_its_head():
    state, xs, dy, dout = wkv_inputs(2, 40, 2, "fp16", seed=27)
    y, out = ab.RWKV7_TRAIN_OP(state, *xs)
    xs[2][0, 20, 70] = float("nan")             # a key of sequence 0, head 1, step 20
    y2, out2 = ab.RWKV7_TRAIN_OP(state, *xs)
    assert torch.equal(y2[1], y[1]) and torch.equal(y2[0, :, :64], y[0, :, :64]) and torch.equal(y2[0, :16], y[0, :16])
    assert bool(torch.isnan(y2[0, 20:, 64:]).all()) and torch.equal(out2[1], out[1]) and bool(torch.isnan(out2[0, 1, :, 6]).all())


def test_recurrence_of_one_tensor_in_two_places():
    """Its gradient is the sum of both places'."""
    state, xs, dy, _ = wkv_inputs(1, 30, 1, "bf16", seed=29)
    x = xs[0].detach().requires_grad_()
    y, _ = ab.RWKV7_TRAIN_OP(state, x, xs[1], x, xs[3], xs[4], xs[5])
    got, = torch.autograd.grad(y, x, dy)
    r, k = (xs[0].detach().clone().requires_grad_() for _ in range(2))
    y2, _ = ab.RWKV7_TRAIN_OP(state, r, xs[1], k, xs[3], xs[4], xs[5])
    dr, dk = torch.autograd.grad(y2, (r, k), dy)
    assert torch.equal(y, y2) and torch.equal(got, dr + dk)


# ------------------------------------------------------------------------------------------------------------------
# the norms
# ------------------------------------------------------------------------------------------------------------------
def norm_exact(x, w, b, eps, groups):
    g = x.reshape(*x.shape[:-1], groups, -1)
    c = g - g.mean(-1, keepdim=True)
    y = (c / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)).reshape(x.shape)
    y = y if w is None else y * w
    return y if b is None else y + b


def norm_check(x, w, b, eps=1e-5, groups=1, dy=None, size=0.0):
    leaves = [t.detach().requires_grad_() for t in (x, w, b) if t is not None]
    it = iter(leaves)
    lx, lw, lb = (None if t is None else next(it) for t in (x, w, b))
    y = ab.layer_norm(lx, lw, lb, eps=eps, groups=groups)
    dy = torch.randn(y.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(y.dtype) if dy is None else dy
    got = torch.autograd.grad(y, leaves, dy)
    exact = [t.detach().double().requires_grad_() for t in leaves]
    it = iter(exact)
    ye = norm_exact(*(None if t is None else next(it) for t in (x, w, b)), eps, groups)
    want = torch.autograd.grad(ye, exact, dy.double())
    close(y, ye.detach(), "y")
    for p, q in zip(got, want):
        close(p, q, "grad", size=size)
    with torch.no_grad():
        assert torch.equal(ab.layer_norm(lx, lw, lb, eps=eps, groups=groups), y)


def norm_inputs(n, Cn, dtype, wtype=None, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + 31 * n + Cn)
    x = (2 * torch.randn(n, Cn, device="cuda", generator=g) + torch.randn(n, 1, device="cuda", generator=g)).to(DT[dtype])
    w = (0.8 + 0.4 * torch.rand(Cn, device="cuda", generator=g)).to(DT[wtype or dtype])
    return x, w, (0.1 * torch.randn(Cn, device="cuda", generator=g)).to(DT[wtype or dtype])


@pytest.mark.parametrize("dtype,wtype", [("fp16", "fp16"), ("bf16", "bf16"), ("fp32", "fp32"), ("fp16", "fp32"), ("bf16", "fp32")])
@pytest.mark.parametrize("n,Cn,groups", [(1, 768, 1), (5, 1, 1), (3, 33, 1), (300, 768, 1), (129, 1000, 1), (64, 2560, 1), (17, 4096, 1), (9, 8192, 1), (3, 20001, 1),
                                         (1, 64, 1), (70, 768, 12), (33, 2560, 40), (200, 4096, 64), (7, 96, 3), (5, 100, 4), (9, 1024, 2), (6, 12, 12)])
def test_layer_norm_and_its_gradients(n, Cn, groups, dtype, wtype):
    if Cn == groups or Cn == 1:     # groups of one value: the output is the bias, gradients by x and weight are 0
        x, w, b = norm_inputs(n, Cn, dtype, wtype)
        leaves = [t.requires_grad_() for t in (x, w, b)]
        y = ab.layer_norm(*leaves, groups=groups)
        assert torch.equal(y, b.to(y.dtype).expand(n, Cn))
        dx, dw, db = torch.autograd.grad(y, leaves, torch.ones_like(y))
        assert float(dx.abs().max()) == 0 and float(dw.abs().max()) == 0 and bool((db == n).all())
        return
    norm_check(*norm_inputs(n, Cn, dtype, wtype), eps=64e-5 if groups > 1 else 1e-5, groups=groups)


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
def test_layer_norm_of_strided_rows_and_missing_weights(dtype):
    x, w, b = norm_inputs(40, 2304, dtype)
    norm_check(x[:, 256:1280], w[:1024], b[:1024])                      # a slice of wider rows
    norm_check(x[::2], w, b)
    norm_check(x[:, 1:1001], w[1:1001], b[3:1003])                      # odd addresses
    norm_check(x.view(4, 10, 2304).transpose(0, 1), w, b)               # rows without one stride
    norm_check(x.t().contiguous().t()[:, :768], w[:768], None)
    norm_check(x, None, None)
    # dx = rstd (e - mean(e) - xh mean(e xh)) with e = 1 everywhere is 0: what is left of three terms of at most 1, each within some u, at rstd below 1
    norm_check(x, None, b, dy=torch.ones((), device="cuda", dtype=x.dtype).expand(x.shape), size=1.0)
    norm_check(x[:, :768], w[:768], b[:768], groups=12, dy=x[:, 768:1536])   # an upstream gradient with strides


def test_layer_norm_of_many_rows_adds_the_weights_gradients_in_one_order():
    x, w, b = norm_inputs(5001, 768, "bf16")
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = ab.layer_norm(*leaves)
    dy = torch.randn_like(y)
    first = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    assert all(torch.equal(p, q) for p, q in zip(first, torch.autograd.grad(y, leaves, dy)))
    norm_check(x, w, b, dy=dy)


def test_layer_norm_of_nothing_and_of_constants():
    x, w, b = norm_inputs(0, 64, "fp16")
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = ab.layer_norm(*leaves)
    dx, dw, db = torch.autograd.grad(y, leaves, torch.empty_like(y))
    assert y.shape == (0, 64) and dx.shape == (0, 64) and float(dw.abs().sum()) == 0 and float(db.abs().sum()) == 0
    x = torch.full((3, 256), 7.0, device="cuda", dtype=torch.bfloat16)
    assert float(ab.layer_norm(x).abs().max()) == 0
    x[1, 5] = float("nan")
    y = ab.layer_norm(x)
    assert bool(torch.isnan(y[1]).all()) and float(y[0].abs().max()) == 0 and float(y[2].abs().max()) == 0


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("Cn,groups", [(768, 1), (1000, 1), (2560, 1), (33, 1), (5000, 1), (12288, 1), (2560, 40), (96, 12), (96, 1), (4104, 1)])
def test_layer_norm_of_rows_of_one_value_is_the_bias(Cn, groups, dtype):
    """The sum of Cn equal values of few bits is exact, and so has their mean to be, whether or not 1 / Cn is: with rstd = 316 (eps 1e-5, no variance) a mean of
    1000 that is off by half a step, 3e-5, would come out as 0.01."""
    x = torch.tensor([7.0, 1000.0, -1000.0, 96.0], device="cuda").to(DT[dtype])[:, None].expand(4, Cn).contiguous()
    b = torch.randn(Cn, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).to(DT[dtype])
    assert float(ab.layer_norm(x, groups=groups).abs().max()) == 0
    leaf = x.clone().requires_grad_()
    y = ab.layer_norm(leaf, torch.ones_like(b).requires_grad_(), b, groups=groups)
    assert torch.equal(y, b.expand(4, Cn))


@pytest.mark.parametrize("n,Cn,groups,dtype", [(70001, 33, 1, "bf16"), (30000, 64, 1, "fp16"), (20000, 128, 2, "bf16"), (5000, 1024, 16, "fp32")])
def test_layer_norm_of_many_short_rows(n, Cn, groups, dtype):
    norm_check(*norm_inputs(n, Cn, dtype), groups=groups)


def test_layer_norm_gradients_of_some_inputs():
    x, w, b = norm_inputs(50, 512, "bf16")
    dy = torch.randn_like(x)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    want = torch.autograd.grad(ab.layer_norm(*leaves), leaves, dy)
    for i in range(3):
        mine = [t.detach() for t in (x, w, b)]
        mine[i].requires_grad_()
        assert torch.equal(torch.autograd.grad(ab.layer_norm(*mine), mine[i], dy)[0], want[i])
    lb = b.detach().requires_grad_()
    assert torch.equal(torch.autograd.grad(ab.layer_norm(x, None, lb), lb, dy)[0], want[2])


# ------------------------------------------------------------------------------------------------------------------
# log-probabilities and losses
# ------------------------------------------------------------------------------------------------------------------
def logit_inputs(n, V, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + 7 * n + V)
    x = (3 * torch.randn(n, V, device="cuda", generator=g)).to(DT[dtype])
    ids = torch.randint(V, (n,), device="cuda", generator=g)
    return x, torch.where(torch.rand(n, device="cuda", generator=g) < 0.5, x.argmax(-1), ids), g


def logp_exact(x, ids):
    return torch.log_softmax(x, -1).gather(-1, ids[..., None])[..., 0]


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("n,V", [(1, 1), (3, 7), (1, 65536), (5, 1000), (40, 4099), (150, 50277), (600, 2048), (2, 200003)])
def test_token_logp_and_its_gradient(n, V, dtype):
    x, ids, g = logit_inputs(n, V, dtype)
    mask = torch.rand(n, device="cuda", generator=g) < 0.8
    dl = torch.randn(n, device="cuda", generator=g)
    for m in (None, mask):
        lx = x.detach().requires_grad_()
        logp = ab.token_logp(lx, ids, m)
        dx, = torch.autograd.grad(logp, lx, dl)
        xe = x.double().requires_grad_()
        le = logp_exact(xe, ids) * (1.0 if m is None else m.double())
        want, = torch.autograd.grad(le, xe, dl.double())
        # a sum of exponentials held in 32 bits, each good to 2^-22: its logarithm is off by 2^-21 at most, also where the result is 0 (a vocabulary of one)
        close(logp, le.detach(), "logp", size=2.0 ** -21 / F32)
        # (there the gradient is 0 as well, the difference of the upstream gradient and itself times that)
        close(dx, want, "dlogits", size=2.0 ** -21 / F32 * float(dl.abs().max()))
        if m is not None:
            assert bool((logp[~m] == 0).all()) and bool((dx[~m] == 0).all())
        with torch.no_grad():
            assert torch.equal(ab.token_logp(lx, ids, m), logp)


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
def test_token_logp_does_not_look_at_masked_rows(dtype):
    x, ids, _ = logit_inputs(6, 3001, dtype)
    mask = torch.tensor([1, 0, 1, 0, 1, 0], device="cuda").bool()
    want = ab.token_logp(x, ids)
    x[1], x[3, 5], x[5] = float("nan"), float("inf"), -float("inf")
    bad = ids.clone()
    bad[1], bad[3], bad[5] = -100, 1 << 40, -1
    lx = x.requires_grad_()
    logp = ab.token_logp(lx, bad, mask)
    assert torch.equal(logp, want * mask)
    dx, = torch.autograd.grad(logp.sum(), lx)
    assert bool((dx[~mask] == 0).all()) and bool(torch.isfinite(dx).all())
    assert _lib.device_status() == 0
    nobody = ab.token_logp(lx, bad, torch.zeros_like(mask))
    assert bool((nobody == 0).all())


def test_token_logp_of_infinities():
    """Tokens that a program has ruled out, the chosen one among them; rows of nothing but -inf and rows with NaN give NaN, as the formula does."""
    x, ids, _ = logit_inputs(5, 1003, "fp32")
    x[0, 100:900] = -float("inf")
    ids[0] = 5
    x[1, 7], ids[1] = -float("inf"), 7
    x[2] = -float("inf")
    x[3, 17] = float("nan")
    x[4, 3], ids[4] = 1e30, 3
    lx = x.requires_grad_()
    out = ab.token_logp(lx, ids)
    logp, want = out.detach(), logp_exact(x.detach().double(), ids)
    assert float(logp[1]) == -float("inf") and bool(torch.isnan(logp[2])) and bool(torch.isnan(logp[3])) and abs(float(logp[4])) <= 2.0 ** -21
    close(logp[:1], want[:1])
    dx, = torch.autograd.grad(out, lx, torch.ones_like(logp))
    assert bool((dx[0, 100:900] == 0).all()) and abs(float(dx[0].double().sum())) < 1e-5
    p = torch.softmax(x.detach()[1].double(), -1)
    close(dx[1, 8:], -p[8:])


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
def test_token_logp_of_the_types_ends(dtype):
    """Rows of the type's lowest value but for a few, or throughout (what some programs mask with), and of large values."""
    x, ids, _ = logit_inputs(6, 2049, dtype)
    low, high = torch.finfo(x.dtype).min, torch.finfo(x.dtype).max
    x[0, 3:2000] = low
    x[1] = low
    x[2] = high
    x[3, 1000:] = high
    x[4], x[4, 7] = low, high
    x[5] += 1000
    ids[0], ids[3], ids[4] = 2048, 1500, 7
    lx = x.requires_grad_()
    logp = ab.token_logp(lx, ids)
    xe = x.detach().double().requires_grad_()
    want = logp_exact(xe, ids)
    close(logp, want, size=2.0 ** -21 / F32)
    close(torch.autograd.grad(logp.sum(), lx)[0], torch.autograd.grad(want.sum(), xe)[0], size=2.0 ** -21 / F32)


def test_token_logp_reports_ids_outside_the_vocabulary():
    x, ids, _ = logit_inputs(4, 100, "fp16")
    assert _lib.device_status() == 0
    ids[1], ids[2] = 100, -1
    logp = ab.token_logp(x, ids)
    want = ab.token_logp(x, ids.clamp(0, 99))
    assert torch.equal(logp, want) and _lib.device_status() == 8


def test_token_logp_of_strided_logits_and_short_ids():
    x, ids, _ = logit_inputs(12, 5000, "bf16")
    wide = x[:, 3:4003]
    want = ab.token_logp(wide.contiguous(), ids.clamp(max=3999))
    lx = wide.detach().requires_grad_()
    got = ab.token_logp(lx, ids.clamp(max=3999).int())
    close(got, want.double(), "logp")       # (a row is added up from one 16-byte boundary to the next: other addresses, another order)
    dx, = torch.autograd.grad(got.sum(), lx)
    xe = wide.detach().double().requires_grad_()
    close(dx, torch.autograd.grad(logp_exact(xe, ids.clamp(max=3999)).sum(), xe)[0], "dlogits")
    cube = x.view(3, 4, 5000).transpose(0, 1)
    assert torch.equal(ab.token_logp(cube, ids.view(3, 4).t()), ab.token_logp(x, ids).view(3, 4).t())
    assert ab.token_logp(x[:0], ids[:0]).shape == (0,)


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
def test_losses_of_rows_that_share_their_logits(dtype):
    """One row of logits for many ids, by expand() or as a window over a longer one: gradients come back summed, as torch adds up what it expanded."""
    x, ids, g = logit_inputs(6, 700, dtype)
    dl = torch.randn(6, device="cuda", generator=g)
    A = torch.randn(6, device="cuda", generator=g)
    row = x[0].clone()
    for shared in (lambda t: t.expand(6, 700), lambda t: t.as_strided((6, 400), (60, 1))):
        one = row.detach().requires_grad_()
        wide = shared(one)
        at = ids % wide.shape[1]
        dense = wide.detach().contiguous().requires_grad_()
        logp, want = ab.token_logp(wide, at), ab.token_logp(dense, at)
        assert torch.equal(logp, want)
        got, = torch.autograd.grad(logp, wide, dl, retain_graph=True)
        d, = torch.autograd.grad(want, dense, dl)
        assert torch.equal(got, d)
        if wide.stride(0) == 0:
            assert torch.equal(torch.autograd.grad(logp, one, dl)[0], d.sum(0))
        with torch.no_grad():
            assert all(torch.equal(p, q) for p, q in zip(ab.policy_loss_grad(wide, at, None, A), ab.policy_loss_grad(dense, at, None, A)))
            assert all(torch.equal(p, q) for p, q in zip(ab.policy_loss(wide, at, None, A), ab.policy_loss(dense, at, None, A)))
    cube = row.expand(2, 3, 700)
    assert all(torch.equal(p, q) for p, q in zip(ab.preference_loss(cube, ids.view(2, 3), A[:2]), ab.preference_loss(cube.contiguous(), ids.view(2, 3), A[:2])))


def test_token_logp_of_more_than_2_to_the_31_logits():
    V, n = 65536, 33000
    x = torch.zeros(n, V, dtype=torch.float16, device="cuda")
    x[-1], x[-2, 5] = 0.5, 3.0
    ids = torch.full((n,), 5, device="cuda")
    lx = x.requires_grad_()
    logp = ab.token_logp(lx, ids)
    want = logp_exact(x.detach()[-3:].double(), ids[-3:])
    close(logp[-3:], want)
    dx, = torch.autograd.grad(logp.sum(), lx)
    close(dx[-1], (torch.nn.functional.one_hot(ids[-1:], V).double() - 1.0 / V)[0])
    assert float(dx[0, 5]) > 0.99 and float(dx[40, 6]) < 0


def policy_exact(x, ids, old, A, mask, ref_logp, clip, kl, denom):
    logp = logp_exact(x, ids)
    ratio = torch.exp(logp - (logp.detach() if old is None else old.double()))
    each = -torch.min(ratio * A, torch.clamp(ratio, 1 - clip[0], 1 + clip[1]) * A)
    if ref_logp is not None:
        gap = ref_logp.double() - logp
        each = each + kl * (torch.exp(gap) - gap - 1)
    live = torch.ones_like(logp) if mask is None else mask.double()
    return (each * live).sum() / (denom or max(1.0, float(live.sum()))), logp * live


def policy_inputs(n, V, dtype, seed=0):
    x, ids, g = logit_inputs(n, V, dtype, seed)
    logp = logp_exact(x.double(), ids).float()
    r = lambda: torch.randn(n, device="cuda", generator=g)  # noqa: E731
    old = logp + 0.2 * r()
    ratio = torch.exp(logp - old)
    for edge in (0.8, 1.2, 0.9, 1.3):       # off the borders: there the gradient jumps
        old = torch.where((ratio - edge).abs() < 1e-3, old + 0.01, old)
    return x, ids, old, r(), torch.rand(n, device="cuda", generator=g) < 0.8, logp + 0.4 * r()


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("n,V", [(1, 17), (24, 65536), (37, 1003), (300, 4096), (5, 131071)])
@pytest.mark.parametrize("form", ["all", "plain", "on_policy"])
def test_policy_loss_and_its_gradient(n, V, dtype, form):
    x, ids, old, A, mask, ref = policy_inputs(n, V, dtype)
    scale = 4096.0 if dtype == "fp16" else 1.0
    if form == "all":
        old_, more = old, {"mask": mask, "ref_logp": ref, "clip": (0.1, 0.3), "kl": 0.05, "denom": None}
    elif form == "plain":
        old_, more = old, {"mask": None, "ref_logp": None, "clip": (0.2, 0.2), "kl": 0.0, "denom": 2.5 * n}
    else:
        old_, more = None, {"mask": mask, "ref_logp": None, "clip": (0.2, 0.2), "kl": 0.0, "denom": None}
    xe = x.double().requires_grad_()
    le, logpe = policy_exact(xe, ids, old_, A.double(), **more)
    want, = torch.autograd.grad(le * scale, xe)
    lx = x.detach().requires_grad_()
    loss, logp = ab.policy_loss(lx, ids, old_, A, **more)
    assert loss.requires_grad and not logp.requires_grad
    dx, = torch.autograd.grad(loss * scale, lx)
    # the loss is a sum of terms of both signs: its error is relative to their sizes, at most max(|A|) e^1 + 1
    assert abs(float(loss) - float(le)) <= F32 * (float(A.abs().max()) * 3 + 1)
    close(logp, logpe.detach(), "logp")
    close(dx, want, "dlogits")
    with torch.no_grad():
        assert torch.equal(ab.policy_loss(lx, ids, old_, A, **more)[0], loss)
    loss2, logp2, dx2 = ab.policy_loss_grad(lx, ids, old_, A, scale=scale, **more)
    assert torch.equal(loss2, loss) and torch.equal(logp2, logp)
    close(dx2, want, "dlogits, one pass")
    here = x.clone()
    loss3, logp3, dx3 = ab.policy_loss_grad(here, ids, old_, A, scale=scale, out=here, **more)
    assert dx3.data_ptr() == here.data_ptr() and torch.equal(dx3, dx2) and torch.equal(loss3, loss) and torch.equal(logp3, logp)


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("n,V", [(160, 500), (9, 4099), (160, 20011)])
def test_policy_gradients_where_a_factor_is_nothing_or_exponentials_are_large(n, V, dtype):
    """Advantages of 0 (a group whose rewards are all equal), a reference without weight, ratios and penalties beyond what an exponential holds in 32 bits: one pass and
    autograd both, in each of the kernels. The coefficient of a row whose exponential e is finite in 64 bits is taken there: what is left is its rounding, beside e's own
    relative error, which is the log-probability's absolute one of 2^-21 at most."""
    x, ids, old, A, mask, ref = policy_inputs(n, V, dtype, seed=3)
    mask[:] = True
    A = A.abs() + 0.5
    logp = logp_exact(x.double(), ids).float()
    none = {"mask": mask, "clip": (0.2, 0.2), "denom": None}

    def both(old_, A_, **more):
        lx = x.detach().requires_grad_()
        loss, _ = ab.policy_loss(lx, ids, old_, A_, **more)
        one, _, dx = ab.policy_loss_grad(x, ids, old_, A_, **more)
        assert torch.equal(one, loss)
        return loss, torch.autograd.grad(loss, lx)[0], dx

    def check(old_, A_, **more):
        xe = x.double().requires_grad_()
        le, _ = policy_exact(xe, ids, old_, A_.double(), **none, **more)
        want, = torch.autograd.grad(le, xe)
        assert bool(torch.isfinite(want).all())
        loss, *got = both(old_, A_, **none, **more)
        assert abs(float(loss) - float(le)) <= (F32 + 2.0 ** -21) * max(1.0, abs(float(le)))
        for g in got:
            close(g, want, "dlogits", more=2.0 ** -21)
    zero = torch.where(torch.arange(n, device="cuda") % 3 == 0, torch.zeros_like(A), A)
    far = torch.where(torch.arange(n, device="cuda") % 3 == 0, logp - 100.0, old)
    check(far, zero, ref_logp=None, kl=0.0)                              # a ratio of e^100 with an advantage of 0
    check(far, zero, ref_logp=ref, kl=0.05)
    check(old, A, ref_logp=torch.where(torch.arange(n, device="cuda") % 4 == 1, logp + 100.0, ref), kl=0.0)
    # e^89.5 is beyond 32 bits, a tenth of a millionth of it is not (and, times a probability, what the type holds)
    if dtype != "fp16":
        check(old, A, ref_logp=torch.where(torch.arange(n, device="cuda") == 1, logp + 89.5, ref), kl=1e-7)
    # beyond 64 bits a factor of 0 is still 0
    want = both(old, zero, ref_logp=None, kl=0.0, **none)
    for got in (both(torch.where(zero == 0, logp - 800.0, old), zero, ref_logp=None, kl=0.0, **none), both(old, zero, ref_logp=logp + 800.0, kl=0.0, **none)):
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    # with another sign the loss has no bound; a clipped ratio has one, and no gradient
    gone = torch.where(torch.arange(n, device="cuda") == 2, logp - 800.0, old)
    loss, *got = both(gone, A, ref_logp=None, kl=0.0, **none)
    assert bool(torch.isfinite(loss)) and all(bool((g[2] == 0).all()) and bool(torch.isfinite(g).all()) for g in got)
    assert float(both(gone, -A, ref_logp=None, kl=0.0, **none)[0]) == float("inf")


@pytest.mark.parametrize("n,V", [(7, 1000), (7, 3001), (160, 20011)])
def test_policy_gradient_of_small_gaps(n, V):
    """Where the advantage is 0 the penalty's kl (1 - exp(ref - logp)) is the whole gradient. Rows of equal logits: exponentials and their sum are exact, so that the coefficient
    is a matter of its own arithmetic. It comes from 64 bits (2^-52 of a log-probability of about 10, which over a gap of 1e-5 is 2e-10); up to six roundings to 32 bits follow
    (the coefficient, the scale, the sum's reciprocal, products), 4e-7. A logarithm in 32 bits, 5e-7 off, would put it off by 5 %."""
    x = torch.zeros(n, V, device="cuda")
    ids = torch.arange(n, device="cuda") * 3 % V
    logp = -torch.log(torch.tensor(float(V), dtype=torch.float64, device="cuda"))
    gap = 10.0 ** -(1 + torch.arange(n, device="cuda", dtype=torch.float64) % 5)
    ref = (logp + gap).float()
    A = torch.zeros(n, device="cuda")
    xe = x.double().requires_grad_()
    le, _ = policy_exact(xe, ids, None, A.double(), None, ref, (0.2, 0.2), 0.05, None)
    want, = torch.autograd.grad(le, xe)
    lx = x.requires_grad_()
    loss, _ = ab.policy_loss(lx, ids, None, A, ref_logp=ref, kl=0.05)
    two, = torch.autograd.grad(loss, lx)
    one = ab.policy_loss_grad(x.detach(), ids, None, A, ref_logp=ref, kl=0.05)[2]
    for got in (one, two):
        assert bool(((got.double() - want).abs() <= 1e-6 * want.abs()).all()), float(((got.double() - want).abs() / want.abs()).max())


def test_policy_loss_of_no_tokens():
    x, ids, old, A, mask, ref = policy_inputs(9, 1000, "fp16")
    x[2], ids[3], old[4], A[5], ref[6] = float("nan"), -100, float("nan"), float("inf"), float("nan")
    nobody = torch.zeros_like(mask)
    lx = x.requires_grad_()
    loss, logp = ab.policy_loss(lx, ids, old, A, mask=nobody, ref_logp=ref, kl=0.1)
    assert float(loss) == 0 and bool((logp == 0).all()) and float(torch.autograd.grad(loss, lx)[0].abs().max()) == 0
    loss, logp, dx = ab.policy_loss_grad(lx, ids, old, A, mask=nobody, ref_logp=ref, kl=0.1)
    assert float(loss) == 0 and bool((dx == 0).all()) and _lib.device_status() == 0
    loss, logp, dx = ab.policy_loss_grad(x[:0], ids[:0], old[:0], A[:0])
    assert float(loss) == 0 and dx.shape == (0, 1000)


def test_policy_loss_of_broadcast_advantages():
    """One advantage per answer, as group-normalised rewards are."""
    x, ids, old, _, mask, _ = policy_inputs(30, 999, "bf16")
    A = torch.tensor([[1.0], [-0.5], [0.25]], device="cuda")
    cube = lambda t: t.view(3, 10, *t.shape[1:])  # noqa: E731
    loss, logp, dx = ab.policy_loss_grad(cube(x), cube(ids), cube(old), A, mask=cube(mask))
    loss2, logp2, dx2 = ab.policy_loss_grad(x, ids, old, A.expand(3, 10).reshape(-1), mask=mask)
    assert torch.equal(loss, loss2) and torch.equal(logp.view(-1), logp2) and torch.equal(dx.view_as(dx2), dx2)


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("P,T,V,smoothing", [(1, 1, 100, 0.0), (2, 37, 65536, 0.0), (3, 20, 1001, 0.1), (5, 9, 50277, 0.0)])
def test_preference_loss_and_its_gradient(P, T, V, smoothing, dtype):
    x, ids, g = logit_inputs(2 * P * T, V, dtype)
    x, ids = x.view(2 * P, T, V), ids.view(2 * P, T)
    n = torch.randint(1, T + 1, (2 * P,), device="cuda", generator=g)
    mask = torch.arange(T, device="cuda")[None] < n[:, None]
    if P > 2:
        mask[1] = False                                                 # an answer without tokens
    scale = 4096.0 if dtype == "fp16" else 1.0
    ref = (logp_exact(x.double(), ids) * mask).sum(-1).float() + 3 * torch.randn(2 * P, device="cuda", generator=g)
    xe = x.double().requires_grad_()
    se = (logp_exact(xe, ids) * mask).sum(-1)
    d = se - ref.double()
    m = 0.1 * (d[:P] - d[P:])
    le = (torch.nn.functional.softplus(-m) * (1 - smoothing) + torch.nn.functional.softplus(m) * smoothing).mean()
    want, = torch.autograd.grad(le * scale, xe)
    lx = x.detach().requires_grad_()
    loss, sums = ab.preference_loss(lx, ids, ref, mask=mask, beta=0.1, label_smoothing=smoothing)
    dx, = torch.autograd.grad(loss * scale, lx)
    assert abs(float(loss) - float(le)) <= F32 * abs(float(le))
    close(sums, se.detach(), "sums")
    close(dx, want, "dlogits")
    assert bool((dx[~mask] == 0).all())


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("n,V", [(160, 9001), (149, 16384), (150, 70001), (333, 57352)])
def test_policy_loss_of_many_long_rows(n, V, dtype):
    """At least a row per SM: the ring of copies, rows that fit it and rows that do not, masked ones among them."""
    x, ids, old, A, mask, ref = policy_inputs(n, V, dtype)
    scale = 65536.0 if dtype == "fp16" else 1.0
    more = {"mask": mask, "ref_logp": ref, "clip": (0.1, 0.3), "kl": 0.05, "denom": None}
    x[~mask] = float("nan")
    xe = torch.where(mask[:, None], x, torch.zeros_like(x)).double().requires_grad_()
    le, logpe = policy_exact(xe, ids, old, A.double(), **more)
    want, = torch.autograd.grad(le * scale, xe)
    loss, logp, dx = ab.policy_loss_grad(x, ids, old, A, scale=scale, **more)
    assert abs(float(loss) - float(le)) <= F32 * (float(A.abs().max()) * 3 + 1)
    close(logp, logpe.detach(), "logp")
    close(dx, want, "dlogits")
    here = x.clone()
    again = ab.policy_loss_grad(here, ids, old, A, scale=scale, out=here, **more)
    assert torch.equal(again[0], loss) and torch.equal(again[1], logp) and torch.equal(here, dx)
    lx = x.requires_grad_()
    loss2, logp2 = ab.policy_loss(lx, ids, old, A, **more)
    dx2, = torch.autograd.grad(loss2 * scale, lx)
    assert torch.equal(logp2, logp)
    close(dx2, want, "dlogits, two passes")
    assert _lib.device_status() == 0


def test_losses_of_next_tokens_copy_their_logits_once():
    """logits[:, :-1] of several sequences has no one stride between rows: it is copied, and the copy is what the backward pass reads."""
    x, ids, g = logit_inputs(2 * 33, 60000, "fp32")
    cube, ids = x.view(2, 33, 60000), ids.view(2, 33)
    A = torch.randn(2, 32, device="cuda", generator=g)
    size = 2 * 32 * 60000 * 4
    for f in (lambda t: ab.token_logp(t, ids[:, 1:]).sum(), lambda t: ab.policy_loss(t, ids[:, 1:], None, A)[0], lambda t: ab.preference_loss(t, ids[:, 1:], A[:, 0])[0]):
        leaf = cube.detach().requires_grad_()
        part = leaf[:, :-1]
        loss = f(part)
        dense = part.detach().contiguous().requires_grad_()
        want, = torch.autograd.grad(f(dense), dense)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        got, = torch.autograd.grad(loss, part)
        assert torch.cuda.max_memory_allocated() - before < 1.5 * size      # the gradient, and no second copy
        assert torch.equal(got, want)


def test_layer_norm_of_rows_with_two_strides_copies_them_once():
    x, w, b = norm_inputs(2 * 1025, 4096, "fp32")
    leaf = x.view(2, 1025, 4096).requires_grad_()
    part = leaf[:, 1:]
    y = ab.layer_norm(part, w, b)
    dy = torch.randn_like(y)
    dense = part.detach().contiguous().requires_grad_()
    want, = torch.autograd.grad(ab.layer_norm(dense, w, b), dense, dy)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got, = torch.autograd.grad(y, part, dy)
    assert torch.cuda.max_memory_allocated() - before < 1.5 * 2 * 1024 * 4096 * 4
    assert torch.equal(got, want) and torch.equal(y, ab.layer_norm(dense, w, b))


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("V", [16385, 16391, 32771, 7 * 16384 - 3, 7 * 16384 + 5, 8 * 16384 - 7, 57341, 57347])
def test_policy_loss_over_the_ends_of_long_rows(V, dtype):
    """Rows just beyond what clusters take, and around the ring's seven chunks (16384 values of two bytes each, 8192 of four), on every address that their type allows; the id and a
    value that outweighs the rest stand at the ends in turn, where a row's first and last pieces are not copied. A sum of exponentials good to 2^-22 each: its logarithm is
    off by 2^-21, and a log-probability of up to 30 is rounded by 2^-20 more at most."""
    n = 152
    x, ids, old, A, mask, ref = policy_inputs(n, V, dtype, seed=V)
    ends = torch.tensor([0, 1, V - 2, V - 1], device="cuda")
    rows = torch.arange(n, device="cuda")
    top, ids = ends[rows % 4], ends[rows // 4 % 4]
    x[rows, top] = 14.0
    mask[rows[::11]] = False
    logp = logp_exact(x.double(), ids)
    old, ref = (logp + 0.05 * old.sin()).float(), (logp + 0.3 * ref.cos()).float()
    scale = 65536.0 if dtype == "fp16" else 1.0
    more = {"mask": mask, "ref_logp": ref, "clip": (0.1, 0.3), "kl": 0.05, "denom": None}
    xe = x.double().requires_grad_()
    le, logpe = policy_exact(xe, ids, old, A.double(), **more)
    want, = torch.autograd.grad(le * scale, xe)
    x[~mask] = float("nan")
    here = x.clone()
    lx = x.requires_grad_()
    loss, logp = ab.policy_loss(lx, ids, old, A, **more)
    two, = torch.autograd.grad(loss * scale, lx)
    one = ab.policy_loss_grad(x.detach(), ids, old, A, scale=scale, **more)
    place = ab.policy_loss_grad(here, ids, old, A, scale=scale, out=here, **more)
    for a, b, g in ((loss, logp, two), one, place):
        assert abs(float(a) - float(le)) <= F32 * (float(A.abs().max()) * 3 + 1)
        assert float((b.detach().double() - logpe.detach()).abs().max()) <= 2.0 ** -21 + 2.0 ** -20
        close(g, want, "dlogits")
        # the ids' own values, each for itself: coefficient (1 - p), where p is off by its exponential's 2^-22, the sum's as much and, for logits of 14, 2.7e-7 of log2(e)'s own rounding
        most = (1.1 * float(A.abs().max()) + 0.1) * scale / float(mask.sum())
        own = want[rows, ids]
        assert bool(((g.double()[rows, ids] - own).abs() <= torch.finfo(g.dtype).eps / 2 * own.abs() + 2.0 ** -20 * most + 2.0 ** -25).all())
    assert _lib.device_status() == 0


def test_preference_loss_of_no_steps():
    x, ids = torch.zeros(2, 0, 50, device="cuda"), torch.zeros(2, 0, dtype=torch.int64, device="cuda")
    lx = x.requires_grad_()
    loss, sums = ab.preference_loss(lx, ids, torch.tensor([1.0, -2.0], device="cuda"), beta=0.5)
    assert abs(float(loss) - float(torch.nn.functional.softplus(torch.tensor(1.5)))) < 1e-6 and float(sums.abs().sum()) == 0
    assert torch.autograd.grad(loss, lx)[0].shape == (2, 0, 50)


# ------------------------------------------------------------------------------------------------------------------
# streams, graphs, and all of them together
# ------------------------------------------------------------------------------------------------------------------
def small_step(p, ids, mask, old, A):
    """A block without its adapters, the head and a loss, with this package's operators; p: fp32 masters, used in bf16."""
    q = {k: t.bfloat16() for k, t in p.items()}
    B, T = ids.shape
    D = q["emb"].shape[1]
    H = D // 64
    x = ab.layer_norm(q["emb"][ids], q["ln1_w"], q["ln1_b"])
    r, w, k, v = ((x @ q[n]) for n in ("r", "w", "k", "v"))
    w = -torch.nn.functional.softplus(-w) - 0.5
    kk = torch.nn.functional.normalize(k.view(B, T, H, 64), dim=-1).view(B, T, D)
    y, _ = ab.RWKV7_TRAIN_OP(p["state"].expand(B, -1, -1, -1), r, w, k, v, -kk, kk * torch.sigmoid(x))
    y = ab.layer_norm(y, q["lnx_w"], q["lnx_b"], eps=64e-5, groups=H)
    x = ab.layer_norm(q["emb"][ids] + y @ q["o"], q["lno_w"], q["lno_b"])
    return ab.policy_loss(x @ q["head"], ids.roll(-1, 1), old, A, mask=mask)[0]


def small_step_exact(p, ids, mask, old, A):
    B, T = ids.shape
    D = p["emb"].shape[1]
    H = D // 64
    x = norm_exact(p["emb"][ids], p["ln1_w"], p["ln1_b"], 1e-5, 1)
    r, w, k, v = ((x @ p[n]) for n in ("r", "w", "k", "v"))
    w = -torch.nn.functional.softplus(-w) - 0.5
    kk = torch.nn.functional.normalize(k.view(B, T, H, 64), dim=-1).view(B, T, D)
    y, _ = wkv_exact(p["state"].expand(B, -1, -1, -1), (r, w, k, v, -kk, kk * torch.sigmoid(x)))
    y = norm_exact(y, p["lnx_w"], p["lnx_b"], 64e-5, H)
    x = norm_exact(p["emb"][ids] + y @ p["o"], p["lno_w"], p["lno_b"], 1e-5, 1)
    return policy_exact(x @ p["head"], ids.roll(-1, 1), old, A.double(), mask, None, (0.2, 0.2), 0.0, None)[0]


def small_problem():
    g = torch.Generator(device="cuda").manual_seed(5)
    n = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    D, V, B, T = 128, 500, 2, 21
    p = {"emb": n(V, D), "state": 0.1 * n(1, D // 64, 64, 64), "head": n(D, V) / D ** 0.5}
    for m in "rwkvo":
        p[m] = n(D, D) / D ** 0.5
    for m in ("ln1", "lnx", "lno"):
        p[m + "_w"], p[m + "_b"] = 1 + 0.1 * n(D), 0.1 * n(D)
    p = {k: t.bfloat16().float().requires_grad_() for k, t in p.items()}
    ids = torch.randint(V, (B, T), device="cuda", generator=g)
    mask = torch.arange(T, device="cuda")[None] < torch.tensor([[T - 1], [9]], device="cuda")
    A = n(B, 1)
    return p, ids, mask, A


def test_a_training_step_of_all_operators_together():
    """Gradients of a small network against those of the same formulas in 64 bits. Between the operators activations and gradients are rounded to bf16
    some twelve times on the longest way (2^-9 of each value on average): 12^0.5 * 2^-9 = 0.7 %, and where they are differences of larger ones up
    to a few times that, so 4 % of the 2-norm."""
    p, ids, mask, A = small_problem()
    old = None
    loss = small_step(p, ids, mask, old, A)
    got = torch.autograd.grad(loss, list(p.values()))
    e = {k: t.detach().double().requires_grad_() for k, t in p.items()}
    le = small_step_exact(e, ids, mask, old, A)
    want = torch.autograd.grad(le, list(e.values()))
    assert abs(float(loss) - float(le)) <= 0.01 * float(A.abs().max())
    for name, a, b in zip(p, got, want):
        assert float((a.double() - b).norm()) <= 0.04 * float(b.norm()), (name, float((a.double() - b).norm() / b.norm()))


def test_on_another_stream_and_in_captured_graphs():
    p, ids, mask, A = small_problem()

    def step():
        # leaves of this pass alone: torch ties a leaf to the stream of its first use, which a capture elsewhere may not wait for
        q = {k: t.detach().requires_grad_() for k, t in p.items()}
        loss = small_step(q, ids, mask, None, A)
        return (loss.detach(),) + torch.autograd.grad(loss, list(q.values()))
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
        step()
    torch.cuda.current_stream().wait_stream(side)
    index_add = {"emb"}     # torch's own gradient of an index uses atomics
    same = lambda a, b: all(torch.equal(x, y) for n, x, y in zip(("loss", *p), a, b) if n not in index_add)  # noqa: E731
    assert same(got, want)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for _ in range(2):
        for g, out in graphs:
            for t in out:
                t.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert same(out, want)


def test_entries_take_a_state_in_place_and_refuse_bad_pointers():
    state, xs, _, _ = wkv_inputs(1, 9, 1, "fp16")
    y, out = ab.RWKV7_TRAIN_OP(state, *xs)
    s = _lib.Wkv7Seq(_lib.DT_F16, 1, 9, 1)
    for i, x in enumerate(xs):
        s.x[i], s.batch_stride[i], s.step_stride[i] = x.data_ptr(), x.stride(0), x.stride(1)
    here, y2 = state.clone(), torch.empty_like(y)
    s.state = here.data_ptr()
    st = torch.cuda.current_stream().cuda_stream
    assert _lib.lib.ab_wkv7_seq_fwd(C.byref(s), y2.data_ptr(), here.data_ptr(), st) == 0
    assert torch.equal(y2, y) and torch.equal(here, out)
    assert _lib.lib.ab_wkv7_seq_fwd(C.byref(s), y2.data_ptr() + 2, here.data_ptr(), st) == -1 and b"boundary" in _lib.lib.ab_last_error()


@pytest.mark.parametrize("n,V,denom", [(37, 500, 0.0), (37, 5000, 3.0), (160, 20011, 3.0), (16400, 64, 0.0)])
def test_policy_entries_keep_to_the_scratch_that_the_header_names(n, V, denom):
    x, ids, old, A, mask, ref = policy_inputs(n, V, "fp16")
    t = _lib.LogitRows(_lib.DT_F16, V, n, V, x.data_ptr(), ids.data_ptr(), mask.data_ptr())
    p = _lib.Policy(old.data_ptr(), A.data_ptr(), ref.data_ptr(), 0.2, 0.2, 0.05, denom)
    loss, logp, stats, g, dx = (torch.empty(s, device="cuda") for s in (2, n, 2 * n, n, 0))
    dx = torch.empty_like(x)
    st = torch.cuda.current_stream().cuda_stream
    for size, call in ((2 * n + 1, lambda s: _lib.lib.ab_policy_loss_fwd(C.byref(t), C.byref(p), loss.data_ptr(), logp.data_ptr(), stats.data_ptr(), g.data_ptr(), s, st)),
                       (n + 1, lambda s: _lib.lib.ab_policy_loss_grad(C.byref(t), C.byref(p), 1.0, loss.data_ptr() + 4, logp.data_ptr(), dx.data_ptr(), s, st))):
        scratch = torch.full((size + 64,), 7.25, dtype=torch.float64, device="cuda")
        assert call(scratch.data_ptr()) == 0
        assert bool((scratch[size:] == 7.25).all())
    want, wlogp, wdx = ab.policy_loss_grad(x, ids, old, A, mask=mask, ref_logp=ref, kl=0.05, denom=denom or None)
    assert float(loss[0]) == float(want) and float(loss[1]) == float(want) and torch.equal(logp, wlogp) and torch.equal(dx, wdx)


def test_what_cannot_be_right_is_refused():
    x, ids, old, A, mask, ref = policy_inputs(6, 500, "fp16")
    buf = torch.empty(6 * 500 + 8, dtype=torch.float16, device="cuda")
    with pytest.raises(RuntimeError):           # out lies across the logits
        ab.policy_loss_grad(buf[:3000].view(6, 500), ids, old, A, out=buf[8:].view(6, 500))
    for bad in (x[:, ::2], x.float(), x[:5]):
        with pytest.raises(RuntimeError):
            ab.policy_loss_grad(x, ids, old, A, out=bad)
    wide = buf[:3000].view(6, 500)[:, :400]
    with pytest.raises(RuntimeError, match="overlaps"):                # out over a part of the rows that lie between padding
        ab.policy_loss_grad(wide, ids % 400, old, A, out=buf[8:2408].view(6, 400))
    for denom in (-1.0, 0.0, float("nan"), 1e-60):                     # (1e-60 is 0 in 32 bits)
        with pytest.raises(RuntimeError):
            ab.policy_loss(x, ids, old, A, denom=denom)
    with pytest.raises(RuntimeError):
        ab.policy_loss(x, ids, old, A, denom=-1.0)
    with pytest.raises(RuntimeError):
        ab.policy_loss(x, ids, old, A, clip=(1.5, 0.2))
    with pytest.raises(RuntimeError):
        ab.policy_loss(x, ids, old, A, mask=mask.float())
    with pytest.raises(RuntimeError):
        ab.policy_loss(x, ids, old.cpu(), A)
    with pytest.raises(RuntimeError):
        ab.token_logp(x, ids[:5])
    with pytest.raises(RuntimeError):
        ab.preference_loss(x.view(3, 2, 500), ids.view(3, 2), old[:3])
    y = torch.zeros(2, 5, 64, device="cuda", dtype=torch.float16)
    for args in ((None, y.float(), y, y, y, y, y), (None, y, y, y, y, y, y[:1]), (torch.zeros(2, 1, 64, 64, device="cuda", dtype=torch.float16), y, y, y, y, y, y),
                 (None, y, y, y, y, y, y, torch.tensor([1, 2], device="cuda")), (None, *(t[..., :63] for t in (y,) * 6))):
        with pytest.raises(RuntimeError):
            ab.RWKV7_TRAIN_OP(*args)
    for args in ((y, y[0, 0, :63]), (y, y[0, 0].float(), y[0, 0]), (y, None, None, 1e-5, 5), (y, y[0, 0].bfloat16())):
        with pytest.raises(RuntimeError):
            ab.layer_norm(*args)


def test_gradients_are_first_order_and_of_what_was_given():
    x, w, b = norm_inputs(4, 256, "fp32")
    lx = x.requires_grad_()
    y = ab.layer_norm(lx, w, b)
    with pytest.raises(RuntimeError, match="again"):
        torch.autograd.grad(y.sum(), lx, create_graph=True)
    lg, ids, g = logit_inputs(4, 300, "fp16")
    lg.requires_grad_()
    z = lg * 1.0
    loss, _ = ab.policy_loss(z, ids, None, torch.ones(4, device="cuda"))
    ab.policy_loss_grad(z, ids, None, torch.ones(4, device="cuda"), out=z.detach())      # the logits are written over: autograd says so
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(loss, lg)


def test_forward_mode_derivatives_are_refused():
    """A tangent is an error, not a derivative of zero; with and without a gradient asked for."""
    import torch.autograd.forward_ad as forward_ad
    x, w, b = norm_inputs(4, 256, "fp32")
    lg, ids, _ = logit_inputs(4, 300, "fp16")
    one, pairs = torch.ones(4, device="cuda"), (lg.view(4, 1, 300), ids.view(4, 1))
    state, xs, _, _ = wkv_inputs(1, 5, 1, "fp16")
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for f in (lambda: ab.layer_norm(dual(x), w, b), lambda: ab.layer_norm(x, dual(w), b), lambda: ab.layer_norm(x, w, dual(b)), lambda: ab.layer_norm(dual(x.requires_grad_())),
                  lambda: ab.token_logp(dual(lg), ids), lambda: ab.policy_loss(dual(lg), ids, None, one), lambda: ab.policy_loss(lg, ids, None, dual(one)),
                  lambda: ab.policy_loss_grad(dual(lg), ids, None, one), lambda: ab.preference_loss(dual(pairs[0]), pairs[1], one),
                  lambda: ab.RWKV7_TRAIN_OP(dual(state), *xs), lambda: ab.RWKV7_TRAIN_OP(state, *xs[:5], dual(xs[5]))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                f()
    ab.layer_norm(x, w, b)


def test_tracing_is_refused_and_slices_are_taken():
    """A trace would hold the outputs' allocation and not the call. (torch.vmap calls the operator slice by slice.)"""
    from torch.fx.experimental.proxy_tensor import make_fx
    x, w, b = norm_inputs(4, 256, "fp32")
    lg, ids, _ = logit_inputs(4, 300, "fp16")
    state, xs, _, _ = wkv_inputs(1, 5, 1, "fp16")
    one = torch.ones(4, device="cuda")
    for f, args in ((lambda t: ab.layer_norm(t, w, b), x), (lambda t: ab.token_logp(t, ids), lg), (lambda t: ab.policy_loss(t, ids, None, one)[0], lg),
                    (lambda t: ab.policy_loss_grad(t, ids, None, one)[2], lg), (lambda t: ab.preference_loss(t.view(4, 1, 300), ids.view(4, 1), one)[0], lg),
                    (lambda t: ab.RWKV7_TRAIN_OP(t, *xs)[0], state)):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            make_fx(f)(args)
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.func.grad(lambda t: f(t).float().sum())(args)
        f(args)
    assert torch.equal(torch.vmap(lambda t: ab.layer_norm(t, w, b))(x), ab.layer_norm(x, w, b))
    # as a compiled program has them
    part = torch.compiler.disable(lambda t: ab.layer_norm(t, w, b))
    assert torch.equal(torch.compile(lambda t: part(t * 2.0) + 1.0, backend="eager")(x), ab.layer_norm(x * 2.0, w, b) + 1.0)


def test_gradients_are_not_written_over_a_leaf_that_wants_one():
    """As torch refuses its own operators in place; outside of a graph, and over logits that are no leaf, it is done."""
    lg, ids, _ = logit_inputs(4, 300, "fp16")
    A = torch.ones(4, device="cuda")
    want = ab.policy_loss_grad(lg, ids, None, A)
    leaf = lg.clone().requires_grad_()
    before = leaf.detach().clone()
    for out in (leaf, leaf.view(4, 300), leaf[:]):
        with pytest.raises(RuntimeError, match="leaf"):
            ab.policy_loss_grad(leaf, ids, None, A, out=out)
        with pytest.raises(RuntimeError, match="leaf"):
            ab.policy_loss_grad(lg, ids, None, A, out=out)
    assert torch.equal(leaf.detach(), before)
    with torch.no_grad():
        assert torch.equal(ab.policy_loss_grad(leaf, ids, None, A, out=leaf)[2], want[2])
    z = lg.clone().requires_grad_() * 1.0
    assert torch.equal(ab.policy_loss_grad(z, ids, None, A, out=z)[2], want[2])


def test_batched_upstream_gradients_are_refused():
    """torch.autograd.grad(is_grads_batched=True) hands wrappers without memory to the backward passes."""
    x, w, b = (t.requires_grad_() for t in norm_inputs(4, 256, "fp32"))
    lg, ids, _ = logit_inputs(4, 300, "fp32")
    lg.requires_grad_()
    state, xs, _, _ = wkv_inputs(1, 5, 1, "fp16")
    state.requires_grad_()
    for y, leaf in ((ab.layer_norm(x, w, b), x), (ab.token_logp(lg, ids), lg), (ab.policy_loss(lg, ids, None, lg.detach()[:, 0])[0], lg), (ab.RWKV7_TRAIN_OP(state, *xs)[1], state)):
        with pytest.raises(RuntimeError, match="cannot be traced or transformed"):
            torch.autograd.grad(y, leaf, torch.ones(2, *y.shape, device="cuda"), is_grads_batched=True, retain_graph=True)
        assert torch.autograd.grad(y, leaf, torch.ones_like(y))[0].shape == leaf.shape


def test_capture_beside_a_living_graph_of_the_same_leaf_is_refused():
    """On the default stream such a graph ties the leaf to that stream, which cannot join a capture; nothing of the process is lost, and without that graph the capture is taken."""
    x = torch.randn(4, 256, device="cuda", requires_grad=True)
    lg, ids, _ = logit_inputs(4, 300, "fp16")
    lg.requires_grad_()
    A = torch.ones(4, device="cuda")
    for leaf, run in ((x, lambda: ab.layer_norm(x).square().sum()), (lg, lambda: ab.token_logp(lg, ids).sum()), (lg, lambda: ab.policy_loss(lg, ids, None, A)[0])):
        leaf.grad = None
        living = run()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with pytest.raises(RuntimeError, match="still lives"):
            with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=s):
                run().backward()
        living.backward()
        want, leaf.grad, living = leaf.grad, None, None
        with torch.cuda.stream(s):
            run().backward()
        leaf.grad = None
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            run().backward()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(leaf.grad, want)


def test_capture_of_some_gradients_beside_a_living_graph_of_another_leaf():
    """Only leaves whose gradient is asked for have to join the capture."""
    x, w, b = (t.requires_grad_() for t in norm_inputs(4, 256, "fp32"))
    living = ab.layer_norm(x.detach(), w, b).square().sum()         # ties weight and bias to the default stream
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        warm, = torch.autograd.grad(ab.layer_norm(x, w, b).square().sum(), x)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        dx, = torch.autograd.grad(ab.layer_norm(x, w, b).square().sum(), x)
    dx.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(dx, warm)
    living.backward()
    assert w.grad is not None and b.grad is not None


def test_under_checkpointing_saved_tensors_on_the_host_and_inference_mode():
    """What programs put around operators: recomputation, saved tensors that come back as other tensors, no autograd at all."""
    from torch.utils.checkpoint import checkpoint
    state, xs, dy, dout = wkv_inputs(2, 35, 2, "bf16", seed=33)
    packed = torch.cat(xs, -1)
    x, w, b = norm_inputs(40, 2304, "bf16")
    lg, ids, _ = logit_inputs(24, 3003, "bf16")
    A = torch.randn(24, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    calls = ((lambda s, p: sum((t.float() * g.float()).sum() for t, g in zip(ab.RWKV7_TRAIN_OP(s, *p.split(128, -1)), (dy, dout))), (state, packed)),
             (lambda x, w, b: ab.layer_norm(x[:, 256:1280], w, b).float().square().sum(), (x, w[:1024].clone(), b[:1024].clone())),
             (lambda t: ab.token_logp(t[:, 3:2003], ids % 2000).square().sum(), (lg,)),
             (lambda t: ab.policy_loss(t.view(2, 12, 3003)[:, :-1], ids.view(2, 12)[:, 1:], None, A.view(2, 12)[:, 1:])[0], (lg,)),
             (lambda t: ab.preference_loss(t.view(2, 12, 3003), ids.view(2, 12), A[:2])[0], (lg,)))
    for f, args in calls:
        def grads(run):
            leaves = [t.detach().clone().requires_grad_() for t in args]
            out = run(leaves)
            return (out.detach(),) + torch.autograd.grad(out, leaves)
        want = grads(lambda leaves: f(*leaves))
        again = grads(lambda leaves: checkpoint(f, *leaves, use_reentrant=False))
        with torch.autograd.graph.save_on_cpu():
            host = grads(lambda leaves: f(*leaves))
        assert all(torch.equal(p, q) for p, q in zip(again, want)) and all(torch.equal(p, q) for p, q in zip(host, want))
        with torch.inference_mode():
            assert torch.equal(f(*[t.clone() for t in args]), want[0])
    with torch.inference_mode():
        here = lg.clone()
        assert torch.equal(ab.policy_loss_grad(here, ids, None, A, out=here)[2], ab.policy_loss_grad(lg, ids, None, A)[2])


def test_two_streams_at_once():
    """Calls that overlap share nothing."""
    p, ids, mask, A = small_problem()
    p2 = {k: t.detach() * 1.25 for k, t in p.items()}

    def step(values):
        q = {k: t.detach().requires_grad_() for k, t in values.items()}
        loss = small_step(q, ids, mask, None, A)
        return (loss.detach(),) + torch.autograd.grad(loss, [t for n, t in q.items() if n != "emb"])
    want = step(p), step(p2)
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, values in enumerate((p, p2)):
            with torch.cuda.stream(streams[i]):
                got[i].append(step(values))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(g, want[i]))
