"""GPU: draws under filters where it is close: a row's own top-k in clusters, uniform numbers and top-p at the borders of the sums.

Every call writes into ids that were set to an impossible one before, so that a row that is not written shows."""
import pytest
import torch

import albatross_b200 as ab

pytestmark = pytest.mark.gpu

NONE = -77
DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
GAP = 1e-9     # of the sum: nearer to a border either neighbour may be drawn (weights are whole multiples of 2^-44)


class Row:
    """One row of logits under filters, by the definition in 64 bits: the values in order and the sums of what is kept."""

    def __init__(self, x, T=1.0, k=0, p=1.0, m=0.0):
        values, self.order = torch.sort(x.double(), descending=True, stable=True)
        self.w = torch.exp((values - values[0]) / T)
        n = k if 0 < k < len(x) else len(x)
        cum = torch.cumsum(self.w[:n], 0)
        if p < 1:
            n = 1 + int((cum[:-1] < p * cum[-1]).sum())
            # (top-p's border is where it should be: not within rounding of a sum)
            assert p == 0 or float((cum - p * cum[-1]).abs().min()) > GAP * float(cum[-1])
        n = max(1, min(n, int((self.w >= m).sum())))
        self.cum = cum[:n]

    def draw(self, u):
        """ids and log-probabilities for uniform numbers [n], and which of them are clear of every border"""
        X = u.double() * self.cum[-1]
        at = torch.searchsorted(self.cum, X, right=True).clamp(max=len(self.cum) - 1)
        before = torch.where(at > 0, self.cum[at - 1], -1.0)
        clear = (X - before > GAP * self.cum[-1]) & (self.cum[at] - X > GAP * self.cum[-1])
        return self.order[at], torch.log(self.w[at] / self.cum[-1]), clear

    def borders(self, count=160, seed=0):
        """uniform numbers next to the borders of `count` ranks, the first and the last ones among them: on both sides, and one step of 2^-24 further"""
        n = len(self.cum)
        g = torch.Generator(device="cuda").manual_seed(seed + n)
        ranks = torch.cat([torch.arange(min(n, 12), device="cuda"), torch.arange(max(0, n - 12), n, device="cuda"), torch.randint(0, n, (count,), device="cuda", generator=g)])
        step = torch.floor(self.cum[ranks] / self.cum[-1] * 2.0 ** 24)
        steps = torch.cat([step - 1, step, step + 1, step + 2, torch.tensor([0.0, 1.0], device="cuda", dtype=torch.float64)])
        return (steps.clamp(0, 2 ** 24 - 1) / 2 ** 24).float()


def hold(x, u, ids, logp, T=1.0, k=0, p=1.0, m=0.0):
    """Log-probabilities: the sum of 32-bit exponentials is off by 2^-19 at most, and the result is rounded to 32 bits."""
    want, want_p, clear = Row(x, T, k, p, m).draw(u)
    assert not bool((ids == NONE).any()), "ids that were not written"
    bad = (ids != want) & clear
    assert not bool(bad.any()), (int(bad.sum()), u[bad][:5].tolist(), ids[bad][:5].tolist(), want[bad][:5].tolist())
    off = (logp.double() - want_p).abs()[clear]
    assert bool((off <= 2.0 ** -24 * want_p.abs()[clear] + 2.0 ** -19).all()), float(off.max())
    return int(clear.sum())


def check(x, u, T=1.0, k=0, p=1.0, m=0.0):
    """x [V], drawn from by every number of u, as one batch and in small ones (which are divided among blocks in other ways)."""
    for at in (slice(None), *(slice(i, i + n) for i, n in ((0, 1), (1, 1), (2, 3), (5, 20), (25, 40)))):
        v = u[at]
        out = torch.full((len(v),), NONE, device="cuda")
        ids, logp = ab.sampler_batch(x.expand(len(v), -1), v, temperature=T, top_k=k, top_p=p, min_p=m, out=out)
        clear = hold(x, v, ids[:, 0], logp[:, 0], T, k, p, m)
        assert len(v) < len(u) or clear >= 0.4 * len(u)


def normal(V, std=1.0, seed=0, dtype="fp32"):
    g = torch.Generator(device="cuda").manual_seed(97 * seed + V)
    return (torch.randn(V, device="cuda", generator=g) * std).to(DT[dtype])


@pytest.mark.parametrize("dtype,V", [("fp32", 65536), ("fp32", 4099), ("fp32", 20011), ("fp16", 70001), ("bf16", 200003), ("fp32", 1 << 18)])
def test_a_top_k_of_each_row_in_clusters(dtype, V):
    """The bound that k of a block's maxima reach, searched in two passes whose words do not meet: the same ids call after call."""
    for n in (1, 2, 9, 18, 37, 75, 160):
        x = torch.stack([normal(V, 1.0 + r % 4, seed=r, dtype=dtype) for r in range(n)])
        u = torch.rand(n, device="cuda", generator=torch.Generator(device="cuda").manual_seed(n))
        ks = [1 + (7 * r) % 75 for r in range(n)]
        k = torch.tensor(ks, device="cuda", dtype=torch.int32)
        first = None
        for _ in range(20):
            out = torch.full((n,), NONE, device="cuda")
            ids, logp = ab.sampler_batch(x, u, top_k=k, out=out)
            if first is None:
                first = ids.clone(), logp.clone()
                for r in range(0, n, 1 + n // 20):
                    if ks[r] > 1:
                        want, _, clear = Row(x[r], k=ks[r]).draw(u[r:r + 1])
                        assert not bool(clear) or int(ids[r]) == int(want)
            assert torch.equal(ids, first[0]) and torch.equal(logp, first[1])


def two_steps_and_a_ramp():
    """Half a bin below the largest value lie 999 others: what they weigh is taken for more than it is."""
    x = torch.full((5000,), -0.0035, dtype=torch.float64)
    x[0] = 0.0
    x[1000:] = torch.linspace(-0.02, -1.0, 4000, dtype=torch.float64)
    return x.float().cuda()


def heavy_values_at_the_border():
    """Two heavy values, the second one at top-p's border: what is kept is more than p of the sum."""
    return torch.cat([torch.zeros(1), torch.full((1,), 0.9).log(), torch.full((1024,), 0.8).log(), torch.full((3000,), -10.0)]).cuda()


def few_large_values(large, equals, seed):
    """A few distinct large values in front of many equals, and a flat tail."""
    g = torch.Generator().manual_seed(seed)
    tail = -1.0 - 0.3 * torch.rand(9000, generator=g)
    return torch.cat([4.0 + 0.004 * torch.arange(large).flip(0).float(), torch.full((equals,), 3.0), tail]).cuda()


@pytest.mark.parametrize("p", [1.0, 0.9, 0.5, 0.0024])
def test_a_draw_from_the_top_and_an_end_far_below(p):
    """The draw's values and those at top-p's end in two lists, the first of which begins with the largest value: every uniform number gets an id,
    and the right one."""
    even = (torch.arange(512, device="cuda") + 0.5) / 512
    for x in (two_steps_and_a_ramp(), heavy_values_at_the_border(), few_large_values(1, 900, 0), few_large_values(2, 1000, 1),
              few_large_values(40, 1023, 2), few_large_values(3, 1500, 3)):
        row = Row(x, p=p)
        check(x, torch.cat([row.borders(), even]), p=p)
        check(x, torch.cat([row.borders(), even]) * 2.0 ** -6, p=p)


def test_uniform_numbers_between_a_list_and_its_estimate():
    x = two_steps_and_a_ramp()
    check(x, 0.3160 + 0.0020 * torch.rand(300, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)), p=0.9)
    check(heavy_values_at_the_border(), 0.30 + 0.2 * torch.rand(300, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)), p=0.0024)


FILTERS = [{}, {"p": 0.9}, {"p": 0.3}, {"p": 0.999}, {"p": 0.9, "m": 0.05}, {"m": 0.01}, {"m": 1e-5}, {"k": 50}, {"k": 50, "p": 0.8},
           {"k": 500, "p": 0.95}, {"k": 3000, "p": 0.9}, {"T": 0.4, "p": 0.95}, {"T": 2.5, "p": 0.7}]


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("f", FILTERS, ids=lambda f: "_".join(f"{a}{b}" for a, b in f.items()) or "all")
def test_uniform_numbers_at_borders(f, dtype):
    """On both sides of the borders between one id and the next, in every kernel and however the values lie."""
    for x in (normal(5003, 0.1, 1, dtype), normal(5003, 3.0, 2, dtype), normal(65536, 0.02, 3, dtype), normal(65536, 1.5, 4, dtype), normal(70001, 4.0, 5, dtype),
              normal(65536, 1.0, 6, "bf16").to(DT[dtype]), few_large_values(40, 700, 7).to(DT[dtype])):
        check(x, Row(x, **f).borders(60), **f)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_uniform_numbers_on_borders(dtype):
    """Weights of 1, 1/2, 1/4 ..: sums are exact, a uniform number that meets one belongs to the next id, and top-p that meets one keeps nothing
    behind it."""
    x = (torch.arange(3000, device="cuda") % 9).to(DT[dtype]) * -1.0
    T = 1.0 / torch.log(torch.tensor(2.0, dtype=torch.float64)).item()
    for p in (1.0, 0.5, 0.25):
        values, order = torch.sort(x.double(), descending=True, stable=True)
        cum = torch.cumsum(torch.exp2(values), 0)
        if p < 1:
            cum = cum[:1 + int((cum[:-1] < p * cum[-1]).sum())]
        u = torch.floor(cum[::7] / cum[-1] * 2.0 ** 24) / 2.0 ** 24
        for v in (u.float(), (torch.arange(256, device="cuda") / 256).float()):
            X = v.double() * cum[-1]
            want = order[torch.searchsorted(cum, X, right=True).clamp(max=len(cum) - 1)]
            out = torch.full((len(v),), NONE, device="cuda")
            ids, _ = ab.sampler_batch(x.expand(len(v), -1), v, temperature=T, top_p=p, out=out)
            assert torch.equal(ids[:, 0], want)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_top_p_at_borders(dtype):
    """The sum up to a rank and a little less or more as top-p: what is kept ends with that rank, or with the next one."""
    for x in (normal(5003, 0.5, 11, dtype), normal(65536, 1.5, 12, dtype), normal(70001, 3.0, 13, dtype)):
        whole = Row(x)
        last = torch.full((4,), 1 - 2.0 ** -24, device="cuda")
        for rank in (0, 1, 2, 50, 700, 3000):
            for off in (-1e-7, -1e-8, 1e-8, 1e-7):
                p = float(whole.cum[rank] / whole.cum[-1]) + off
                if float((whole.cum - p * whole.cum[-1]).abs().min()) > GAP * float(whole.cum[-1]) and p < 1:
                    check(x, torch.cat([last, Row(x, p=p).borders(4)]), p=p)


def test_draws_carry_no_gradient():
    """Logits that require a gradient are drawn from; what comes out has none, as the function says, and the gradient by token_logp is not touched."""
    x = normal(2000, 1.0, 20).expand(4, -1).clone().requires_grad_()
    u = torch.linspace(0.1, 0.9, 4, device="cuda")
    ids, logp = ab.sampler_batch(x, u, top_p=0.9)
    assert not ids.requires_grad and not logp.requires_grad and "no gradients" in ab.sampler_batch.__doc__
    with torch.no_grad():
        again, again_p = ab.sampler_batch(x, u, top_p=0.9)
    assert torch.equal(ids, again) and torch.equal(logp, again_p)
    ab.token_logp(x, ids[:, 0]).sum().backward()
    assert bool(x.grad.isfinite().all()) and float(x.grad.abs().max()) > 0


@pytest.mark.parametrize("dtype", ["fp16", "fp32"])
def test_ids_among_the_values_of_an_input_are_refused(dtype):
    """Also where the logits' rows lie apart; between rows there is room for ids."""
    size = DT[dtype].itemsize
    big = torch.zeros(6, 1024, device="cuda", dtype=DT[dtype])
    x, u = big[:, 8:1000], torch.full((6,), 0.5, device="cuda")
    x.normal_()
    want = ab.sampler_batch(x, u, top_p=0.9)[0]
    memory = big.view(torch.int64).view(-1)
    row = 1024 * size // 8
    for at in (size, row - 1, 3 * row + 10, 5 * row + size - 5, 1000 * size // 8 - 6):
        with pytest.raises(RuntimeError, match="among the values"):
            ab.sampler_batch(x, u, top_p=0.9, out=memory[at:at + 6])
    assert torch.equal(ab.sampler_batch(x, u, top_p=0.9)[0], want)
    gap = memory[row + 1000 * size // 8:][:6]
    assert torch.equal(ab.sampler_batch(x, u, top_p=0.9, out=gap)[0], want)
    several = torch.zeros(12, device="cuda", dtype=torch.int64)
    numbers = several.view(torch.float32)
    for name, v in (("temperature", 1.0), ("top_p", 0.9), ("min_p", 0.1)):
        numbers.fill_(v)
        for at in (0, 2, 5):
            with pytest.raises(RuntimeError, match="among the values"):
                ab.sampler_batch(x, u, out=several[at // 2:at // 2 + 6], **{name: numbers[at:at + 6]})
    with pytest.raises(RuntimeError, match="among the values"):
        ab.sampler_batch(x, numbers.fill_(0.5)[:6], out=several[:6])
    with pytest.raises(RuntimeError, match="among the values"):
        ab.sampler_batch(x, u, out=several[:6], top_k=several.view(torch.int32)[:6])
    assert torch.equal(ab.sampler_batch(x, u, top_p=0.9, out=several[:6])[0], want)


def test_a_top_k_of_any_whole_type():
    """In 32 bits as it was given, or filtering nothing where those do not hold it; what would be cut to its lowest bits is refused."""
    x, u = normal(1000, 1.0, 21).expand(3, -1), torch.full((3,), 0.999, device="cuda")
    want = ab.sampler_batch(x, u, top_k=5)[0]
    for dtype in (torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64):
        assert torch.equal(ab.sampler_batch(x, u, top_k=torch.full((3,), 5, device="cuda", dtype=dtype))[0], want)
    with pytest.raises(RuntimeError, match="top_k"):
        ab.sampler_batch(x, u, top_k=torch.full((3,), 2 ** 32 + 5, dtype=torch.uint64).cuda())


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("f", [{}, {"p": 0.95}, {"p": 0.9995}], ids=str)
def test_16_bit_values_whose_differences_take_more_than_24(f, dtype):
    """A largest value of 513 (512 in bf16) and many near 2^-15: each difference is rounded the same way, and weighs that much less or more under a large temperature."""
    x = torch.full((1 << 18,), 2.0 ** -15 * 0.99, device="cuda")
    x[:400] = -torch.linspace(1.0, 200.0, 400, device="cuda")
    x[70000] = 513.0
    x = x.to(DT[dtype])
    f = {"T": 51.3, **f}
    check(x, torch.cat([Row(x, **f).borders(60), torch.linspace(0, 0.09, 40, device="cuda")]), **f)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("f", [{}, {"p": 0.9}, {"p": 0.3}, {"p": 0.99, "T": 2.0}], ids=lambda f: "_".join(f"{a}{b}" for a, b in f.items()) or "all")
def test_uniform_numbers_at_growing_distances_from_borders(f, dtype):
    """From 2^-24 to 2^-13 off: where sums of 32-bit exponentials begin to be trusted."""
    for x in (normal(70001, 0.1, 31, dtype), normal(70001, 1.0, 32, dtype), normal(200003, 2.5, 33, dtype)):
        row = Row(x, **f)
        u = row.borders(40)
        off = torch.tensor([s * 2.0 ** j for j in range(12) for s in (-1, 1)], device="cuda") * 2.0 ** -24
        check(x, (u[:, None] + off).clamp(0, 1 - 2.0 ** -24).view(-1), **f)
