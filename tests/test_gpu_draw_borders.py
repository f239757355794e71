"""GPU: draws under filters where it is close: a row's own top-k in clusters, uniform numbers and top-p at the borders of the sums.

Every call writes into ids that were set to an impossible one before, so that a row that is not written shows."""
import pytest
import torch

import albatross_b200 as ab

pytestmark = pytest.mark.gpu

NONE = -77
DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
GAP = 2e-9     # of the sum: nearer to a border either neighbour may be drawn


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
    assert int(clear.sum()) >= 0.9 * len(u), int(clear.sum())
    assert not bool((ids == NONE).any()), "ids that were not written"
    bad = (ids != want) & clear
    assert not bool(bad.any()), (int(bad.sum()), u[bad][:5].tolist(), ids[bad][:5].tolist(), want[bad][:5].tolist())
    off = (logp.double() - want_p).abs()[clear]
    assert bool((off <= 2.0 ** -24 * want_p.abs()[clear] + 2.0 ** -19).all()), float(off.max())


def check(x, u, T=1.0, k=0, p=1.0, m=0.0):
    """x [V], drawn from by every number of u, as one batch and in small ones (which are divided among blocks in other ways)."""
    for at in (slice(None), *(slice(i, i + n) for i, n in ((0, 1), (1, 1), (2, 3), (5, 20), (25, 40)))):
        v = u[at]
        out = torch.full((len(v),), NONE, device="cuda")
        ids, logp = ab.sampler_batch(x.expand(len(v), -1), v, temperature=T, top_k=k, top_p=p, min_p=m, out=out)
        hold(x, v, ids[:, 0], logp[:, 0], T, k, p, m)


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
