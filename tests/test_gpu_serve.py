"""GPU: the draw of ids under filters and the products with 4-bit weights against plain implementations in 64 bits.

Ids are whole numbers: they have to be those of the definition in 64 bits. A uniform number or a top-p that comes within rounding of a border could give
either neighbour; with numbers of 24 random bits that does not happen at these sizes (a border within 1e-9 of the sum, per row, has a chance of 1e-5 where a
row keeps some 10^4 values)."""
import ctypes as C

import numpy as np
import pytest
import torch

import albatross_b200 as ab
from albatross_b200 import _lib

pytestmark = pytest.mark.gpu

DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------------------------
# the draw
# ------------------------------------------------------------------------------------------------------------------
def drawn(x, u, T, k, p, m):
    """One row by the definition: id and log-probability."""
    if np.isnan(x).any() or not (x > -np.inf).any():
        return -1, np.nan
    top = x.max()
    if not T > 0 or k == 1:
        return int(np.argmax(x)), 0.0
    with np.errstate(invalid="ignore", over="ignore"):
        z = np.where(x == top, 0.0, (x - top) / T)
    w = np.exp(z)
    order = np.argsort(-x, kind="stable")
    if 0 < k < len(x):
        order = order[:k]
    if p < 1:
        cum = np.cumsum(w[order])
        order = order[:1 + int(np.count_nonzero(cum[:-1] < p * cum[-1]))]
    kept = np.concatenate([order[:1], order[1:][w[order[1:]] >= m]]) if m > 0 else order     # (a NaN filters nothing)
    cum = np.cumsum(w[kept])
    i = min(int(np.searchsorted(cum, u * cum[-1], side="right")), len(kept) - 1)
    return int(kept[i]), float(np.log(w[kept[i]]) - np.log(cum[-1])) if w[kept[i]] > 0 else -np.inf


def each(v, rows):
    return v.double().cpu().tolist() if torch.is_tensor(v) else [v] * rows


def check(logits, u, T=1.0, k=0, p=1.0, m=0.0, **more):
    ids, logp = ab.sampler_batch(logits, u, temperature=T, top_k=k, top_p=p, min_p=m, **more)
    rows = logits.reshape(-1, logits.shape[-1])
    n = rows.shape[0]
    assert ids.shape == logp.shape == (*logits.shape[:-1], 1) and ids.dtype == torch.int64 and logp.dtype == torch.float32
    xs, us, got, got_p = rows.double().cpu().numpy(), u.reshape(-1).double().cpu().tolist(), ids.reshape(-1).tolist(), logp.reshape(-1).double().cpu().tolist()
    for r, (x, v, *f) in enumerate(zip(xs, us, each(T, n), each(k, n), each(p, n), each(m, n))):
        want, want_p = drawn(x, v, f[0], int(f[1]), f[2], f[3])
        assert got[r] == want, (r, v, f, got[r], want)
        # computed in 64 bits but for the sum, then rounded to 32. The sum is one of 32-bit exponentials where top_k does not limit it: 2^-22 for the exponential,
        # and as much again for the additions; in 32-bit logits 2^-24 z ln 2 for the rounding of a difference of z bits, below 2^-20 for z up to 22
        off, sum_off = abs(got_p[r] - want_p), 2.0 ** -21 if logits.dtype != torch.float32 else 2.0 ** -19
        assert (np.isnan(want_p) and np.isnan(got_p[r])) or off <= 2.0 ** -24 * abs(want_p) + sum_off, (r, got_p[r], want_p)
    return ids, logp


def rows_of(n, V, dtype, seed=0, spread=(1.0, 4.0)):
    g = torch.Generator(device="cuda").manual_seed(7919 * seed + 31 * n + V)
    sharp = torch.rand(n, 1, device="cuda", generator=g) * (spread[1] - spread[0]) + spread[0]
    return (torch.randn(n, V, device="cuda", generator=g) * sharp).to(DT[dtype]), torch.rand(n, device="cuda", generator=g)


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("n,V", [(3, 1), (4, 2), (5, 33), (9, 1000), (7, 4099), (5, 32003), (3, 65536), (2, 65537)])
def test_draw_from_the_whole_distribution(n, V, dtype):
    check(*rows_of(n, V, dtype))


FILTERS = [{"k": 1}, {"k": 2}, {"k": 50}, {"k": 3000}, {"p": 0.7}, {"p": 0.05}, {"p": 0.999}, {"m": 0.05}, {"m": 1e-4}, {"T": 0.3}, {"T": 3.0}, {"T": 0.0},
           {"k": 50, "p": 0.9}, {"k": 200, "p": 0.8, "m": 0.02, "T": 0.8}, {"p": 0.95, "m": 0.01, "T": 1.4}, {"k": 7, "m": 0.5}, {"p": 0.0}, {"m": 1.0}, {"m": 2.0}]


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("f", FILTERS, ids=lambda f: "_".join(f"{a}{b}" for a, b in f.items()))
def test_filters(f, dtype):
    check(*rows_of(6, 5003, dtype, seed=3), **f)
    check(*rows_of(3, 50277, dtype, seed=4, spread=(0.2, 3.0)), **f)


LONG = [{}, {"p": 0.9}, {"p": 0.9999}, {"m": 0.001}, {"k": 5000}, {"k": 700, "p": 0.9}, {"T": 3.0, "p": 0.5}, {"T": 0.05}, {"p": 0.7, "m": 0.2}, {"p": 0.95, "m": 1e-4}, {"k": 400, "m": 0.3}]


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("f", LONG, ids=lambda f: "_".join(f"{a}{b}" for a, b in f.items()) or "all")
def test_filters_of_long_and_even_rows(f, dtype):
    """Rows that several blocks share, and rows so even that no small part of them has most of the weight."""
    check(*rows_of(5, 70001, dtype, seed=30, spread=(0.05, 3.0)), **f)
    check(*rows_of(2, 200003, dtype, seed=31, spread=(0.5, 4.0)), **f)
    check(*rows_of(40, 65536, dtype, seed=32, spread=(0.05, 1.5)), **f)


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
def test_k_and_rows_on_either_side_of_the_lines_between_kernels(dtype):
    """k around those that are sorted, streamed and counted, given once and for each row; batches that a row's blocks are counted by."""
    x, u = rows_of(3, 9001, dtype, seed=40, spread=(0.2, 1.0))
    many, v = rows_of(150, 1003, dtype, seed=41, spread=(0.2, 1.0))
    for k in (75, 76, 150, 151, 255, 256, 257, 300, 301, 320, 321, 599, 600, 601):
        check(x, u, 1.0, k, 0.98)
        check(x, u, 1.0, torch.full((3,), k, device="cuda"), 1.0, 1e-3)
        check(many, v, 0.7, k)
    for n in (15, 16, 17, 18, 19, 33, 37, 38, 74, 75):
        x, u = rows_of(n, 33001, dtype, seed=42)
        check(x, u, 1.0, torch.full((n,), 40, device="cuda"), 0.95)
        check(x, u, 1.0, 0, 0.9)


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
def test_each_row_with_filters_of_its_own(dtype):
    n = 200   # more rows than SMs
    x, u = rows_of(n, 2051, dtype, seed=5)
    g = torch.Generator(device="cuda").manual_seed(6)
    r = lambda: torch.rand(n, device="cuda", generator=g)  # noqa: E731
    T = torch.where(r() < 0.2, torch.zeros_like(u), r() * 2)
    k = torch.where(r() < 0.5, (r() * 300).int(), torch.zeros_like(u, dtype=torch.int32))
    p, m = torch.where(r() < 0.5, r(), torch.ones_like(u)), torch.where(r() < 0.4, r() * 0.3, torch.zeros_like(u))
    check(x, u, T, k, p, m)
    check(x.view(4, 50, 2051), u.view(4, 50), T, k.long(), p.double(), m)   # other shapes and types of the same


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("f", [{}, {"k": 5}, {"k": 700}, {"p": 0.5}, {"k": 900, "p": 0.5}, {"p": 0.9, "m": 0.5}], ids=str)
def test_ties(f, dtype):
    """All values equal; a few distinct values; the filters cut through equals, of which the lower ids stay."""
    u = torch.tensor([0.0, 0.25, 0.5, 0.75, 1 - 2.0 ** -24], device="cuda")
    check(torch.full((5, 1024), 1.5, device="cuda", dtype=DT[dtype]), u, **f)
    check(torch.zeros(5, 65536, device="cuda", dtype=DT[dtype]) * -1, u, **f)
    g = torch.Generator(device="cuda").manual_seed(1)
    some = torch.randint(0, 4, (5, 3001), device="cuda", generator=g).to(DT[dtype])
    check(some, torch.rand(5, device="cuda", generator=g), **f)
    signs = torch.where(some > 1, 0.0, -0.0).to(DT[dtype])          # 0 and -0 are equal
    check(signs, torch.rand(5, device="cuda", generator=g), **f)


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
def test_a_top_k_among_many_equals(dtype):
    """More values than threads at the bound, of one key and of several; greedy rows beside them; fewer values than k."""
    g = torch.Generator(device="cuda").manual_seed(3)
    u = torch.rand(6, device="cuda", generator=g)
    for V, k in ((700, 1), (5000, 3), (20011, 256), (65536, 100), (1 << 18, 200)):
        x = torch.randint(0, 3, (6, V), device="cuda", generator=g).to(DT[dtype])
        x[1] = 2.0
        x[2] = (torch.arange(V, device="cuda") % 600).to(DT[dtype]) * 0.125
        x[3, 5:] = -torch.inf
        x[4] = torch.arange(V, device="cuda").flip(0).clamp(max=400).to(DT[dtype])
        T = torch.tensor([1.0, 0.7, 2.0, 1.0, 0.0, 30.0], device="cuda")
        check(x, u, T, k)
        check(x, u, T, k, 0.8, 0.001)


def test_32_bit_logits_that_come_from_16_bits():
    """Thousands of equals in 32-bit rows, and values that differ in their last bit only."""
    x, u = rows_of(4, 65536, "bf16", seed=8, spread=(0.3, 2.0))
    for f in ({}, {"p": 0.9}, {"k": 4000}, {"k": 4000, "p": 0.7}):
        check(x.float(), u, **f)
    g = torch.Generator(device="cuda").manual_seed(2)
    close = 5.0 + torch.randint(0, 3000, (4, 20000), device="cuda", generator=g).float() * 2.0 ** -21
    for f in ({}, {"p": 0.4}, {"k": 10000}, {"T": 1e-4, "p": 0.6}, {"T": 1e6, "k": 700}):
        check(close, u, **f)


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
def test_masked_values_and_rows(dtype):
    x, u = rows_of(9, 3000, dtype, seed=9)
    x[0, 10:] = -torch.inf                                    # ten left
    x[1] = -torch.inf                                         # nothing
    x[2] = -torch.inf
    x[2, 2999] = 0.5                                          # one
    x[3, 7] = torch.nan
    x[4, 5] = x[4, 77] = torch.inf
    x[5, 100:] = torch.finfo(x.dtype).min
    x[6] = torch.finfo(x.dtype).min                           # all of the lowest value
    x[7, :] = torch.finfo(x.dtype).max
    x[8, 0] = torch.finfo(x.dtype).max
    x[8, 1:9] = -torch.inf
    for f in ({}, {"k": 30}, {"p": 0.8}, {"m": 0.1}, {"k": 2000, "p": 0.9, "m": 0.01}, {"T": 0.0}, {"T": 1e-30}, {"T": 1e30}):
        check(x, u, **f)
    nan = x.clone()
    nan[:, 2999] = -torch.nan                                 # of the other sign
    assert (ab.sampler_batch(nan, u)[0] == -1).all()


def test_ends_of_the_uniform_numbers():
    x, _ = rows_of(6, 999, "fp16", seed=10)
    u = torch.tensor([0.0, 1 - 2.0 ** -24, 1.0, 2.0, -1.0, float("nan")], device="cuda")
    ids, logp = ab.sampler_batch(x, u, top_p=0.9)
    v = [0.0, 1 - 2.0 ** -24, 1.0, 1.0, 0.0, 0.0]
    for r in range(6):
        want, want_p = drawn(x[r].double().cpu().numpy(), v[r], 1.0, 0, 0.9, 0.0)
        assert int(ids[r]) == want and abs(float(logp[r]) - want_p) < 1e-5


def test_numbers_out_of_range_in_tensors_filter_nothing_or_everything():
    x, u = rows_of(6, 999, "fp16", seed=11)
    t = lambda *v: torch.tensor(v, device="cuda")  # noqa: E731
    nan, inf = float("nan"), float("inf")
    check(x, u, T=t(-1.0, 0.0, inf, nan, 1e38, 1e-38))
    check(x, u, p=t(-1.0, 0.0, inf, nan, 1.0, 1e-38))
    check(x, u, m=t(-1.0, 0.0, inf, nan, 1.0, 1e-38))
    check(x, u, k=torch.tensor([-5, 0, 999, 2 ** 31 - 1, 998, 1], device="cuda", dtype=torch.int32))
    check(x, u, k=torch.tensor([2 ** 32 + 5, -2 ** 32 + 5, 2 ** 31, 2 ** 62, 3, 2 ** 32 + 1], device="cuda"))


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
def test_rows_on_any_address_and_stride(dtype):
    big, u = rows_of(20, 2103, dtype, seed=12)
    for lo in range(0, 9):
        check(big[:, lo:lo + 2000], u, p=0.9)
    check(big[::3, 5:1500], u[::3], k=40)                     # rows apart; uniform numbers apart
    check(big[:, ::2], u, k=40)                               # values apart: copied
    check(big.t().contiguous().t()[:, :700], u, p=0.5)
    check(big[:1].expand(20, -1), u, p=0.9)                   # one row, many draws
    check(big[3], u[3], p=0.9)                                # no batch at all
    check(big.view(2, 10, 2103)[:, :-1], u[:18].view(2, 9))   # two strides between rows


def test_rows_outside_of_the_batch_do_not_count():
    big = torch.full((8, 3000), torch.nan, device="cuda", dtype=torch.float16)
    x, u = rows_of(4, 2001, "fp16", seed=13)
    big[2:6, 501:2502] = x
    out = torch.full((8,), 77, device="cuda")
    ids, _ = check(big[2:6, 501:2502], u, p=0.9, out=out[2:6])
    assert ids.data_ptr() == out[2:6].data_ptr() and out[:2].tolist() == [77, 77] and out[6:].tolist() == [77, 77]


def test_large_vocabulary_and_many_rows():
    check(*rows_of(2, 1 << 18, "fp16", seed=14), p=0.9)
    check(*rows_of(2, 1 << 18, "fp32", seed=14), p=0.9)
    check(*rows_of(1, (1 << 18) - 3, "bf16", seed=14))
    check(*rows_of(2000, 65, "fp16", seed=15), p=0.9)


def test_offsets_beyond_32_bits():
    """More than 2^32 bytes, and 2^31 values, of logits; the last rows as by themselves."""
    n, V = 34000, 65536
    x = torch.zeros(n, V, device="cuda", dtype=torch.float16)
    tail, u = rows_of(20, V, "fp16", seed=22)
    x[-20:] = tail
    v = torch.cat([torch.full((n - 20,), 0.5, device="cuda"), u])
    for f in ({}, {"top_k": 40}, {"top_p": 0.8, "min_p": 0.01}):
        ids, logp = ab.sampler_batch(x, v, **f)
        want, want_p = ab.sampler_batch(tail, u, **f)
        assert torch.equal(ids[-20:], want) and torch.equal(logp[-20:], want_p)
        assert bool((ids[:-20] == ids[0]).all())
    check(tail, u)
    del x
    x = torch.zeros(20000, V, device="cuda")
    x[-20:] = tail.float()
    ids, _ = ab.sampler_batch(x, torch.cat([torch.full((20000 - 20,), 0.5, device="cuda"), u]), top_k=40)
    assert torch.equal(ids[-20:], ab.sampler_batch(tail, u, top_k=40)[0]) and bool((ids[:-20] == 20).all())   # 40 equals: the 21st


def test_no_rows():
    ids, logp = ab.sampler_batch(torch.empty(0, 100, device="cuda"), torch.empty(0, device="cuda"))
    assert ids.shape == logp.shape == (0, 1)


def test_draws_follow_the_distribution():
    """Evenly spread uniform numbers hit each value as often as its share says, to one."""
    x, _ = rows_of(1, 37, "fp32", seed=16, spread=(1.0, 1.0))
    n = 4096
    u = (torch.arange(n, device="cuda") + 0.5) / n
    ids, logp = ab.sampler_batch(x.expand(n, -1), u, temperature=0.7, top_k=20)
    w = torch.softmax(x[0].double() / 0.7, 0)
    keep = torch.zeros_like(w).scatter_(0, x[0].topk(20).indices, 1.0)
    share = w * keep / (w * keep).sum()
    assert ((torch.bincount(ids[:, 0], minlength=37) - n * share).abs() <= 1.0).all()
    assert torch.allclose(logp[:, 0].double(), share[ids[:, 0]].log(), atol=1e-6)


def test_pinned_ids_streams_graphs_and_repeats():
    x, u = rows_of(40, 50277, "fp16", seed=17)
    ids, logp = check(x, u, p=0.9)
    host = torch.zeros(40, dtype=torch.int64).pin_memory()
    ab.sampler_batch(x, u, top_p=0.9, out=host)
    torch.cuda.synchronize()
    assert host.tolist() == ids[:, 0].tolist()
    # two streams at once, different rows
    y, v = rows_of(40, 50277, "fp16", seed=18)
    other, s = ab.sampler_batch(y, v, top_k=50), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        with torch.cuda.stream(s):
            b = ab.sampler_batch(y, v, top_k=50)
        a = ab.sampler_batch(x, u, top_p=0.9)
        torch.cuda.synchronize()
        assert torch.equal(a[0], ids) and torch.equal(a[1], logp) and torch.equal(b[0], other[0]) and torch.equal(b[1], other[1])
    graph, gx, gu = torch.cuda.CUDAGraph(), x.clone(), u.clone()
    with torch.cuda.graph(graph):
        gi, gp = ab.sampler_batch(gx, gu, top_p=0.9)
    for seed in (19, 20):
        nx, nu = rows_of(40, 50277, "fp16", seed=seed)
        gx.copy_(nx), gu.copy_(nu)
        graph.replay()
        i, q = ab.sampler_batch(nx, nu, top_p=0.9)
        assert torch.equal(gi, i) and torch.equal(gp, q)


def test_log_probabilities_are_those_of_token_logp_without_filters():
    x, u = rows_of(30, 65536, "fp16", seed=21)
    ids, logp = ab.sampler_batch(x, u)
    want = ab.token_logp(x, ids[:, 0])
    assert torch.allclose(logp[:, 0], want, rtol=2e-6, atol=2e-6)   # (token_logp: sums in 32 bits)


# ------------------------------------------------------------------------------------------------------------------
# 4-bit products
# ------------------------------------------------------------------------------------------------------------------
def int4_inputs(M, N, K, group, zero, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed * 1009 + M + 3 * N + 5 * K + group)
    codes = torch.randint(0, 16, (N, K), device="cuda", generator=g, dtype=torch.uint8)
    w = codes[:, 0::2] | (codes[:, 1::2] << 4)
    scale = (0.01 * torch.exp(0.5 * torch.randn(N, K // group, device="cuda", generator=g))).to(DT[dtype])
    z = torch.randint(0, 16, (N, K // group), device="cuda", generator=g, dtype=torch.uint8) if zero else None
    return torch.randn(M, K, device="cuda", generator=g).to(DT[dtype]), w, scale, z


def int4_check(x, w, scale, zero, y=None):
    """A sum of a chunk is made by eight MMAs that may cut off what is below the last place of their 32-bit sums, 16 terms each (128 * 2^-23 of the sum of
    the terms' sizes at the very most); scaling and adding up chunks adds 2^-24 each. 2^-16 of the terms' sizes covers a single value. For random signs
    errors go with the roots of those numbers: 2e-5 of the 2-norm, beside the result's own rounding."""
    y = ab.linear_int4(x, w, scale, zero) if y is None else y
    q = torch.stack([w & 15, w >> 4], -1).view(scale.shape[0], scale.shape[1], -1).double()
    full = ((q - (8.0 if zero is None else zero.double()[..., None])) * scale.double()[..., None]).view(w.shape[0], -1)
    flat = x.reshape(-1, x.shape[-1]).double()
    want, size = flat @ full.T, flat.abs() @ full.abs().T
    half = torch.finfo(x.dtype).eps / 2
    assert y.shape == (*x.shape[:-1], w.shape[0]) and y.dtype == x.dtype
    d = (y.reshape(want.shape).double() - want).abs()
    tiny = torch.finfo(x.dtype).smallest_normal * half * 2
    assert bool((d <= half * want.abs() + 2.0 ** -16 * size + tiny).all()), float(d.max())
    assert float(d.norm()) <= (half + 2e-5) * float(want.norm()) + tiny * want.numel() ** 0.5
    return y


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("zero", [False, True])
@pytest.mark.parametrize("group,K", [(32, 32), (32, 96), (32, 4096), (64, 64), (64, 192), (64, 2560), (128, 128), (128, 640), (128, 4096), (256, 1024), (384, 768), (2560, 2560), (128, 16384)])
def test_products_with_4_bit_weights(group, K, zero, dtype):
    for M, N in ((1, 1), (1, 17), (1, 300), (2, 40), (3, 148), (5, 1000), (8, 64), (9, 33), (16, 200), (17, 90), (40, 31)):
        int4_check(*int4_inputs(M, N, K, group, zero, dtype))


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("M,N,K,group", [(1, 4096, 4096, 128), (1, 768, 768, 64), (8, 10240, 2560, 64), (16, 4096, 16384, 128), (16, 2049, 16384, 64), (8, 4096, 16384, 32),
                                         (1, 65536, 4096, 128), (2, 65537, 1024, 32), (1, 8, 65536, 128), (16, 130, 49152, 128), (1, 5, 262144, 64)])
def test_products_with_4_bit_weights_of_model_sizes(M, N, K, group, dtype):
    int4_check(*int4_inputs(M, N, K, group, True, dtype, seed=1))


@pytest.mark.parametrize("M", [1, 9, 16, 40])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_products_where_clusters_divide_the_inputs_and_passes_run_side_by_side(group, M):
    """Outputs around those up to which four and eight blocks share the inputs, pieces fewer than blocks, rows that make one pass, two and several."""
    for N in (1, 31, 33, 960, 1023, 1024, 1025, 2240, 2303, 2305):
        int4_check(*int4_inputs(M, N, 4224, group, False, "fp16", seed=2))
    for K in (896, 1024, 1152, 1920, 2048, 2176):
        int4_check(*int4_inputs(M, 515, K, group, True, "bf16", seed=3))
    int4_check(*int4_inputs(M, 16385, 4096, group, False, "fp16", seed=4))


def test_a_matrix_of_more_than_32_bits_of_bytes():
    N, K = 131072 + 7, 65536
    g = torch.Generator(device="cuda").manual_seed(9)
    w = torch.randint(0, 256, (N, K // 2), device="cuda", generator=g, dtype=torch.uint8)
    scale = (0.01 + 0.01 * torch.rand(N, K // 128, device="cuda", generator=g)).half()
    x = torch.randn(2, K, device="cuda", generator=g).half()
    y = ab.linear_int4(x, w, scale)
    for rows in (slice(0, 50), slice(N // 2, N // 2 + 50), slice(N - 50, N)):
        int4_check(x, w[rows].clone(), scale[rows], None, y[:, rows])


def test_quantizer_and_its_product():
    g = torch.Generator(device="cuda").manual_seed(5)
    w = 0.02 * torch.randn(513, 1024, device="cuda", generator=g)
    w[3] = 0.0
    w[4, :128] = 0.5
    for zeros in (False, True):
        for group in (32, 64, 128, 512):
            m = ab.quantize_int4(w, group, zeros)
            step = m.scale.float().repeat_interleave(group, 1)
            # half a step; and where a code is cut off at 0 or 15, what rounding the scale and the zero point moved the ends by: another half
            assert bool(((m.dequantize() - w).abs() <= 1.01 * step + 1e-7).all()) and bool((m.dequantize()[3] == 0).all())
            x = torch.randn(3, 1024, device="cuda", generator=g).half()
            int4_check(x, *m)


def test_special_activations_and_scales():
    x, w, scale, zero = int4_inputs(4, 50, 512, 64, True, "fp16")
    x[1] = 0
    x[2, 100] = torch.inf
    x[3, 7] = torch.nan
    y = ab.linear_int4(x, w, scale, zero)
    assert bool((y[1] == 0).all()) and bool(y[3].isnan().all())
    q = torch.stack([w & 15, w >> 4], -1).view(50, 512)[:, 100].int() - zero[:, 1].int()
    assert bool((y[2].isinf() == (q != 0)).all()) and bool((y[2].isnan() == (q == 0)).all())
    int4_check(x[:1], w, scale, zero)
    scale[5, 3] = torch.nan                                   # another group's scale reaches no other row or group
    scale[6] = 0
    y = ab.linear_int4(x[:2], w, scale, zero)
    assert bool(y[0, 5].isnan()) and float(y[0, 6]) == 0
    keep = [i for i in range(50) if i not in (5, 6)]
    int4_check(x[:2], w[keep], scale[keep], zero[keep], y[:, keep])


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_activations_of_any_shape_and_stride(dtype):
    big, w, scale, zero = int4_inputs(24, 70, 1024, 128, True, dtype)
    wide = torch.cat([big, big], 1)
    for lo in (0, 1, 3, 8):
        int4_check(wide[:, lo:lo + 1024], w, scale, zero)
    int4_check(wide[::5, 8:1032], w, scale, zero)
    int4_check(wide[:, ::2], w, scale, zero)
    int4_check(big[0], w, scale, zero)
    int4_check(big.view(2, 3, 4, 1024), w, scale, zero)
    int4_check(big[:1].expand(5, -1), w, scale, zero)
    int4_check(big, w[7:40], scale[7:40], zero[7:40])         # some of the outputs
    assert ab.linear_int4(big[:0], w, scale, zero).shape == (0, 70)


def test_products_repeat_bit_for_bit_on_streams_and_in_graphs():
    a, b = int4_inputs(1, 4096, 4096, 128, False, "fp16"), int4_inputs(6, 3000, 16384, 32, True, "fp16", seed=3)
    ya, yb = ab.linear_int4(*a), ab.linear_int4(*b)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        with torch.cuda.stream(s):
            again_b = ab.linear_int4(*b)
        again_a = ab.linear_int4(*a)
        torch.cuda.synchronize()
        assert torch.equal(again_a, ya) and torch.equal(again_b, yb)
    graph, x = torch.cuda.CUDAGraph(), a[0].clone()
    with torch.cuda.graph(graph):
        y = ab.linear_int4(x, *a[1:])
    for scale in (2.0, 0.5):
        x.copy_(a[0] * scale)
        graph.replay()
        assert torch.equal(y, ya * scale)


def test_weights_made_just_before_the_product():
    """The kernel may start early, but reads nothing before what was launched ahead of it is done."""
    x, w, scale, zero = int4_inputs(1, 4096, 4096, 64, True, "fp16")
    want = ab.linear_int4(x, w, scale, zero)
    torch.cuda.synchronize()
    for _ in range(20):
        w2, s2, z2, x2 = w.clone(), scale.clone(), zero.clone(), x.clone()
        got = ab.linear_int4(x2, w2, s2, z2)
        w2.zero_(), s2.zero_(), z2.zero_(), x2.zero_()
        assert torch.equal(got, want)


# ------------------------------------------------------------------------------------------------------------------
# refusals
# ------------------------------------------------------------------------------------------------------------------
def test_what_does_not_fit_is_refused():
    x, u = rows_of(4, 100, "fp16")
    for bad in (dict(u=u[:3]), dict(u=u.double()), dict(u=u.cpu()), dict(x=x.int()), dict(x=x.cpu()), dict(x=x[:, :0]), dict(x=torch.zeros(4, (1 << 18) + 1, device="cuda")),
                dict(temperature=-1.0), dict(temperature=float("nan")), dict(top_p=-0.1), dict(top_p=float("nan")), dict(min_p=-0.1), dict(temperature=u[:2]), dict(top_p=u.cpu()),
                dict(top_k=u), dict(top_p=torch.ones(4, device="cuda", dtype=torch.int32)), dict(out=torch.zeros(4, device="cuda")), dict(out=torch.zeros(4, dtype=torch.int64)),
                dict(out=torch.zeros(3, dtype=torch.int64, device="cuda")), dict(out=torch.zeros(8, dtype=torch.int64, device="cuda")[::2]),
                dict(x=x, out=x.view(torch.int64)[:, 0].as_strided((4,), (1,)))):
        args = {"x": x, "u": u, **bad}
        with pytest.raises(RuntimeError):
            ab.sampler_batch(args.pop("x"), args.pop("u"), **args)
    x, w, scale, zero = int4_inputs(2, 10, 256, 64, True, "fp16")
    for bad in (dict(x=x.float()), dict(x=x[:, :128]), dict(x=x.cpu()), dict(w=w.int()), dict(w=w[:, :64]), dict(w=w.cpu()), dict(w=w.t().contiguous().t()), dict(w=w[0]),
                dict(scale=scale.bfloat16()), dict(scale=scale[:, :3]), dict(scale=scale[:9]), dict(scale=scale.repeat_interleave(4, 1)), dict(scale=scale.cpu()), dict(zero=zero.int()),
                dict(zero=zero[:, :2]), dict(x=x.clone().requires_grad_()), dict(w=torch.cat([w, w], 0).view(-1)[8:8 + w.numel()].view(w.shape))):
        args = {"x": x, "w": w, "scale": scale, "zero": zero, **bad}
        with pytest.raises(RuntimeError):
            ab.linear_int4(**args)
    with torch.no_grad():
        ab.linear_int4(x.clone().requires_grad_(), w, scale, zero)
    assert _lib.device_status() == 0


def test_shapes_that_make_too_many_inputs_are_refused():
    x = torch.zeros(1, 1 << 20, device="cuda", dtype=torch.float16)
    w, s = torch.zeros(1, 1 << 19, device="cuda", dtype=torch.uint8), torch.ones(1, 1 << 13, device="cuda", dtype=torch.float16)
    with pytest.raises(RuntimeError, match="too many"):
        ab.linear_int4(x, w, s)


def test_tracing_is_refused():
    from torch.fx.experimental.proxy_tensor import make_fx
    x, u = rows_of(2, 50, "fp16")
    with pytest.raises(RuntimeError, match="traced"):
        make_fx(lambda a, b: ab.sampler_batch(a, b)[0])(x, u)
