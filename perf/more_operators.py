"""Performance cases of the operators around a sampled token (the draw itself, products with 4-bit weights in groups) and of the
gradient norm that training ends with, with their plain forms.

    listed()          the fixed cases          draw(rng)   one more case of the same ranges
    prepare(case, s)  what a program has in hand before the call
    run(state)        one pass: the plain form, or (own = True) the calls a user makes
    work(case)        bytes / flops a pass cannot do without
    exact(case, s)    the same outputs in 64 bits

Kinds of cases:
    sample  `sampler_batch`: one id per row of logits under a temperature, top-k, top-p and min-p, from given uniform numbers, and its
            log-probability under the distribution it was drawn from
    int4    `linear_int4`: a few rows of activations by a matrix of 4-bit codes with a scale, and perhaps a zero point, for each group of inputs
    clip    `clip_grad_norm`: the norm over all gradients of a model, the loss scale taken out, and the gradients clipped into the optimizer's buffers

Sizes are those of the models (256, 768, 2560 and 4096 wide, hidden layers four times as wide, a vocabulary of 65536) and odd ones.
"""
import numpy as np
import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
SIZE = {"fp16": 2, "bf16": 2, "fp32": 4}
LOSS_SCALE = {"fp16": 65536.0, "bf16": 1.0, "fp32": 1.0}


# ------------------------------------------------------------------------------------------------------------------
# the cases
# ------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one user's next token
        {"name": "sample_1x65536_fp16_top_p", "kind": "sample", "rows": 1, "V": 65536, "dtype": "fp16", "each": False, "T": 1.0, "k": 0, "p": 0.7, "m": 0.0},
        # a rollout for learning: the whole distribution, rows on odd addresses
        {"name": "sample_37x50277_bf16_all", "kind": "sample", "rows": 37, "V": 50277, "dtype": "bf16", "each": False, "T": 1.0, "k": 0, "p": 1.0, "m": 0.0},
        # a serving batch in which each request has filters of its own
        {"name": "sample_320x65536_fp16_each", "kind": "sample", "rows": 320, "V": 65536, "dtype": "fp16", "each": True, "T": 1.0, "k": 0, "p": 1.0, "m": 0.0},
        # many rows of 32-bit logits, everything at once
        {"name": "sample_512x65536_fp32_k50", "kind": "sample", "rows": 512, "V": 65536, "dtype": "fp32", "each": False, "T": 0.8, "k": 50, "p": 0.95, "m": 0.02},
        # a projection for one token
        {"name": "int4_1_4096x4096_g128_fp16", "kind": "int4", "rows": 1, "N": 4096, "K": 4096, "group": 128, "zero": False, "dtype": "fp16"},
        # the way back from the hidden layer: few outputs, a long axis, small groups with zero points
        {"name": "int4_1_4096x16384_g32_bf16", "kind": "int4", "rows": 1, "N": 4096, "K": 16384, "group": 32, "zero": True, "dtype": "bf16"},
        # a few users at once into the hidden layer
        {"name": "int4_8_16384x4096_g64_fp16", "kind": "int4", "rows": 8, "N": 16384, "K": 4096, "group": 64, "zero": True, "dtype": "fp16"},
        # the vocabulary's head
        {"name": "int4_1_65536x4096_g128_fp16", "kind": "int4", "rows": 1, "N": 65536, "K": 4096, "group": 128, "zero": False, "dtype": "fp16"},
        # a toy model's gradients, 32-bit throughout: latency
        {"name": "clip_l2_d256_fp32", "kind": "clip", "L": 2, "D": 256, "V": 512, "value_head": False, "dtype": "fp32", "out": "fp32", "over": True},
        # the smallest model in fp16 under a loss scale, into 32-bit gradients
        {"name": "clip_l12_d768_fp16", "kind": "clip", "L": 12, "D": 768, "V": 65536, "value_head": False, "dtype": "fp16", "out": "fp32", "over": True},
        # a value head's single bias in front leaves everything on odd addresses; a norm below the limit
        {"name": "clip_l6_d2560_odd_bf16", "kind": "clip", "L": 6, "D": 2560, "V": 50277, "value_head": True, "dtype": "bf16", "out": "fp32", "over": False},
        # four blocks of the widest model with its embedding and head
        {"name": "clip_l4_d4096_bf16", "kind": "clip", "L": 4, "D": 4096, "V": 65536, "value_head": False, "dtype": "bf16", "out": "bf16", "over": True},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(("sample", "sample", "int4", "int4", "clip"))
    if kind == "sample":
        V, dtype = rng.choice((1000, 32003, 50277, 65536, 65536, _log(rng, 33, 65536))), rng.choice(("fp16", "fp16", "bf16", "fp32"))
        return {"kind": kind, "rows": _log(rng, 1, 512), "V": V, "dtype": dtype, "each": rng.random() < 0.4, "T": rng.choice((0.5, 0.8, 1.0, 1.3)),
                "k": rng.choice((0, 0, 1, _log(rng, 2, 1000), 50)), "p": rng.choice((1.0, round(0.3 + 0.69 * rng.random(), 3))), "m": rng.choice((0.0, 0.0, 0.05))}
    if kind == "int4":
        group = rng.choice((32, 64, 128))
        K = group * _log(rng, max(1, 256 // group), 16384 // group)
        return {"kind": kind, "rows": _log(rng, 1, 16), "N": _log(rng, 64, min(65536, (1 << 27) // K)), "K": K, "group": group, "zero": rng.random() < 0.5,
                "dtype": rng.choice(("fp16", "bf16"))}
    D, dtype = rng.choice((256, 512, 768, 1000, 2048, 2560)), rng.choice(("fp16", "bf16", "fp32"))
    return {"kind": kind, "L": _log(rng, 1, 12 if D < 2000 else 6), "D": D, "V": _log(rng, 512, 65536), "value_head": rng.random() < 0.3, "dtype": dtype,
            "out": rng.choice((dtype, "fp32")) if dtype != "fp16" else "fp32", "over": rng.random() < 0.6}


# ------------------------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------------------------
class _Draws:
    """Tensors on the GPU from one seed, in the order they are asked for."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(1000003 * (int(seed) + 1))

    def normal(self, *shape, std=1.0, mean=0.0):
        return torch.empty(shape, device="cuda").normal_(mean, std, generator=self.g)

    def uniform(self, *shape, lo=0.0, hi=1.0):
        return torch.empty(shape, device="cuda").uniform_(lo, hi, generator=self.g)

    def ints(self, *shape, lo=0, hi):
        return torch.randint(lo, hi, shape, device="cuda", generator=self.g)


def _shapes(case):
    """The shapes of a model's trainable tensors, in the order of its checkpoint."""
    L, D, V = case["L"], case["D"], case["V"]
    ranks = (128, 128, 96, 480) if D >= 4096 else (64, 64, 32, 128) if D >= 768 else (32, 32, 16, 48)
    out = [(1, D), (1,)] if case["value_head"] else []
    out += [(V, D), (D,), (D,)]
    for i in range(L):
        out += [(D,)] * 4 + [(1, 1, D)] * 6
        for j, r in enumerate(ranks):
            if j != 2 or i > 0:
                out += ([(1, 1, D)] if j < 3 else []) + [(D, r), (r, D)]
        out += [(1, 1, D), (1, 1, D), (D // 64, 64) if D % 64 == 0 else (D,)] + [(D, D)] * 4 + [(D,), (D,), (1, 1, D), (4 * D, D), (D, 4 * D)]
    return out + [(D,), (D,), (V, D)]


def _numel(shape):
    n = 1
    for d in shape:
        n *= d
    return n


def _views(flat, shapes):
    out, at = [], 0
    for s in shapes:
        n = _numel(s)
        out.append(flat[at:at + n].view(s))
        at += n
    return out


def prepare(case, seed):
    d, kind, dt = _Draws(seed), case["kind"], DTYPES[case["dtype"]]
    s = {"case": case}
    if kind == "sample":
        rows, V = case["rows"], case["V"]
        # some rows are sure of their next token, others are not
        s["logits"] = (d.normal(rows, V) * d.uniform(rows, 1, lo=1.0, hi=4.0)).to(dt)
        s["u"] = d.uniform(rows)
        if case["each"]:
            s["T"] = torch.where(d.uniform(rows) < 0.1, torch.zeros(rows, device="cuda"), d.uniform(rows, lo=0.4, hi=1.4))
            s["k"] = torch.where(d.uniform(rows) < 0.5, d.ints(rows, lo=1, hi=200), 0).to(torch.int32)
            s["p"] = torch.where(d.uniform(rows) < 0.6, d.uniform(rows, lo=0.3, hi=1.0), torch.ones(rows, device="cuda"))
            s["m"] = torch.where(d.uniform(rows) < 0.3, d.uniform(rows, lo=0.0, hi=0.2), torch.zeros(rows, device="cuda"))
        else:
            s |= {n: case[n] for n in "Tkpm"}
    elif kind == "int4":
        N, K, G = case["N"], case["K"], case["group"]
        codes = d.normal(N, K).mul_(2.7).add_(8.0).round_().clamp_(0, 15).to(torch.uint8)
        s["w"] = codes[:, 0::2] | (codes[:, 1::2] << 4)
        s["scale"] = (0.0075 * torch.exp(0.2 * d.normal(N, K // G))).to(dt)
        s["zero"] = d.ints(N, K // G, lo=6, hi=11).to(torch.uint8) if case["zero"] else None
        s["x"] = d.normal(case["rows"], K).to(dt)
    else:
        shapes = _shapes(case)
        n = sum(_numel(x) for x in shapes)
        s["scale"] = LOSS_SCALE[case["dtype"]]
        s["limit"] = 1.0
        norm = 3.0 if case["over"] else 0.7
        s["flat"] = d.normal(n, std=norm / n ** 0.5 * s["scale"]).to(dt)
        s["flat_out"] = torch.empty(n, dtype=DTYPES[case["out"]], device="cuda")
        s["grads"], s["out"] = _views(s["flat"], shapes), _views(s["flat_out"], shapes)
    return s


# ------------------------------------------------------------------------------------------------------------------
# plain forms
# ------------------------------------------------------------------------------------------------------------------
def _plain_sample(s):
    """In 64 bits: which token is kept, and which is drawn, is decided next to borders. The likelier token comes first, of equals that of the lower id."""
    x, u = s["logits"], s["u"].double()[:, None]
    T, k, p, m = (s[n].double()[:, None] if torch.is_tensor(s[n]) else torch.full_like(u, s[n]) for n in "Tkpm")
    values, index = torch.sort(x, dim=-1, descending=True, stable=True)      # equals keep their order
    gap = values.double() - values[:, :1].double()
    e = torch.exp(gap / T.clamp_min(1e-300))
    rank = torch.arange(x.shape[1], device=x.device)[None]
    keep = ((k <= 0) | (rank < k)) & ((T > 0) | (rank < 1))
    e = e * keep
    before = torch.cumsum(e, -1) - e
    keep &= (before < p * e.sum(-1, keepdim=True)) | (p >= 1)
    keep &= e >= m
    keep[:, 0] = True
    e = e * keep
    cum = torch.cumsum(e, -1)
    at = (cum <= u * cum[:, -1:]).sum(-1, keepdim=True)
    return {"ids": index.gather(1, at), "logp": torch.log(e.gather(1, at) / cum[:, -1:]).float()}


def _plain_int4(s):
    w, scale, x = s["w"], s["scale"].float(), s["x"]
    N, groups = scale.shape
    q = torch.stack([w & 15, w >> 4], -1).view(N, groups, -1).float()
    zero = s["zero"].float()[..., None] if s["zero"] is not None else 8.0
    full = ((q - zero) * scale[..., None]).view(N, -1)
    return {"y": (x.float() @ full.T).to(x.dtype)}


def _plain_clip(s):
    """The gradients lie one behind the other, so that all of them are one long vector; its sum of squares is added up in 64 bits."""
    g = s["flat"].float()
    norm = s["scale"] * torch.sqrt((g * g).sum(dtype=torch.float64))
    factor = s["scale"] * torch.clamp(s["limit"] / norm, max=1.0)
    return {"norm": norm.float(), "grads": (g * factor.float()).to(s["flat_out"].dtype)}


# ------------------------------------------------------------------------------------------------------------------
# the framework's calls
# ------------------------------------------------------------------------------------------------------------------
def _called(s):
    import albatross_b200 as ab
    kind = s["case"]["kind"]
    if kind == "sample":
        ids, logp = ab.sampler_batch(s["logits"], s["u"], temperature=s["T"], top_k=s["k"], top_p=s["p"], min_p=s["m"])
        return {"ids": ids, "logp": logp}
    if kind == "int4":
        return {"y": ab.linear_int4(s["x"], s["w"], s["scale"], s["zero"])}
    norm = ab.clip_grad_norm(s["grads"], s["limit"], scale=s["scale"], out=s["out"])
    return {"norm": norm, "grads": s["flat_out"]}


def run(s):
    if own:
        return _called(s)
    with torch.no_grad():
        return {"sample": _plain_sample, "int4": _plain_int4, "clip": _plain_clip}[s["case"]["kind"]](s)


# ------------------------------------------------------------------------------------------------------------------
# what a pass needs
# ------------------------------------------------------------------------------------------------------------------
def work(case):
    kind, e = case["kind"], SIZE[case["dtype"]]
    if kind == "sample":
        n = case["rows"] * case["V"]
        return {"bytes": float(e) * n + (32.0 if case["each"] else 16.0) * case["rows"], "flops": 4.0 * n}
    if kind == "int4":
        N, K, M = case["N"], case["K"], case["rows"]
        return {"bytes": N * K / 2 + N * (K // case["group"]) * (3.0 if case["zero"] else 2.0) + 2.0 * M * (K + N), "flops": 2.0 * M * N * K}
    n = sum(_numel(x) for x in _shapes(case))
    return {"bytes": float(e + SIZE[case["out"]]) * n, "flops": 3.0 * n}


# ------------------------------------------------------------------------------------------------------------------
# the same in 64 bits, written from the definitions
# ------------------------------------------------------------------------------------------------------------------
def _exact_sample(s):
    """Row by row on the host."""
    ids, logp = [], []
    each = lambda n: s[n].double().tolist() if torch.is_tensor(s[n]) else [float(s[n])] * s["case"]["rows"]  # noqa: E731
    for x, u, T, k, p, m in zip(s["logits"].double().cpu().numpy(), s["u"].double().tolist(), *(each(n) for n in "Tkpm")):
        if T == 0:
            ids.append(int(np.argmax(x)))
            logp.append(0.0)
            continue
        w = np.exp((x - x.max()) / T)
        order = np.argsort(-x, kind="stable")
        if k > 0:
            order = order[:int(k)]
        if p < 1:
            cum = np.cumsum(w[order])
            order = order[:1 + int(np.count_nonzero(cum[:-1] < p * cum[-1]))]
        kept = np.concatenate([order[:1], order[1:][w[order[1:]] >= m]])
        cum = np.cumsum(w[kept])
        i = kept[np.searchsorted(cum, u * cum[-1], side="right")]
        ids.append(int(i))
        logp.append(float(np.log(w[i] / cum[-1])))
    return {"ids": torch.tensor(ids)[:, None], "logp": torch.tensor(logp, dtype=torch.float64)[:, None]}


def _exact_int4(s):
    N, groups = s["scale"].shape
    y = []
    for lo in range(0, N, 8192):
        w, scale = s["w"][lo:lo + 8192].int(), s["scale"][lo:lo + 8192].double()
        q = torch.empty(w.shape[0], 2 * w.shape[1], dtype=torch.float64, device=w.device)
        q[:, 0::2], q[:, 1::2] = w % 16, w // 16
        q = q.view(w.shape[0], groups, -1) - (8 if s["zero"] is None else s["zero"][lo:lo + 8192].double().unsqueeze(2))
        y.append(torch.einsum("mgi,ngi,ng->mn", s["x"].double().view(-1, groups, q.shape[2]), q, scale))
    return {"y": torch.cat(y, 1)}


def _exact_clip(s):
    norm = s["scale"] * sum(float(torch.linalg.vector_norm(g.double())) ** 2 for g in s["grads"]) ** 0.5
    factor = s["scale"] * (min(1.0, s["limit"] / norm))
    return {"norm": torch.tensor(norm, dtype=torch.float64), "grads": s["flat"].double() * factor}


def exact(case, seed):
    s = prepare(case, seed)
    return {"sample": _exact_sample, "int4": _exact_int4, "clip": _exact_clip}[case["kind"]](s)
