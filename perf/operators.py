"""Performance cases of the operators that learn from sampled tokens, with their plain forms.

    listed()          the fixed cases          draw(rng)   one more case of the same ranges
    prepare(case, s)  what a program has in hand before the call
    run(state)        one pass: the plain form, or (own = True) the calls a user makes
    work(case)        bytes / flops a pass cannot do without
    exact(case, s)    the same outputs in 64 bits

Kinds of cases:
    wkv7        the WKV-7 recurrence over whole sequences, `RWKV7_TRAIN_OP`, with the gradients of all its inputs
    layer_norm  `layer_norm`: a block's norms (ln1, ln2, ln_out) and, in groups of a head, the norm behind the recurrence (ln_x)
    token_logp  `token_logp`: log-probabilities of given ids under logits (what a sampler's or a reference model's were)
    policy      `policy_loss` / `policy_loss_grad`: clipped ratios against the sampling policy, with a penalty for leaving a reference
    preference  `preference_loss`: pairs of answers, a better and a worse one

`grad` False is the forward pass alone. Sizes are those of the models (768, 2048, 2560 and 4096 wide, heads of 64, a vocabulary of
65536) and odd ones. Gradients of fp16 logits are scaled by 65536, as training in fp16 does.
"""
import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
SIZE = {"fp16": 2, "bf16": 2, "fp32": 4}
HEAD = 64
LOSS_SCALE = {"fp16": 65536.0, "bf16": 1.0, "fp32": 1.0}
CLIP = (0.2, 0.28)
KL = 0.05
BETA = 0.1


# ------------------------------------------------------------------------------------------------------------------
# the cases
# ------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one short sequence through the smallest model's heads: launch and chain latency
        {"name": "wkv7_b1_t37_h12_fp16", "kind": "wkv7", "B": 1, "T": 37, "H": 12, "dtype": "fp16", "ragged": False, "grad": True},
        # two long texts of unequal length, 2048 wide: few heads, a long axis
        {"name": "wkv7_b2_t4096_h32_bf16", "kind": "wkv7", "B": 2, "T": 4096, "H": 32, "dtype": "bf16", "ragged": True, "grad": True},
        # a batch of the widest model: what training in earnest calls
        {"name": "wkv7_b8_t1024_h64_fp16", "kind": "wkv7", "B": 8, "T": 1024, "H": 64, "dtype": "fp16", "ragged": False, "grad": True},
        # one row, forward: the smallest call
        {"name": "layer_norm_1x768_fp16", "kind": "layer_norm", "rows": 1, "C": 768, "groups": 1, "dtype": "fp16", "grad": False},
        # the norms of a training batch
        {"name": "layer_norm_8192x4096_bf16", "kind": "layer_norm", "rows": 8192, "C": 4096, "groups": 1, "dtype": "bf16", "grad": True},
        # the norm of each head behind the recurrence, an odd number of rows
        {"name": "layer_norm_4097x2560_g40_fp16", "kind": "layer_norm", "rows": 4097, "C": 2560, "groups": 40, "dtype": "fp16", "grad": True},
        # the log-probability of one sampled token
        {"name": "token_logp_1x65536_fp16", "kind": "token_logp", "rows": 1, "V": 65536, "dtype": "fp16", "grad": False},
        # a vocabulary that leaves rows on odd addresses, with gradients
        {"name": "token_logp_2049x50277_bf16", "kind": "token_logp", "rows": 2049, "V": 50277, "dtype": "bf16", "grad": True},
        # a few tokens, through autograd
        {"name": "policy_24x65536_fp16", "kind": "policy", "rows": 24, "V": 65536, "dtype": "fp16", "kl": True, "fused": False},
        # a batch of sampled answers, loss and gradient in one call
        {"name": "policy_4096x65536_fp16", "kind": "policy", "rows": 4096, "V": 65536, "dtype": "fp16", "kl": True, "fused": True},
        # two pairs of short answers
        {"name": "preference_2x37x65536_fp16", "kind": "preference", "P": 2, "T": 37, "V": 65536, "dtype": "fp16"},
        # four pairs of long ones
        {"name": "preference_4x512x65536_bf16", "kind": "preference", "P": 4, "T": 512, "V": 65536, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(("wkv7", "wkv7", "layer_norm", "layer_norm", "token_logp", "policy", "preference"))
    if kind == "wkv7":
        H, T = rng.choice((4, 12, 32, 40, 64)), _log(rng, 1, 4096)
        return {"kind": kind, "B": _log(rng, 1, max(1, min(64, 8 * 1024 * 64 // (H * T)))), "T": T, "H": H, "dtype": rng.choice(("fp16", "bf16")),
                "ragged": rng.random() < 0.5, "grad": rng.random() < 0.75}
    if kind == "layer_norm":
        groups = rng.choice((0, 0, 1))
        C = rng.choice((768, 2048, 2560, 4096)) if groups else rng.choice((768, 1000, 2048, 2560, 4096, _log(rng, 33, 4096)))
        return {"kind": kind, "rows": _log(rng, 1, 8192), "C": C, "groups": C // HEAD if groups else 1, "dtype": rng.choice(("fp16", "bf16", "fp32")),
                "grad": rng.random() < 0.75}
    V, dtype = rng.choice((1000, 32003, 50277, 65536)), rng.choice(("fp16", "bf16", "fp32"))
    top = 4096 // (2 if dtype == "fp32" else 1)
    if kind == "token_logp":
        return {"kind": kind, "rows": _log(rng, 1, top), "V": V, "dtype": dtype, "grad": rng.random() < 0.6}
    if kind == "policy":
        return {"kind": kind, "rows": _log(rng, 1, top), "V": V, "dtype": dtype, "kl": rng.random() < 0.6, "fused": rng.random() < 0.5}
    P = _log(rng, 1, 8)
    return {"kind": kind, "P": P, "T": _log(rng, 1, top // (2 * P)), "V": V, "dtype": dtype}


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

    def ints(self, *shape, hi):
        return torch.randint(hi, shape, device="cuda", generator=self.g)


def _logits(d, rows, V, dt):
    """Logits and the ids sampled under them, so that most log-probabilities are those of likely tokens."""
    logits = d.normal(rows, V).mul_(3.0).to(dt)
    ids = d.ints(rows, hi=V)
    top = logits.argmax(-1)
    return logits, torch.where(d.uniform(rows) < 0.5, top, ids)


def prepare(case, seed):
    d, kind, dt = _Draws(seed), case["kind"], DTYPES[case["dtype"]]
    s = {"case": case}
    if kind == "wkv7":
        B, T, H = case["B"], case["T"], case["H"]
        C = H * HEAD
        r, k, v = (d.normal(B, T, C, std=0.7).to(dt) for _ in range(3))
        # the decays and removal keys that the model's adapters make
        w = (-torch.nn.functional.softplus(-d.normal(B, T, C)) - 0.5).to(dt)
        kk = torch.nn.functional.normalize(d.normal(B, T, H, HEAD), dim=-1).view(B, T, C)
        a, b = (-kk).to(dt), (kk * torch.sigmoid(d.normal(B, T, C))).to(dt)
        state = d.normal(B, H, HEAD, HEAD, std=0.3)
        s["lengths"] = (T - d.ints(B, hi=T // 2 + 1)).to(torch.int32) if case["ragged"] else None
        s["dy"], s["dstate"] = d.normal(B, T, C, std=0.1).to(dt), d.normal(B, H, HEAD, HEAD, std=0.1)
        s["inputs"] = [t.requires_grad_(case["grad"]) for t in (state, r, w, k, v, a, b)]
    elif kind == "layer_norm":
        n, C = case["rows"], case["C"]
        x = (d.normal(n, C, std=2.0) + d.normal(n, 1)).to(dt)
        weight, bias = d.uniform(C, lo=0.8, hi=1.2).to(dt), d.normal(C, std=0.05).to(dt)
        s["dy"] = d.normal(n, C, std=0.1).to(dt)
        s["eps"] = 64e-5 if case["groups"] > 1 else 1e-5
        s["inputs"] = [t.requires_grad_(case["grad"]) for t in (x, weight, bias)]
    else:
        rows = case["rows"] if kind != "preference" else 2 * case["P"] * case["T"]
        logits, ids = _logits(d, rows, case["V"], dt)
        logp = torch.cat([torch.log_softmax(c, -1, dtype=torch.float32).gather(1, i[:, None])[:, 0] for c, i in zip(logits.split(512), ids.split(512))])
        s["scale"] = LOSS_SCALE[case["dtype"]]
        if kind == "token_logp":
            s["dlogp"] = d.normal(rows).mul_(s["scale"] / rows)
        elif kind == "policy":
            # the policy has moved a little since it sampled; a reference further away; some positions are prompt or padding
            # (ratios that land on the clip's border within rounding are moved off it: either side's gradient is right there)
            s["old"] = logp + d.normal(rows, std=0.15)
            ratio = torch.exp(logp - s["old"])
            for edge in (1.0 - CLIP[0], 1.0 + CLIP[1]):
                s["old"] = torch.where((ratio - edge).abs() < 1e-3, s["old"] + 0.01, s["old"])
            s["ref"] = logp + d.normal(rows, std=0.4) if case["kl"] else None
            s["advantages"] = d.normal(rows)
            s["mask"] = d.uniform(rows) < 0.85
        else:
            P, T = case["P"], case["T"]
            shape = (2 * P, T)
            n = T - d.ints(2 * P, hi=T // 2 + 1)
            s["mask"] = torch.arange(T, device="cuda")[None] < n[:, None]
            s["ref"] = (logp.view(shape) * s["mask"]).sum(-1) + d.normal(2 * P, std=3.0)
            logits, ids = logits.view(*shape, -1), ids.view(shape)
        s["logits"], s["ids"] = logits.requires_grad_(kind == "preference" or (kind == "policy" and not case["fused"]) or case.get("grad", False)), ids
    return s


# ------------------------------------------------------------------------------------------------------------------
# plain forms, in 32 bits
# ------------------------------------------------------------------------------------------------------------------
def _plain_wkv7(s):
    """S_t = S_{t-1} diag(d_t) + (S_{t-1} a_t) b_t^T + v_t k_t^T,  y_t = S_t r_t,  d_t = exp(-exp(w_t)), from the first step to the last one;
    with G for the gradient of S_t, back from the last one."""
    state, r, w, k, v, a, b = s["inputs"]
    B, T, C = r.shape
    H, dt = C // HEAD, r.dtype
    steps = lambda t: t.float().view(B, T, H, HEAD).transpose(0, 1)  # noqa: E731
    r, w, k, v, a, b, dy = (steps(t) for t in (r, w, k, v, a, b, s["dy"]))
    lw = -torch.exp(w)
    if s["lengths"] is not None:  # steps behind a sequence's end leave its state alone
        live = (torch.arange(T, device="cuda")[:, None] < s["lengths"][None]).float()[:, :, None, None]
        r, k, v, a, b, dy, lw = (t * live for t in (r, k, v, a, b, dy, lw))
    dec = torch.exp(lw)
    col, row = (lambda t: t[..., :, None]), (lambda t: t[..., None, :])  # noqa: E731
    S, states, us, ys = state.float(), [], [], []
    for t in range(T):
        states.append(S)
        u = torch.matmul(S, col(a[t]))
        S = S * row(dec[t]) + u * row(b[t]) + col(v[t]) * row(k[t])
        us.append(u[..., 0])
        ys.append(torch.matmul(S, col(r[t]))[..., 0])
    back = lambda t: torch.stack(t).transpose(0, 1).reshape(B, T, C)  # noqa: E731
    out = {"y": back(ys).to(dt), "state": S}
    if not s["case"]["grad"]:
        return out
    G, d = s["dstate"].float(), {n: [None] * T for n in "rwkvab"}
    for t in range(T - 1, -1, -1):
        before = states[t]
        after = states[t + 1] if t + 1 < T else S
        G = G + col(dy[t]) * row(r[t])
        Gt = G.transpose(-1, -2)
        d["r"][t] = torch.matmul(after.transpose(-1, -2), col(dy[t]))[..., 0]
        d["v"][t] = torch.matmul(G, col(k[t]))[..., 0]
        d["k"][t] = torch.matmul(Gt, col(v[t]))[..., 0]
        d["b"][t] = torch.matmul(Gt, col(us[t]))[..., 0]
        du = torch.matmul(G, col(b[t]))
        d["a"][t] = torch.matmul(before.transpose(-1, -2), du)[..., 0]
        d["w"][t] = (G * before).sum(-2) * dec[t] * lw[t]
        G = G * row(dec[t]) + du * row(a[t])
    out["dstate"] = G
    for n in "rwkvab":
        g = torch.stack(d[n])
        out["d" + n] = (g * live if s["lengths"] is not None else g).transpose(0, 1).reshape(B, T, C).to(dt)
    return out


def _plain_layer_norm(s):
    x, weight, bias = s["inputs"]
    n, C = x.shape
    g, dt = s["case"]["groups"], x.dtype
    xf, wf, bf = x.float().view(n, g, C // g), weight.float().view(g, -1), bias.float().view(g, -1)
    c = xf - xf.mean(-1, keepdim=True)
    rstd = torch.rsqrt((c * c).mean(-1, keepdim=True) + s["eps"])
    xh = c * rstd
    out = {"y": (xh * wf + bf).view(n, C).to(dt)}
    if s["case"]["grad"]:
        dy = s["dy"].float().view(n, g, -1)
        dxh = dy * wf
        dx = (dxh - dxh.mean(-1, keepdim=True) - xh * (dxh * xh).mean(-1, keepdim=True)) * rstd
        out |= {"dx": dx.view(n, C).to(dt), "dweight": (dy * xh).sum(0).view(C).to(dt), "dbias": dy.sum(0).view(C).to(dt)}
    return out


def _softmax_parts(logits, ids):
    """exp(x - max) and its sum in 32 bits, and the log-probability of the ids, which are added up over long answers, in 64."""
    x = logits.float()
    m = x.amax(-1, keepdim=True)
    at = x.gather(-1, ids[..., None]) - m
    e = torch.exp(x - m)
    total = e.sum(-1, keepdim=True)
    return e, total, (at.double() - torch.log(total.double()))[..., 0]


def _dlogits(e, total, ids, coef, dt):
    """coef * (onehot - softmax)."""
    g = e * (-coef[..., None] / total)
    g.scatter_add_(-1, ids[..., None], coef[..., None])
    return g.to(dt)


def _plain_token_logp(s):
    logits, ids = s["logits"], s["ids"]
    e, total, logp = _softmax_parts(logits, ids)
    out = {"logp": logp.float()}
    if s["case"]["grad"]:
        out["dlogits"] = _dlogits(e, total, ids, s["dlogp"], logits.dtype)
    return out


def _plain_policy(s):
    logits, ids, A, live = s["logits"], s["ids"], s["advantages"].double(), s["mask"].double()
    e, total, logp = _softmax_parts(logits, ids)
    n = live.sum().clamp_min(1.0)
    ratio = torch.exp(logp - s["old"])
    plain, clipped = ratio * A, ratio.clamp(1.0 - CLIP[0], 1.0 + CLIP[1]) * A
    each = -torch.minimum(plain, clipped)
    coef = torch.where(plain <= clipped, -plain, torch.zeros_like(plain))
    if s["ref"] is not None:
        gap = s["ref"] - logp
        each = each + KL * (torch.exp(gap) - gap - 1.0)
        coef = coef + KL * (1.0 - torch.exp(gap))
    coef = (coef * live / n * s["scale"]).float()
    return {"loss": ((each * live).sum() / n).float(), "logp": (logp * live).float(), "dlogits": _dlogits(e, total, ids, coef, logits.dtype)}


def _plain_preference(s):
    logits, ids, live = s["logits"], s["ids"], s["mask"].double()
    P = logits.shape[0] // 2
    e, total, logp = _softmax_parts(logits, ids)
    answers = (logp * live).sum(-1)
    gap = answers - s["ref"]
    margin = BETA * (gap[:P] - gap[P:])
    loss = torch.log1p(torch.exp(-margin.abs())) + (-margin).clamp_min(0.0)
    pull = BETA / (1.0 + torch.exp(margin)) / P
    coef = (torch.cat([-pull, pull])[:, None] * live * s["scale"]).float()
    return {"loss": loss.mean().float(), "logp": answers.float(), "dlogits": _dlogits(e, total, ids, coef, logits.dtype)}


def _plain(s):
    return {"wkv7": _plain_wkv7, "layer_norm": _plain_layer_norm, "token_logp": _plain_token_logp, "policy": _plain_policy,
            "preference": _plain_preference}[s["case"]["kind"]](s)


# ------------------------------------------------------------------------------------------------------------------
# the framework's calls
# ------------------------------------------------------------------------------------------------------------------
def _called(s):
    import albatross_b200 as ab
    case, grad = s["case"], torch.autograd.grad
    if case["kind"] == "wkv7":
        state, r, w, k, v, a, b = s["inputs"]
        y, last = ab.RWKV7_TRAIN_OP(state, r, w, k, v, a, b, lengths=s["lengths"])
        if not case["grad"]:
            return {"y": y, "state": last}
        ds, dr, dw, dk, dv, da, db = grad((y, last), s["inputs"], (s["dy"], s["dstate"]))
        return {"y": y, "state": last, "dstate": ds, "dr": dr, "dw": dw, "dk": dk, "dv": dv, "da": da, "db": db}
    if case["kind"] == "layer_norm":
        y = ab.layer_norm(*s["inputs"], eps=s["eps"], groups=case["groups"])
        if not case["grad"]:
            return {"y": y}
        dx, dweight, dbias = grad(y, s["inputs"], s["dy"])
        return {"y": y, "dx": dx, "dweight": dweight, "dbias": dbias}
    logits, ids = s["logits"], s["ids"]
    if case["kind"] == "token_logp":
        logp = ab.token_logp(logits, ids)
        return {"logp": logp, "dlogits": grad(logp, logits, s["dlogp"])[0]} if case["grad"] else {"logp": logp}
    if case["kind"] == "policy":
        more = {"mask": s["mask"], "ref_logp": s["ref"], "clip": CLIP, "kl": KL if case["kl"] else 0.0}
        if case["fused"]:
            loss, logp, dlogits = ab.policy_loss_grad(logits, ids, s["old"], s["advantages"], scale=s["scale"], **more)
        else:
            loss, logp = ab.policy_loss(logits, ids, s["old"], s["advantages"], **more)
            dlogits, = grad(loss * s["scale"], logits)
        return {"loss": loss, "logp": logp, "dlogits": dlogits}
    loss, logp = ab.preference_loss(logits, ids, s["ref"], mask=s["mask"], beta=BETA)
    return {"loss": loss, "logp": logp, "dlogits": grad(loss * s["scale"], logits)[0]}


def run(s):
    if own:
        return _called(s)
    with torch.no_grad():
        return _plain(s)


# ------------------------------------------------------------------------------------------------------------------
# what a pass needs
# ------------------------------------------------------------------------------------------------------------------
def work(case):
    kind, e = case["kind"], SIZE[case["dtype"]]
    if kind == "wkv7":
        n, heads = case["B"] * case["T"] * case["H"], case["B"] * case["H"]
        if not case["grad"]:
            return {"bytes": 7.0 * e * n * HEAD + 2.0 * 16384 * heads, "flops": 9.0 * 4096 * n}
        # forward, and back with the states it needs made once more
        return {"bytes": 14.0 * e * n * HEAD + 4.0 * 16384 * heads, "flops": (9.0 + 7.0 + 21.0) * 4096 * n}
    if kind == "layer_norm":
        n = case["rows"] * case["C"]
        return {"bytes": ((4.0 if case["grad"] else 2.0) * n + 4.0 * case["C"]) * e, "flops": (16.0 if case["grad"] else 6.0) * n}
    rows = case["rows"] if kind != "preference" else 2 * case["P"] * case["T"]
    n = rows * case["V"]
    grad = case.get("grad", True)
    return {"bytes": (2.0 if grad else 1.0) * e * n + 24.0 * rows, "flops": (6.0 if grad else 4.0) * n}


# ------------------------------------------------------------------------------------------------------------------
# the same in 64 bits: the definitions, differentiated by autograd
# ------------------------------------------------------------------------------------------------------------------
def _exact_wkv7(s):
    x = [t.detach().double().requires_grad_(s["case"]["grad"]) for t in s["inputs"]]
    state, r, w, k, v, a, b = x
    B, T, C = r.shape
    n = [T] * B if s["lengths"] is None else s["lengths"].tolist()
    ends, ys, S = sorted(set(n)), [], state
    alive = torch.tensor(n, device="cuda")[:, None, None, None]
    head = lambda z, t: z[:, t].view(B, C // HEAD, HEAD)  # noqa: E731
    for t in range(T):
        d = torch.exp(-torch.exp(head(w, t)))
        new = torch.einsum("bhij,bhj->bhij", S, d) + torch.einsum("bhij,bhj,bhl->bhil", S, head(a, t), head(b, t)) \
            + torch.einsum("bhi,bhj->bhij", head(v, t), head(k, t))
        y = torch.einsum("bhij,bhj->bhi", new, head(r, t))
        if t < ends[0]:
            S = new
        else:
            S, y = torch.where(alive > t, new, S), torch.where(alive[..., 0] > t, y, torch.zeros_like(y))
        ys.append(y.reshape(B, C))
    y = torch.stack(ys, 1)
    out = {"y": y.detach(), "state": S.detach()}
    if s["case"]["grad"]:
        got = torch.autograd.grad((y, S), x, (s["dy"].double(), s["dstate"].double()))
        out |= dict(zip(("dstate", "dr", "dw", "dk", "dv", "da", "db"), got))
    return out


def _exact_layer_norm(s):
    x = [t.detach().double().requires_grad_(s["case"]["grad"]) for t in s["inputs"]]
    g = x[0].view(x[0].shape[0], s["case"]["groups"], -1)
    var, mean = torch.var_mean(g, dim=-1, correction=0, keepdim=True)
    y = ((g - mean) / torch.sqrt(var + s["eps"])).reshape(x[0].shape) * x[1] + x[2]
    out = {"y": y.detach()}
    if s["case"]["grad"]:
        out |= dict(zip(("dx", "dweight", "dbias"), torch.autograd.grad(y, x, s["dy"].double())))
    return out


def _exact_losses(s):
    kind, case = s["case"]["kind"], s["case"]
    z = s["logits"].detach().double().requires_grad_(kind != "token_logp" or case["grad"])
    logp = torch.log_softmax(z, -1).gather(-1, s["ids"][..., None]).squeeze(-1)
    if kind == "token_logp":
        out = {"logp": logp.detach()}
        if case["grad"]:
            out["dlogits"], = torch.autograd.grad(logp, z, s["dlogp"].double())
        return out
    live = s["mask"].double()
    if kind == "policy":
        A = s["advantages"].double()
        ratio = torch.exp(logp - s["old"].double())
        each = -torch.min(ratio * A, torch.clamp(ratio, 1 - CLIP[0], 1 + CLIP[1]) * A)
        if s["ref"] is not None:
            gap = s["ref"].double() - logp
            each = each + KL * (torch.expm1(gap) - gap)
        loss, said = (each * live).sum() / max(1.0, float(live.sum())), logp * live
    else:
        said = (logp * live).sum(-1)
        better, worse = (said - s["ref"].double()).chunk(2)
        loss = torch.nn.functional.softplus(-BETA * (better - worse)).mean()
    dlogits, = torch.autograd.grad(loss * s["scale"], z)
    return {"loss": loss.detach(), "logp": said.detach(), "dlogits": dlogits}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.enable_grad():
        return {"wkv7": _exact_wkv7, "layer_norm": _exact_layer_norm}.get(case["kind"], _exact_losses)(s)
