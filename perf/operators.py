"""Workloads of the training operators that go with a reward or a preference instead of a label map: the log-probability of given labels, the
clipped policy loss, the preference loss, and AdamW over many tensors with states in 32 or in 8 bits.

``run`` computes one pass of an operator: with ``own`` false in elementary torch operations, with ``own`` true through the package's
entry points.  ``exact`` gives the same in 64 bits, from the definitions.
"""
import math

import torch

own = False

DEV = "cuda"
BLOCK = 64    # elements that share a power of two in the 8-bit states
ALIGN = 256   # every tensor's states start at a multiple of this many elements
MASK = 0xFFFFFFFF


# ---------------------------------------------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the optimiser step of the DeepLab network as written (32 tensors, 65.1 M parameters), clipped by the gradients' global norm
        dict(name="adamw 32-bit, ref net, clipped", op="adamw", net="ref", state="f32", grad="f32", max_norm=1.0),
        # the same network at an eighth of its width: 32 small tensors, where the launches' latency is what counts
        dict(name="adamw 32-bit, narrow net", op="adamw", net="narrow", state="f32", grad="f32", max_norm=0.0),
        # 8-bit states for the same network: what a run takes that wants the memory for activations
        dict(name="adamw 8-bit, ref net", op="adamw", net="ref", state="u8", grad="f32", max_norm=0.0),
        # several hundred tensors of every size, gradients as a data-parallel job's bf16 exchange leaves them, clipped
        dict(name="adamw 8-bit, 320 tensors, bf16 gradients", op="adamw", net="many", count=320, total=200_000_000, state="u8", grad="bf16",
             max_norm=1.0),
        # a batch of 16 label maps of 41 x 41 pixels over 21 classes (rows padded to 24), sampled from the network and rewarded
        dict(name="policy loss, 16 maps 41x41x21", op="policy", rows=16 * 41 * 41, classes=21, ldl=24, dtype="f32"),
        # a batch of token sequences over a large vocabulary
        dict(name="policy loss, 4096 x 65536 bf16", op="policy", rows=4096, classes=65536, ldl=65536, dtype="bf16"),
        # a few rows of an odd, very wide vocabulary: the rows alone do not fill the card
        dict(name="policy loss, 7 x 128001 bf16", op="policy", rows=7, classes=128001, ldl=128001, dtype="bf16"),
        # 12 pairs of label maps
        dict(name="preference loss, 12 pairs of maps", op="preference", pairs=12, longest=41 * 41, ragged=False, classes=21, ldl=24, dtype="f32"),
        # 8 pairs of token sequences of up to 512 tokens, packed one behind the other
        dict(name="preference loss, 8 pairs x 32768 bf16", op="preference", pairs=8, longest=512, ragged=True, classes=32768, ldl=32768,
             dtype="bf16"),
        # log-probabilities of a batch of label maps at the full resolution of the image
        dict(name="label logp, 16 maps 321x321x21", op="logp", rows=16 * 321 * 321, classes=21, ldl=24, dtype="f32", backward=False),
        # scores of a reference model, in 32 bits, an odd number of classes
        dict(name="label logp, 1500 x 100003 f32", op="logp", rows=1500, classes=100003, ldl=100003, dtype="f32", backward=False),
        # forward and gradient, as a loss of one's own over the log-probabilities needs them
        dict(name="label logp and gradient, 4001 x 32768", op="logp", rows=4001, classes=32768, ldl=32768, dtype="bf16", backward=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _ldl(rng, classes):
    to = rng.choice((1, 4, 8))
    return (classes + to - 1) // to * to


def draw(rng):
    op = rng.choice(("adamw", "adamw", "policy", "preference", "logp"))
    if op == "adamw":
        count = _log_int(rng, 1, 400)
        return dict(op="adamw", net="many", count=count, total=_log_int(rng, 1000 * count, 150_000_000), state=rng.choice(("f32", "u8")),
                    grad=rng.choice(("f32", "bf16")), max_norm=rng.choice((0.0, 1.0)))
    classes = _log_int(rng, 2, 131072)
    ldl, dtype = _ldl(rng, classes), rng.choice(("f32", "bf16"))
    most = 120_000_000 // ldl   # rows
    if op == "preference":
        pairs = _log_int(rng, 1, max(1, min(24, most // 2)))
        return dict(op=op, pairs=pairs, longest=_log_int(rng, 1, max(1, min(2048, most // (2 * pairs)))), ragged=rng.random() < 0.7,
                    classes=classes, ldl=ldl, dtype=dtype)
    case = dict(op=op, rows=_log_int(rng, 1, max(1, min(1_000_000, most))), classes=classes, ldl=ldl, dtype=dtype)
    if op == "logp":
        case["backward"] = rng.random() < 0.5
    return case


# ---------------------------------------------------------------------------------------------------------------------------------
# what a program has in hand
# ---------------------------------------------------------------------------------------------------------------------------------
def _net_shapes(width, fc_width, classes):
    """(elements, is a filter, is the classifier) of the DeepLab network's tensors, conv1_1 .. fc8."""
    c = [3] + [width * k for k in (1, 1, 2, 2, 4, 4, 4, 8, 8, 8, 8, 8, 8)]
    got = []
    for i in range(13):
        got += [(9 * c[i] * c[i + 1], 1, 0), (c[i + 1], 0, 0)]
    for k, ci, co, last in ((4, 8 * width, fc_width, 0), (1, fc_width, fc_width, 0), (1, fc_width, classes, 1)):
        got += [(k * k * ci * co, 1, last), (co, 0, last)]
    return got


def _tensors(case):
    """(elements, weight decay, multiplier of the learning rate) of every tensor."""
    if case["net"] == "many":
        k, total = case["count"], case["total"]
        share = [1.0 / (1 + (37 * i) % k) for i in range(k)]   # a long tail of small tensors, in no order of size
        unit = total / sum(share)
        return [(max(1, int(unit * s) | 1), 0.0 if i % 3 == 2 else 0.01, 1.0) for i, s in enumerate(share)]
    width, fc = (64, 4096) if case["net"] == "ref" else (8, 512)
    return [(n, 0.01 if filt else 0.0, (10.0 if last else 1.0) * (1.0 if filt else 2.0)) for n, filt, last in _net_shapes(width, fc, 21)]


def _round_up(n, to):
    return (n + to - 1) // to * to


def _prepare_adamw(case, gen):
    t = _tensors(case)
    lens = [_round_up(n, ALIGN) for n, _, _ in t]
    total = sum(lens)

    def normal(scale, dtype=torch.float32):
        return (torch.randn(total, generator=gen, device=DEV) * scale).to(dtype)

    inside = torch.zeros(total, dtype=torch.bool, device=DEV)   # the places between two tensors hold nothing
    at, starts = 0, []
    for (n, _, _), length in zip(t, lens):
        inside[at:at + n] = True
        starts.append(at)
        at += length
    # gradients of tensors whose scales differ, trained weights, moments of a run that has gone for a while
    scale = torch.exp(torch.randn(len(t), generator=gen, device=DEV) - 6.0)
    scale = torch.repeat_interleave(scale, torch.tensor(lens, device=DEV))
    s = dict(op="adamw", state=case["state"], lr=1e-4, b1=0.9, b2=0.999, eps=1e-8, max_norm=case["max_norm"], seed=12345,
             w=normal(0.05) * inside, g=(normal(1.0) * scale * inside).to(torch.bfloat16 if case["grad"] == "bf16" else torch.float32),
             steps=torch.full((1,), 100, dtype=torch.int64, device=DEV),
             lens=torch.tensor(lens, device=DEV), wd=torch.tensor([x[1] for x in t], device=DEV), ls=torch.tensor([x[2] for x in t], device=DEV),
             starts=starts, sizes=[x[0] for x in t])
    m = normal(0.3) * scale * inside
    r = normal(0.4).abs() * scale * inside + scale * inside * 0.1
    if case["state"] == "f32":
        s["m"], s["v"] = m, r * r
    else:   # values that the 8-bit states can hold: nearest ones of the formats
        s["m"], s["r"] = _kept(m.abs().double(), 0.5, 3).copysign(m.double()).float(), _kept(r.double(), 0.5, 4).float()
    if own:
        from em_adapt_tensorflow_amd import ops
        views = [(s["w"][a:a + n], s["g"][a:a + n]) for a, n in zip(starts, s["sizes"])]
        opt = ops.AdamW([v[0] for v in views], [v[1] for v in views], state=case["state"], betas=(s["b1"], s["b2"]), eps=s["eps"],
                        weight_decay=[x[1] for x in t], lr_scale=[x[2] for x in t], seed=s["seed"])
        opt.steps.copy_(s["steps"])
        if case["state"] == "f32":
            opt.m.copy_(s["m"])
            opt.v.copy_(s["v"])
        else:
            opt.pack(s["m"], s["r"])
        s["opt"] = opt
    return s


def _labels_of(z, classes, gen):
    """Labels sampled from the rows' softmax."""
    out = torch.empty(z.shape[0], dtype=torch.int64, device=DEV)
    step = max(1, 50_000_000 // z.shape[1])
    for i in range(0, z.shape[0], step):
        u = torch.rand(z[i:i + step, :classes].shape, generator=gen, device=DEV).clamp_(1e-12, 1 - 1e-7)
        out[i:i + step] = (z[i:i + step, :classes].float() - torch.log(-torch.log(u))).argmax(1)
    return out


def _scores(z, labels, classes):
    """log softmax of the labels, to make the inputs around."""
    out = torch.empty(z.shape[0], dtype=torch.float32, device=DEV)
    step = max(1, 50_000_000 // z.shape[1])
    for i in range(0, z.shape[0], step):
        p = torch.log_softmax(z[i:i + step, :classes].float(), 1)
        out[i:i + step] = p.gather(1, labels[i:i + step, None])[:, 0]
    return out


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    if case["op"] == "adamw":
        return _prepare_adamw(case, gen)
    host = torch.Generator().manual_seed(int(seed))
    s = dict(op=case["op"], classes=case["classes"], backward=case.get("backward", True))
    if case["op"] == "preference":
        n = 2 * case["pairs"]
        lens = torch.full((n,), case["longest"])
        if case["ragged"]:   # the same lengths for every seed, in another order
            lens = lens - torch.arange(n) * (case["longest"] // 2) // n
            lens = lens[torch.randperm(n, generator=host)]
        s["seq_start"] = torch.cat([torch.zeros(1, dtype=torch.int64), lens.cumsum(0)]).to(DEV)
        rows = int(lens.sum())
    else:
        rows = case["rows"]
    z = torch.randn((rows, case["ldl"]), generator=gen, device=DEV, dtype=torch.float32).mul_(2.5)
    s["z"] = z = z.to(torch.bfloat16 if case["dtype"] == "bf16" else torch.float32)
    s["labels"] = labels = _labels_of(z, case["classes"], gen)

    def normal(n, scale):
        return torch.randn(n, generator=gen, device=DEV) * scale

    if case["op"] == "preference":
        logp = _scores(z, labels, case["classes"]).double()
        sums = torch.cat([torch.zeros(1, dtype=torch.float64, device=DEV), logp.cumsum(0)])
        s["ref"] = ((sums[s["seq_start"][1:]] - sums[s["seq_start"][:-1]]).float() + normal(n, 4.0))
        s["beta"], s["smooth"] = 0.1, 0.05
    elif case["op"] == "policy":
        logp = _scores(z, labels, case["classes"])
        s["old"] = logp + normal(rows, 0.15)
        s["ref"] = logp + normal(rows, 0.3)
        s["adv"] = normal(rows, 1.0)
        s["weight"] = (torch.rand(rows, generator=gen, device=DEV) > 0.1).float()
        s["labels"][s["weight"] == 0] = 255 if case["classes"] <= 255 else -1   # void pixels; tokens of the prompt
        s["low"], s["high"], s["kl"], s["scale"] = 0.2, 0.28, 0.04, 1.0 / rows
    elif s["backward"]:
        s["dlogp"] = normal(rows, 1.0 / rows)
    return s


# ---------------------------------------------------------------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------------------------------------------------------------
def _kept(x, draw, bits):
    """What a float of 4 exponent bits and `bits` mantissa bits with the block's power of two keeps of x >= 0 (f64): the multiple of its
    step below x + draw * step.  The block's largest value is in the uppermost binade, or at its end."""
    x = x.view(-1, BLOCK)
    top = x.amax(1, keepdim=True)
    mant, e = torch.frexp(top)
    k = e - 1 + (2 * mant > 2 - 2.0 ** -bits).to(e.dtype)
    q = torch.ldexp(torch.ones_like(x), torch.maximum(torch.frexp(x)[1] - 1, k - 14) - bits)
    got = torch.floor(x / q + (draw.view(-1, BLOCK) if isinstance(draw, torch.Tensor) else draw)) * q
    if bits == 4:   # a root is never stored as zero unless it is
        got = torch.where(x > 0, torch.maximum(got, torch.ldexp(torch.ones_like(top), k - 14 - bits)), got)
    return got.view(-1)


def _mix(h):
    h = ((h ^ (h >> 16)) * 0x85EBCA6B) & MASK
    h = ((h ^ (h >> 13)) * 0xC2B2AE35) & MASK
    return h ^ (h >> 16)


def _draws(seed, step, n):
    """32 random bits for every element of a step: the package's counter-based generator with seed * 2^32 + step."""
    s1 = _mix((step & MASK) ^ _mix(torch.full_like(step, (seed + 0x9E3779B9) & MASK)))
    s2 = _mix((s1 + 0x7F4A7C15) & MASK)
    h = ((torch.arange(n, device=DEV) * 0x9E3779B1) & MASK) ^ s1
    h = ((h ^ (h >> 15)) * 0x2C1B3C6D + s2) & MASK
    h = ((h ^ (h >> 12)) * 0x297A2D39) & MASK
    return h ^ (h >> 15)


def _plain_adamw(s):
    g, b1, b2 = s["g"].float(), s["b1"], s["b2"]
    out = {}
    if s["max_norm"] > 0:
        norm = g.double().square().sum(0, keepdim=True).sqrt()
        out["norm"] = norm.float()
        g = g * torch.where(norm > s["max_norm"], s["max_norm"] / norm, 1.0).float()
    s["steps"] += 1
    t = s["steps"].double()
    of = torch.repeat_interleave(torch.arange(s["lens"].numel(), device=DEV), s["lens"] // ALIGN)   # the tensor of every ALIGN elements
    rate = ((s["lr"] / (1 - b1 ** t)).float() * s["ls"])[of, None]
    fade = (s["lr"] * s["ls"].double() * s["wd"].double()).float()[of, None]
    root2 = (1 / (1 - b2 ** t).sqrt()).float()
    m = s["m"] * b1 + g * (1 - b1)
    v = (s["v"] if s["state"] == "f32" else s["r"] * s["r"]) * b2 + (g * g) * (1 - b2)
    r = v.sqrt()
    w = s["w"].view(-1, ALIGN)
    w = (w - fade * w) - rate * (m / (r * root2 + s["eps"])).view(-1, ALIGN)
    s["w"].copy_(w.view(-1))
    if s["state"] == "f32":
        s["m"].copy_(m)
        s["v"].copy_(v)
        out |= {"w": s["w"], "m": s["m"], "v": s["v"]}
    else:
        h = _draws(s["seed"], s["steps"], m.numel())
        s["m"].copy_(_kept(m.abs().double(), (h & 0xFFFF).double() / 65536, 3).copysign(m.double()))
        s["r"].copy_(_kept(r.double(), (h >> 16).double() / 65536, 4))
        out |= {"w": s["w"], "m": s["m"].bfloat16(), "r": s["r"].bfloat16()}   # (exact: 4 and 5 bits and a power of two)
    out["steps"] = s["steps"]
    return out


def _one_hot(s, inside):
    return (torch.arange(s["z"].shape[1], device=DEV) == s["labels"][:, None]) & inside[:, None]


def _inside(s):
    return (s["labels"] >= 0) & (s["labels"] < s["classes"])


def _at_labels(x, s, inside):
    return x.gather(1, torch.where(inside, s["labels"], 0)[:, None])[:, 0]


def _padded(d, s):
    """d [rows, classes] as the gradient of the padded rows, in their type."""
    out = torch.zeros_like(s["z"])
    out[:, :s["classes"]] = d
    return out


def _gradient(s, z, lse, coef, inside):
    """(one hot - softmax) * coef of every row; rows without a label have none."""
    d = _one_hot(s, inside)[:, :s["classes"]].float() - torch.exp(z - lse[:, None])
    return _padded(torch.where(inside[:, None], d * coef[:, None], 0.0), s)


def _log_sum(z):
    top = z.amax(1)
    return top + torch.log(torch.exp(z - top[:, None]).sum(1))


def _plain_logp(s):
    z, inside = s["z"][:, :s["classes"]].float(), _inside(s)
    lse = _log_sum(z)
    out = {"logp": torch.where(inside, _at_labels(z, s, inside) - lse, 0.0), "lse": lse}
    if s["backward"]:
        out["dlogits"] = _gradient(s, z, lse, s["dlogp"], inside)
    return out


def _plain_policy(s):
    z, inside = s["z"][:, :s["classes"]].float(), _inside(s) & (s["weight"] != 0)
    lse = _log_sum(z.double())   # (64 bits: the clip decides at a border)
    logp = torch.where(inside, _at_labels(z, s, inside) - lse, 0.0)
    ratio = torch.exp(torch.where(inside, logp - s["old"], 0.0))
    adv, weight = s["adv"].double(), torch.where(inside, s["weight"], 0.0).double()
    free, held = -adv * ratio, -adv * ratio.clamp(1 - s["low"], 1 + s["high"])
    clipped = held > free
    gap = torch.where(inside, s["ref"] - logp, 0.0)
    kl = torch.exp(gap) - gap - 1
    part = torch.where(clipped, held, free)
    sums = torch.stack([(weight * (part + s["kl"] * kl)).sum(), (weight * part).sum(), (weight * kl).sum(), (weight * clipped).sum()])
    coef = weight * s["scale"] * (torch.where(clipped, 0.0, free) + s["kl"] * (1 - torch.exp(gap)))
    return {"sums": sums.float(), "logp": logp.float(), "dlogits": _gradient(s, z, lse.float(), coef.float(), inside)}


def _plain_preference(s):
    z, inside = s["z"][:, :s["classes"]].float(), _inside(s)
    lse = _log_sum(z)
    logp = torch.where(inside, _at_labels(z, s, inside) - lse, 0.0).double()
    at, rows = s["seq_start"], torch.arange(z.shape[0], device=DEV)
    sums = torch.cat([torch.zeros(1, dtype=torch.float64, device=DEV), logp.cumsum(0)])
    seq = sums[at[1:]] - sums[at[:-1]]
    ratio = seq - s["ref"].double()
    h = s["beta"] * (ratio[0::2] - ratio[1::2])
    soft = torch.log1p(torch.exp(-h.abs()))
    loss = (1 - s["smooth"]) * (soft - h.clamp(max=0)) + s["smooth"] * (soft + h.clamp(min=0))
    slope = s["beta"] * (s["smooth"] - 1 / (1 + torch.exp(h))) / h.numel()
    coef = torch.stack([slope, -slope], 1).view(-1)[torch.searchsorted(at[1:], rows, right=True)]
    return {"loss": loss.float(), "seq_logp": seq.float(), "dlogits": _gradient(s, z, lse, coef.float(), inside)}


PLAIN = {"adamw": _plain_adamw, "logp": _plain_logp, "policy": _plain_policy, "preference": _plain_preference}


# ---------------------------------------------------------------------------------------------------------------------------------
# the package's calls
# ---------------------------------------------------------------------------------------------------------------------------------
def _own(s):
    from em_adapt_tensorflow_amd import ops
    if s["op"] == "adamw":
        opt = s["opt"]
        opt.step(s["lr"], max_norm=s["max_norm"])
        out = {"w": s["w"], "steps": opt.steps}
        if s["max_norm"] > 0:
            out["norm"] = opt.grad_norm
        if s["state"] == "f32":
            out |= {"m": opt.m, "v": opt.v}
        else:
            out["m"], out["r"] = opt.unpack(torch.bfloat16)
        return out
    z, c = s["z"], s["classes"]
    if s["op"] == "logp":
        logp, lse = ops.label_logp(z, s["labels"], c)
        out = {"logp": logp, "lse": lse}
        if s["backward"]:
            out["dlogits"] = ops.label_logp_bwd(z, s["labels"], lse, s["dlogp"], c)
        return out
    if s["op"] == "policy":
        sums, logp, d = ops.policy_loss(z, s["labels"], s["old"], s["adv"], c, ref_logp=s["ref"], weights=s["weight"], clip_low=s["low"],
                                        clip_high=s["high"], kl_coef=s["kl"], grad_scale=s["scale"])
        return {"sums": sums, "logp": logp, "dlogits": d}
    loss, seq, d = ops.preference_loss(z, s["labels"], s["seq_start"], s["ref"], c, beta=s["beta"], label_smoothing=s["smooth"])
    return {"loss": loss, "seq_logp": seq, "dlogits": d}


def run(state):
    return _own(state) if own else PLAIN[state["op"]](state)


# ---------------------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "adamw":
        n = sum(x[0] for x in _tensors(case))
        grad = 2 if case["grad"] == "bf16" else 4
        if case["state"] == "f32":
            return {"bytes": n * (grad + 8 + 16), "flops": 15.0 * n}
        # weights, gradient, two states of 8 bits and 2 exponents a block, read and written; the states' values in 16 bits written
        return {"bytes": n * (grad + 8 + 4 + 4.0 / BLOCK + 4), "flops": 25.0 * n}
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "preference":
        n = 2 * case["pairs"]
        rows = sum(case["longest"] - (i * (case["longest"] // 2) // n if case["ragged"] else 0) for i in range(n))
    else:
        rows = case["rows"]
    c, ldl = case["classes"], case["ldl"]
    if case["op"] == "logp" and not case["backward"]:
        return {"bytes": rows * (c * size + 16.0), "flops": 4.0 * rows * c}
    per_row = {"logp": 20.0, "policy": 28.0, "preference": 8.0}[case["op"]]
    return {"bytes": rows * (c * size + ldl * size + per_row), "flops": 8.0 * rows * c}


# ---------------------------------------------------------------------------------------------------------------------------------
# 64 bits, from the definitions
# ---------------------------------------------------------------------------------------------------------------------------------
def _exact_kept(x, sign, draw, bits):
    """The stored value of sign * x by the formats' own grid: with the block's exponent k, x is a whole number of steps 2^(e - bits) in the
    binade e, and steps of the smallest binade (k - 14) below that; the random draw in [0, 1) of a step is added before the cut."""
    blocks = x.view(-1, BLOCK)
    top = blocks.max(1).values
    k = torch.floor(torch.log2(torch.where(top > 0, top, 1.0)))
    k = torch.where(top >= 2.0 ** (k + 1), k + 1, torch.where(top < 2.0 ** k, k - 1, k))
    k = torch.where(top > 2.0 ** k * (2 - 2.0 ** -bits), k + 1, k)
    k = torch.repeat_interleave(k, BLOCK)
    e = torch.floor(torch.log2(torch.where(x > 0, x, 1.0)))
    e = torch.where(x >= 2.0 ** (e + 1), e + 1, torch.where(x < 2.0 ** e, e - 1, e))
    step = 2.0 ** (torch.where(x > 0, torch.maximum(e, k - 14), k - 14) - bits)
    got = torch.floor(x / step + draw) * step
    if bits == 4:
        got = torch.where((x > 0) & (got == 0), 2.0 ** (k - 14 - bits), got)
    return got * sign


def _exact_adamw(case, s):
    from_state = {k: (v.double() if isinstance(v, torch.Tensor) else v) for k, v in s.items()}
    g, w = from_state["g"], from_state["w"].clone()
    m, v = from_state["m"], from_state["v"] if case["state"] == "f32" else from_state["r"] ** 2
    t, lr, b1, b2 = int(s["steps"]) + 1, s["lr"], s["b1"], s["b2"]
    out = {"steps": torch.tensor([t], device=DEV)}
    if s["max_norm"] > 0:
        norm = math.sqrt(float((g * g).sum()))
        out["norm"] = torch.tensor([norm], dtype=torch.float64, device=DEV)
        g = g * min(1.0, s["max_norm"] / norm)
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    for (n, wd, ls), a in zip(_tensors(case), s["starts"]):
        i = slice(a, a + n)
        w[i] -= lr * ls * wd * w[i] + lr * ls * (m[i] / (1 - b1 ** t)) / ((v[i] / (1 - b2 ** t)).sqrt() + s["eps"])
    out["w"] = w
    if case["state"] == "f32":
        out |= {"m": m, "v": v}
    else:
        h = _draws(s["seed"], s["steps"] + 1, m.numel())   # (random numbers are inputs)
        out["m"] = _exact_kept(m.abs(), torch.sign(m), (h % 65536).double() / 65536, 3)
        out["r"] = _exact_kept(v.sqrt(), 1.0, (h // 65536).double() / 65536, 4)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "adamw":
        return _exact_adamw(case, s)
    c, rows = case["classes"], s["z"].shape[0]
    labels = s["labels"]
    used = (labels >= 0) & (labels < c)
    if case["op"] == "policy":
        used &= s["weight"] != 0
    step = max(1, 60_000_000 // case["ldl"])
    lse = torch.empty(rows, dtype=torch.float64, device=DEV)
    logp = torch.zeros(rows, dtype=torch.float64, device=DEV)
    for i in range(0, rows, step):
        z = s["z"][i:i + step, :c].double()
        lse[i:i + step] = torch.logsumexp(z, 1)
        logp[i:i + step] = torch.where(used[i:i + step], z.gather(1, labels[i:i + step].clamp(0, c - 1)[:, None])[:, 0] - lse[i:i + step], 0.0)
    if case["op"] == "logp":
        out = {"logp": logp, "lse": lse}
        if not case["backward"]:
            return out
        coef = s["dlogp"].double()
    elif case["op"] == "policy":
        a, wt = s["adv"].double()[used], s["weight"].double()[used]
        ratio = torch.exp(logp[used] - s["old"].double()[used])
        q = s["ref"].double()[used] - logp[used]
        bounded = torch.minimum(torch.maximum(ratio, torch.full_like(ratio, 1 - s["low"])), torch.full_like(ratio, 1 + s["high"]))
        surrogate, kl = torch.maximum(-a * ratio, -a * bounded), torch.expm1(q) - q
        cut = -a * bounded > -a * ratio
        out = {"sums": torch.stack([(wt * (surrogate + s["kl"] * kl)).sum(), (wt * surrogate).sum(), (wt * kl).sum(), wt[cut].sum()]), "logp": logp}
        coef = torch.zeros(rows, dtype=torch.float64, device=DEV)
        coef[used] = wt * s["scale"] * (torch.where(cut, 0.0, -a * ratio) - s["kl"] * torch.expm1(q))
    else:
        at = s["seq_start"].tolist()
        seq = torch.stack([logp[at[i]:at[i + 1]].sum() for i in range(len(at) - 1)])
        d = (seq - s["ref"].double()).view(-1, 2)
        h = s["beta"] * (d[:, 0] - d[:, 1])
        up, down = -torch.nn.functional.logsigmoid(h), -torch.nn.functional.logsigmoid(-h)
        out = {"loss": (1 - s["smooth"]) * up + s["smooth"] * down, "seq_logp": seq}
        slope = s["beta"] / len(h) * (-(1 - s["smooth"]) * torch.sigmoid(-h) + s["smooth"] * torch.sigmoid(h))
        coef = torch.zeros(rows, dtype=torch.float64, device=DEV)
        for i in range(len(h)):
            coef[at[2 * i]:at[2 * i + 1]] = slope[i]
            coef[at[2 * i + 1]:at[2 * i + 2]] = -slope[i]
    d = torch.zeros(s["z"].shape, dtype=torch.float64, device=DEV)
    for i in range(0, rows, step):
        part = -torch.exp(s["z"][i:i + step, :c].double() - lse[i:i + step, None])
        part.scatter_add_(1, labels[i:i + step].clamp(0, c - 1)[:, None], torch.ones_like(part[:, :1]))
        d[i:i + step, :c] = part * torch.where(used[i:i + step], coef[i:i + step], 0.0)[:, None]
    out["dlogits"] = d
    return out
