"""Workloads of the end of a training step: the objective on a model's logits with its gradient, and the update of the parameters.

Operators, each with a plain form in elementary torch operations and the calls that a user makes of repsurf_amd:

  adamw       optim.AdamW over many tensors at once: states in 32 bits, or in 8 bits with one exponent per 256 elements and a
              stochastic rounding whose dither is a fixed function of (seed, step, element); fp32 parameters, or bf16 ones with the
              low half of their fp32 master kept beside them; optionally scaled by the gradients' common norm
  logprobs    objectives.token_logprobs: log softmax(logits)[target] of every row, optionally with its backward pass
  policy      objectives.policy_loss: clipped policy objective with a KL term against a reference policy, forward and backward
  preference  objectives.preference_loss: paired log ratios of packed sequences, forward and backward

Packed batches: `offset` holds the running row ends of the sequences (clouds); rows behind the last one are padding."""
import math
import random

import torch

own = False

IGNORE = -100
LR, BETA1, BETA2, EPS, DECAY, T0 = 1e-3, 0.9, 0.999, 1e-8, 1e-2, 100
BLOCK = 256               # elements that share an exponent of an 8-bit state; tensors start at multiples of it in the flat buffers
CLIP, KL = 0.2, 0.05      # policy: ratio range 1 -+ CLIP, weight of the KL term
BETA = 0.1                # preference: scale of the log ratios

# the classifier's 67 parameter tensors (RepSurf-U, 15 classes)
CLASSIFIER = ("10x10,10,10,10x10,10,10,10,10x10,10,64x64,64,128x64,128,64,64,128,128,64x6,64,64x10,64,64,64,64,64,128x128,128,256x128,256,"
              "128,128,256,256,128x6,128,128x138,128,128,128,128,128,512x256,512,1024x512,1024,512,512,1024,1024,256x6,256,256x266,256,"
              "256,256,256,256,512x1024,512,512,512,256x512,256,256,256,15x256,15")
# two blocks of a generic transformer of width 2048: four square projections, the two matrices of the feed-forward part, two norms
BLOCKS = ",".join(["2048x2048,2048x2048,2048x2048,2048x2048,8192x2048,2048x8192,2048,2048"] * 2)


def listed():
    return [
        # the classifier's whole parameter list, as every one of its training steps updates it: a latency
        {"name": "adamw32_classifier", "op": "adamw", "bits": 32, "type": "float32", "shapes": CLASSIFIER, "clip": 0.0},
        # two blocks of a language model, gradients clipped by their common norm
        {"name": "adamw32_blocks_clip", "op": "adamw", "bits": 32, "type": "float32", "shapes": BLOCKS, "clip": 1.0},
        # bf16 training: an embedding of an odd number of rows, a block of odd width, its norms
        {"name": "adamw32_bf16_embedding", "op": "adamw", "bits": 32, "type": "bfloat16", "shapes": "50001x1024,4099x1023,1023x4099,1023,1023", "clip": 0.0},
        # the same list as the first with its states in 8 bits
        {"name": "adamw8_classifier", "op": "adamw", "bits": 8, "type": "float32", "shapes": CLASSIFIER, "clip": 0.0},
        # the blocks in 8 bits, clipped, bf16 parameters
        {"name": "adamw8_blocks_clip", "op": "adamw", "bits": 8, "type": "bfloat16", "shapes": BLOCKS, "clip": 1.0},
        # where 8-bit states are used for: many parameters on one card
        {"name": "adamw8_large", "op": "adamw", "bits": 8, "type": "float32", "shapes": "65536x2048,8192x8192,8192x8191,8192", "clip": 0.0},
        # the newest token of one sequence, scored: a latency
        {"name": "logprobs_one", "op": "logprobs", "rows": 1, "classes": 100001, "pad": 0, "type": "bfloat16", "banned": 0, "grad": False},
        # a batch of sequences scored by the reference model: nothing but the logits' one read
        {"name": "logprobs_batch", "op": "logprobs", "rows": 8192, "classes": 65536, "pad": 0, "type": "bfloat16", "banned": 0, "grad": False},
        # segmentation's batch of 16 clouds x 4096 points x 13 classes, a label for every point as the action
        {"name": "policy_points", "op": "policy", "sequences": 16, "longest": 4096, "ragged": False, "classes": 13, "pad": 0, "type": "float32",
         "behind": 0, "reduction": "token", "reference": True, "banned": 0},
        # a rollout batch of a language model: an odd vocabulary, prompts that do not count, padding rows behind the last sequence
        {"name": "policy_tokens", "op": "policy", "sequences": 12, "longest": 1000, "ragged": True, "classes": 50001, "pad": 0, "type": "bfloat16",
         "behind": 77, "reduction": "sequence", "reference": True, "banned": 5},
        # pairs of labelings of clouds, 13 classes
        {"name": "preference_points", "op": "preference", "pairs": 8, "longest": 4096, "ragged": True, "classes": 13, "pad": 0, "type": "float32",
         "behind": 0, "smoothing": 0.0, "average": False, "banned": 0},
        # pairs of answers of a language model with a large vocabulary
        {"name": "preference_tokens", "op": "preference", "pairs": 4, "longest": 1024, "ragged": True, "classes": 131072, "pad": 0, "type": "bfloat16",
         "behind": 64, "smoothing": 0.1, "average": False, "banned": 0},
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["adamw", "adamw", "logprobs", "policy", "policy", "preference"])
    if op == "adamw":
        room, shapes = _spread(rng, 1 << 14, 1 << 27), []
        for _ in range(_spread(rng, 2, 120)):
            n = min(_spread(rng, 1, room), room)
            room = max(1, room - n)
            a = _spread(rng, 1, min(n, 8192))
            shapes.append("%dx%d" % (a, n // a) if rng.random() < 0.7 else "%d" % n)
        return {"op": op, "bits": rng.choice([32, 8]), "type": rng.choice(["float32", "bfloat16"]), "shapes": ",".join(shapes),
                "clip": rng.choice([0.0, 1.0, 0.05])}
    classes = _spread(rng, 2, 131072)
    kind = rng.choice(["float32", "bfloat16", "bfloat16", "float16"])
    most = (1 << 28) // classes                      # rows of the largest logits a drawn case has
    common = {"op": op, "classes": classes, "pad": rng.choice([0, 0, rng.randint(1, 63)]), "type": kind,
              "banned": rng.choice([0, min(classes // 4, 7)])}
    if op == "logprobs":
        return {**common, "rows": _spread(rng, 1, min(most, 65536)), "grad": rng.random() < 0.5}
    n = _spread(rng, 1, 24)
    most = max(1, min(8192, most // (2 * n)))
    common.update(longest=_spread(rng, 1, most), ragged=rng.random() < 0.7, behind=rng.choice([0, rng.randint(1, 100)]))
    if op == "policy":
        return {**common, "sequences": n, "reduction": rng.choice(["token", "sequence"]), "reference": rng.random() < 0.7}
    return {**common, "pairs": n, "smoothing": rng.choice([0.0, 0.1]), "average": rng.random() < 0.5}


# ---------------------------------------------------------------------------------------------------------------- sizes
def _sizes(case):
    return [math.prod(int(x) for x in s.split("x")) for s in case["shapes"].split(",")]


def _flat(case):
    """(start of each tensor, elements of a flat buffer): every tensor starts at a multiple of BLOCK elements."""
    starts, at = [], 0
    for n in _sizes(case):
        starts.append(at)
        at += -(-n // BLOCK) * BLOCK
    return starts, at


def _lengths(case):
    n = case["sequences"] if case["op"] == "policy" else 2 * case["pairs"]
    if not case["ragged"]:
        return [case["longest"]] * n
    rng = random.Random(n * 1000003 + case["longest"] * 101 + case["classes"])
    return [rng.randint((case["longest"] + 1) // 2, case["longest"]) for _ in range(n)]


def _rows(case):
    return case["rows"] if case["op"] == "logprobs" else sum(_lengths(case)) + case["behind"]


def _counted(case):
    """rows that count: a sequence's first quarter is its prompt"""
    return case["rows"] if case["op"] == "logprobs" else sum(n - n // 4 for n in _lengths(case))


def work(case):
    if case["op"] == "adamw":
        n, p = sum(_sizes(case)), 2 if case["type"] == "bfloat16" else 4
        low = 2 if p == 2 else 0                                                    # the masters' low halves
        state = 16 if case["bits"] == 32 else 4 + 4 / BLOCK                         # read and written
        told = (0 if case["bits"] == 32 else 4) + (4 if p == 2 else 0)              # 8-bit states as values, masters in 32 bits
        return {"bytes": n * (p * 3 + 2 * low + state + told), "flops": n * (16 + (2 if case["clip"] else 0))}
    size, v = 4 if case["type"] == "float32" else 2, case["classes"]
    backward = case["op"] != "logprobs" or case["grad"]
    small = _rows(case) * (16 if case["op"] == "logprobs" else 24)
    return {"bytes": size * v * (_counted(case) + (_rows(case) if backward else 0)) + small, "flops": v * _counted(case) * (4 + (4 if backward else 0))}


# --------------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (_prepare_adamw if case["op"] == "adamw" else _prepare_logits)(case, seed, gen)


def _grid(gen, n, octaves, base):
    """positive values with four significant bits, spread over `octaves` powers of two below 2 ** base: what an 8-bit state can hold"""
    k = torch.randint(8, 16, (n,), generator=gen, device="cuda").float() / 8
    return k * torch.exp2((base - torch.randint(0, octaves, (n,), generator=gen, device="cuda")).float())


def _prepare_adamw(case, seed, gen):
    dtype = getattr(torch, case["type"])
    starts, total = _flat(case)
    sizes = _sizes(case)

    def flat(values):
        """zero in front of the next tensor's start, as a buffer of separate tensors is"""
        for a, n in zip(starts, sizes):
            values[a + n: a + -(-n // BLOCK) * BLOCK] = 0
        return values

    s = {"case": case, "t": T0, "seed": seed & 0x7FFFFFFF}
    s["p"] = flat((torch.randn(total, generator=gen, device="cuda") * 0.05)).to(dtype)
    s["g"] = flat(torch.randn(total, generator=gen, device="cuda") * 2e-3).to(dtype)
    sign = torch.randint(0, 2, (total,), generator=gen, device="cuda").float() * 2 - 1
    m = flat(_grid(gen, total, 6, -11) * sign)
    v = flat(_grid(gen, total, 9, -17))
    if own:
        from repsurf_amd.optim import AdamW
        shapes = [[int(x) for x in t.split("x")] for t in case["shapes"].split(",")]
        cut = lambda x: [x[a:a + n].view(*shape) for a, n, shape in zip(starts, sizes, shapes)]  # noqa: E731
        params = [torch.nn.Parameter(x) for x in cut(s["p"])]
        for p, g in zip(params, cut(s["g"])):
            p.grad = g
        opt = AdamW(params, lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY, state_bits=case["bits"],
                    max_grad_norm=case["clip"] or None, seed=s["seed"])
        opt.load_state_dict({"state": {i: {"step": torch.tensor(float(T0)), "exp_avg": a, "exp_avg_sq": b} for i, (a, b) in enumerate(zip(cut(m), cut(v)))},
                             "param_groups": opt.state_dict()["param_groups"]})
        s["opt"] = opt
    else:
        s.update(m=m, v=v)
        if dtype != torch.float32:
            s["master"] = s["p"].float()
    return s


def _prepare_logits(case, seed, gen):
    rows, v = _rows(case), case["classes"]
    dtype = getattr(torch, case["type"])
    whole = torch.empty(rows, v + case["pad"], dtype=dtype, device="cuda").normal_(0.0, 2.0, generator=gen)
    logits = whole[:, :v]                                                            # a row pitch of its own where the vocabulary is padded
    target = torch.randint(case["banned"], v, (rows,), generator=gen, device="cuda")
    here = torch.arange(rows, device="cuda")
    logits[here, target] += (torch.rand(rows, generator=gen, device="cuda") * 0.9 * math.log(v)).to(dtype)   # the taken actions are likely ones
    if case["banned"]:
        logits[:, :case["banned"]] = -math.inf                                       # actions that are never allowed
    s = {"case": case, "target": target, "logits": logits}
    if case["op"] == "logprobs":
        if case["grad"]:
            s["upstream"] = torch.randn(rows, generator=gen, device="cuda")
            s["logits"].requires_grad_(own)
        return s
    lengths = _lengths(case)
    ends = torch.tensor(lengths).cumsum(0)
    s["offset"] = ends.to(torch.int32).cuda()
    ignored, at = [], 0
    for n in lengths:
        ignored += range(at, at + n // 4)
        at += n
    ignored += range(at, rows)
    target[torch.tensor(ignored, dtype=torch.long, device="cuda")] = IGNORE
    picked = torch.empty(rows, device="cuda")
    for a in range(0, rows, 1024):
        z = logits[a:a + 1024].float()
        picked[a:a + 1024] = z.gather(1, target[a:a + 1024, None].clamp_min(0))[:, 0] - z.logsumexp(1)
    picked[target == IGNORE] = 0
    noise = lambda scale, n: torch.randn(n, generator=gen, device="cuda") * scale  # noqa: E731
    if case["op"] == "policy":
        s["old"] = picked + noise(0.15, rows)                                        # the policy that acted, a few updates ago
        s["reference"] = picked + noise(0.3, rows) if case["reference"] else None
        s["advantages"] = noise(1.0, rows)
    else:
        sums = torch.stack([x.sum(dtype=torch.float64) / (max(1, n - n // 4) if case["average"] else 1) for x, n in zip(picked.split(lengths + [case["behind"]]), lengths)])
        scale = torch.tensor([0.2 if case["average"] else 0.3 * math.sqrt(n) for n in lengths], device="cuda")
        s["reference"] = (sums + noise(1.0, len(lengths)) * scale).float()
    s["logits"].requires_grad_(own)
    return s


# ---------------------------------------------------------------------------------------------------------- plain forms
def _mix(x):
    """an integer hash of 32 bits in 64-bit words: the odd words are the fractions of the square roots of 2 and 3"""
    x = ((x ^ (x >> 16)) * 0x6A09E667) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0xBB67AE85) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _dither(seed, t, n):
    """two 16-bit numbers for each of n elements: the first for exp_avg, the second for exp_avg_sq"""
    block = torch.arange(n // BLOCK, device="cuda")
    key = _mix((_mix(torch.tensor((seed + t * 0x9E3779B9) & 0xFFFFFFFF, device="cuda")) + block) & 0xFFFFFFFF)
    r = _mix((key[:, None] + torch.arange(BLOCK, device="cuda") * 0x9E3779B9) & 0xFFFFFFFF).view(-1)
    return r >> 16, r & 0xFFFF


def _round8(x, octaves, d):
    """x to 4 significant bits: on the grid of its own power of two, at most `octaves` - 1 of them below the block's largest, and
    linear below that; up with the probability of the part that is cut off, as the 16-bit dither d says"""
    e = torch.frexp(x.abs())[1] - 1
    top = torch.where(x == 0, -126, e).view(-1, BLOCK).amax(1, keepdim=True).clamp_min(-126).expand(-1, BLOCK).reshape(-1)
    step = torch.exp2((torch.maximum(torch.where(x == 0, -1000, e), top - (octaves - 1)) - 3).double())
    return (torch.floor(x.abs().double() / step + (d.double() + 0.5) / 65536) * step), step


def _plain_adamw(s):
    case = s["case"]
    s["t"] += 1
    g = s["g"].float()
    norm = None
    if case["clip"]:
        norm = g.square().sum(dtype=torch.float64).sqrt().float()
        g = g * torch.clamp(case["clip"] / (norm + 1e-6), max=1.0)
    p = s["p"] if case["type"] == "float32" else s["master"]
    m = s["m"] + (g - s["m"]) * (1 - BETA1)
    v = s["v"] * BETA2 + (1 - BETA2) * g * g
    root = v.sqrt() / math.sqrt(1 - BETA2 ** s["t"]) + EPS
    p.copy_(p * (1 - LR * DECAY) - LR / (1 - BETA1 ** s["t"]) * (m / root))
    if case["bits"] == 8:
        dm, dv = _dither(s["seed"], s["t"], m.numel())
        q, _ = _round8(m, 14, dm)
        m = torch.where(m < 0, -q, q).float()
        q, step = _round8(v, 30, dv)
        v = torch.where((q == 0) & (v > 0), step, q).float()        # a second moment never becomes nothing
    s["m"], s["v"] = m, v
    out = {"p": p, "norm": norm}
    if case["type"] != "float32":
        s["p"].copy_(p)
        out.update(p=s["p"], master=p)
    narrow = torch.bfloat16 if case["bits"] == 8 else torch.float32      # an 8-bit state's values have four significant bits
    out.update(exp_avg=m.to(narrow), exp_avg_sq=v.to(narrow))
    return out


def _plain_rows(s):
    """(log-probability of each row's target in 64 bits, zero where the row does not count; probabilities in 32 bits; the rows that count)"""
    z = s["logits"].float()
    counts = s["target"] != IGNORE
    top = z.amax(1, keepdim=True)
    e = (z - top).exp()
    total = e.sum(1, dtype=torch.float64)
    taken = s["target"].clamp_min(0)[:, None]
    logp = (z.gather(1, taken) - top)[:, 0].double() - total.log()
    return torch.where(counts, logp, 0.0), e / total.float()[:, None], counts


def _plain_gradient(s, p, c):
    """c (rows) * (one at the target - p), rounded to the logits' type"""
    c = c.float()[:, None]
    g = p * -c
    taken = s["target"].clamp_min(0)[:, None]
    g.scatter_add_(1, taken, c)
    return g.to(s["logits"].dtype)


def _owner(s):
    """each row's sequence; the padding rows' is one behind the last"""
    return torch.searchsorted(s["offset"].long(), torch.arange(s["logits"].shape[0], device="cuda"), right=True)


def _plain_policy(s):
    case = s["case"]
    logp, p, counts = _plain_rows(s)
    if case["reduction"] == "token":
        w = counts.double() / counts.sum().clamp_min(1)
    else:
        owner, n = _owner(s), s["offset"].numel()
        held = torch.zeros(n + 1, dtype=torch.float64, device="cuda").index_add_(0, owner, counts.double())
        w = counts.double() / held.clamp_min(1)[owner] / n
    a, ratio = s["advantages"].double(), (logp - s["old"].double()).exp()
    inside = torch.minimum(ratio * a, ratio.clamp(1 - CLIP, 1 + CLIP) * a)
    cut = torch.where(a >= 0, ratio > 1 + CLIP, ratio < 1 - CLIP)
    c = torch.where(cut, 0.0, -a * ratio)
    each, kl = -inside, torch.zeros_like(logp)
    if s["reference"] is not None:
        d = s["reference"].double() - logp
        kl = torch.expm1(d) - d
        each = each + KL * kl
        c = c - KL * torch.expm1(d)
    return {"loss": (w * each).sum().float(), "logp": logp.float(), "kl": (w * kl).sum().float(), "clipped": (w * cut).sum().float(),
            "gradient": _plain_gradient(s, p, torch.where(counts, w * c, 0.0))}


def _plain_preference(s):
    case = s["case"]
    logp, p, counts = _plain_rows(s)
    owner, n = _owner(s), 2 * case["pairs"]
    zero = torch.zeros(n + 1, dtype=torch.float64, device="cuda")
    sums, held = zero.index_add(0, owner, logp)[:n], zero.index_add(0, owner, counts.double())[:n].clamp_min(1)
    each = 1 / held if case["average"] else torch.ones_like(held)
    rewards = BETA * (sums * each - s["reference"].double())
    h = rewards[: n // 2] - rewards[n // 2:]
    up, down = torch.log1p(torch.exp(-h.abs())) + (-h).clamp_min(0), torch.log1p(torch.exp(-h.abs())) + h.clamp_min(0)     # -log sigmoid(+-h)
    loss = ((1 - case["smoothing"]) * up + case["smoothing"] * down).mean()
    slope = (1 / (1 + torch.exp(-h)) - (1 - case["smoothing"])) * BETA / case["pairs"]
    c = torch.cat([torch.cat([slope, -slope]) * each, zero[:1]])[owner]
    return {"loss": loss.float(), "chosen": rewards[: n // 2].float(), "rejected": rewards[n // 2:].float(),
            "gradient": _plain_gradient(s, p, torch.where(counts, c, 0.0))}


def _plain_logprobs(s):
    logp, p, counts = _plain_rows(s)
    out = {"logp": logp.float()}
    if s["case"]["grad"]:
        out["gradient"] = _plain_gradient(s, p, torch.where(counts, s["upstream"], 0.0))
    return out


# ------------------------------------------------------------------------------------------------------------------ run
def run(state):
    case = state["case"]
    if not own:
        return {"adamw": _plain_adamw, "logprobs": _plain_logprobs, "policy": _plain_policy, "preference": _plain_preference}[case["op"]](state)
    if case["op"] == "adamw":
        opt = state["opt"]
        opt.step()
        out = {"p": state["p"], "norm": opt.grad_norm}
        if case["bits"] == 32 and case["type"] == "float32":
            out.update(opt.flat_state())
        else:
            out.update(opt.unpack_state(dtype=torch.bfloat16 if case["bits"] == 8 else torch.float32))
        return out
    from repsurf_amd import objectives
    logits, target = state["logits"], state["target"]
    if case["op"] == "logprobs":
        logp = objectives.token_logprobs(logits, target)
        return {"logp": logp, "gradient": torch.autograd.grad(logp, logits, state["upstream"])[0] if case["grad"] else None}
    if case["op"] == "policy":
        r = objectives.policy_loss(logits, target, state["old"], state["advantages"], ref_logp=state["reference"], offset=state["offset"],
                                   clip=(CLIP, CLIP), kl_coef=KL, reduction=case["reduction"])
        return {"loss": r.loss, "logp": r.logp, "kl": r.kl, "clipped": r.clip_fraction, "gradient": torch.autograd.grad(r.loss, logits)[0]}
    r = objectives.preference_loss(logits, target, state["offset"], state["reference"], beta=BETA, label_smoothing=case["smoothing"],
                                   average=case["average"])
    return {"loss": r.loss, "chosen": r.chosen_rewards, "rejected": r.rejected_rewards, "gradient": torch.autograd.grad(r.loss, logits)[0]}


# ---------------------------------------------------------------------------------------------------------------- exact
def exact(case, seed):
    """The definitions in 64 bits, row by row or block by block."""
    s = prepare(case, seed)
    return _exact_adamw(case, s) if case["op"] == "adamw" else _exact_logits(case, s)


def _exact_state(x, signed, d):
    """the stored value of every element: its neighbours on the grid, the upper one where the dither reaches it"""
    lowest = 13 if signed else 29
    rows = x.view(-1, BLOCK)
    top = torch.floor(torch.log2(rows.abs().amax(1).clamp_min(2.0 ** -126)))
    top = torch.where(torch.exp2(top) > rows.abs().amax(1).clamp_min(2.0 ** -126), top - 1, top)[:, None]
    octave = torch.frexp(rows)[1].double() - 1
    octave = torch.where(rows == 0, top - lowest, torch.maximum(octave, top - lowest))
    units = rows.abs() * torch.exp2(3 - octave)
    below = units.floor()
    goes_up = units - below >= 1 - (d.view(-1, BLOCK).double() + 0.5) / 65536
    kept = below + goes_up
    if not signed:
        kept = torch.where((rows > 0) & (kept == 0), 1.0, kept)
    return (torch.sign(rows) * kept * torch.exp2(octave - 3)).view(-1)


def _exact_adamw(case, s):
    t, g, m, v = T0 + 1, s["g"].double(), s["m"].double(), s["v"].double()
    p = s["p"].double()
    out = {"norm": None}
    if case["clip"]:
        norm = torch.linalg.vector_norm(g)
        g *= min(1.0, case["clip"] / (float(norm) + 1e-6))
        out["norm"] = norm
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g ** 2
    p = (1 - LR * DECAY) * p - LR * (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)).sqrt() + EPS)
    out["p"] = p
    if case["type"] != "float32":
        out["master"] = p
    if case["bits"] == 8:
        dm, dv = _dither(s["seed"], t, m.numel())
        m, v = _exact_state(m, True, dm), _exact_state(v, False, dv)
    out.update(exp_avg=m, exp_avg_sq=v)
    return out


def _exact_logits(case, s):
    rows = s["logits"].shape[0]
    counts = (s["target"] >= 0).tolist()
    bounds = [0] + ([rows] if case["op"] == "logprobs" else s["offset"].tolist() + [rows])
    logp = torch.zeros(rows, dtype=torch.float64, device="cuda")
    here = torch.tensor([i for i in range(rows) if counts[i]], device="cuda")
    for part in here.split(512):
        logp[part] = torch.log_softmax(s["logits"][part].double(), 1).gather(1, s["target"][part, None])[:, 0]
    held = [sum(counts[a:b]) for a, b in zip(bounds, bounds[1:])]
    spans = list(zip(bounds, bounds[1:], held))[: len(bounds) - 1 if case["op"] == "logprobs" else len(bounds) - 2]
    c = torch.zeros(rows, dtype=torch.float64, device="cuda")
    if case["op"] == "logprobs":
        out = {"logp": logp}
        if not case["grad"]:
            return out
        c = s["upstream"].double()
    elif case["op"] == "policy":
        w = torch.zeros_like(c)
        for a, b, n in spans:
            w[a:b] = 1.0 / max(1, sum(held[:-1])) if case["reduction"] == "token" else 1.0 / max(1, n) / len(spans)
        w = w * (s["target"] >= 0)
        free = logp.clone().requires_grad_(True)
        with torch.enable_grad():
            ratio, a = torch.exp(free - s["old"].double()), s["advantages"].double()
            loss = (w * -torch.min(ratio * a, torch.clamp(ratio, 1 - CLIP, 1 + CLIP) * a)).sum()
            kl = torch.zeros((), dtype=torch.float64, device="cuda")
            if s["reference"] is not None:
                d = s["reference"].double() - free
                kl = (w * (torch.exp(d) - 1 - d)).sum()
            c, = torch.autograd.grad(loss + KL * kl, free)
        r = ratio.detach()
        cut = ((a > 0) & (r > 1 + CLIP)) | ((a < 0) & (r < 1 - CLIP))
        out = {"loss": (loss + KL * kl).detach(), "logp": logp, "kl": kl.detach(), "clipped": (w * cut).sum()}
    else:
        free = logp.clone().requires_grad_(True)
        with torch.enable_grad():
            each = torch.stack([free[a:b].sum() / (max(1, n) if case["average"] else 1) for a, b, n in spans])
            rewards = BETA * (each - s["reference"].double())
            chosen, rejected = rewards.chunk(2)
            h = chosen - rejected
            ls = torch.nn.functional.logsigmoid
            loss = -((1 - case["smoothing"]) * ls(h) + case["smoothing"] * ls(-h)).mean()
            c, = torch.autograd.grad(loss, free)
        c = c * (s["target"] >= 0)
        out = {"loss": loss.detach(), "chosen": chosen.detach(), "rejected": rejected.detach()}
    g = torch.zeros(rows, case["classes"], dtype=torch.float64, device="cuda")
    for part in here.split(512):
        x = -torch.softmax(s["logits"][part].double(), 1)
        x[torch.arange(part.numel(), device="cuda"), s["target"][part]] += 1
        g[part] = c[part, None] * x
    out["gradient"] = g
    return out
