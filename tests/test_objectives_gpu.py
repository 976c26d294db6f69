"""repsurf_amd.objectives (csrc/logits.hip) against their formulas in 64 bits (torch on the CPU, autograd for the gradients).

Tolerances, u = 2^-24.  exp(x - M) is exp2 of a product: the difference, the constant and the product are three roundings, each u |x - M| of the
exponent, the instruction one unit (2 u): (3 |x - M| + 2) u relative.  Sums of 8 add three roundings, the rest is fp64: log p is off by
    L = (3 D + 6) u,  D = sum of p |x - M|,   and by u |log p| more where it is stored in fp32.
A gradient c ([j = y] - p_j): p_j's exponential, the sum, its inverse, the product and the fma: |c| p_j (3 |x_j - M| + 2 + 3 D + 6 + 4) u, plus c's own
error, plus half a step of the type it is stored in (u for fp32, 2^-8 for bf16, 2^-11 for fp16, and fp16's 2^-25 at the bottom)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -125, torch.bfloat16: 2.0 ** -125, torch.float16: 2.0 ** -25}
IGN = -100


def logits_of(rows, classes, dtype, seed=0, pad=0, shift=0, scale=2.0):
    """on the device; a pitch of its own and an address off by `shift` elements"""
    g = torch.Generator().manual_seed(seed)
    flat = torch.zeros(rows * (classes + pad) + shift + 8, dtype=dtype)
    z = flat[shift:shift + rows * (classes + pad)].view(rows, classes + pad)[:, :classes]
    z.copy_((torch.randn(rows, classes, generator=g) * scale).to(dtype))
    flat = flat.cuda()
    return flat[shift:shift + rows * (classes + pad)].view(rows, classes + pad)[:, :classes]


def targets_of(rows, classes, seed=0, ignored=0.2):
    g = torch.Generator().manual_seed(100 + seed)
    y = torch.randint(0, classes, (rows,), generator=g)
    y[torch.rand(rows, generator=g) < ignored] = IGN
    return y


class Ref:
    """fp64 leaves, log-probabilities of the targets (0 where a row does not count) and the bounds above"""

    def __init__(self, z, y, behind=None):
        self.z = z.detach().double().cpu().requires_grad_(True)
        rows = torch.arange(len(y))
        self.counts = (y != IGN) & (rows < (len(y) if behind is None else behind))
        safe = torch.where(self.counts[:, None], self.z, torch.zeros_like(self.z))
        lp = torch.log_softmax(safe, 1)
        self.logp = torch.where(self.counts, lp.gather(1, y.clamp_min(0)[:, None])[:, 0], torch.zeros(len(y), dtype=torch.float64))
        with torch.no_grad():
            self.p = lp.exp()
            off = (safe - safe.amax(1, keepdim=True)).abs()
            self.off = torch.where(torch.isfinite(off), off, torch.zeros_like(off))
            self.D = (self.p * self.off).sum(1)
            self.L = (3 * self.D + 6) * U

    def check_logp(self, got):
        want = self.logp.detach()
        assert got.dtype == torch.float32
        assert ((got.detach().double().cpu() - want).abs() <= self.L + U * want.abs()).all()

    def check_grad(self, got, want, dtype, c, dc):
        """c, dc per row: the coefficient and what it may be off"""
        assert got.dtype == dtype and got.shape == want.shape
        c, dc = c.abs()[:, None], dc[:, None]
        tol = c * self.p * (3 * self.off + 12 + 3 * self.D[:, None]) * U + dc * (self.p + (want != 0) * 1.0) + want.abs() * (HALF[dtype] + 2 * U) + TINY[dtype]
        d = (got.double().cpu() - want).abs()
        assert (d <= tol).all(), (d / tol).max()
        assert (got.cpu()[~self.counts] == 0).all()


SIZES = [(1, 1), (7, 1), (5, 2), (300, 13), (9, 40), (64, 64), (33, 65), (17, 255), (6, 1000), (3, 1024), (5, 1025), (4, 4099), (2, 16384), (3, 16385),
         (2, 50001), (1, 131072), (2, 140003)]


@pytest.mark.parametrize("rows,classes", SIZES)
@pytest.mark.parametrize("dtype", list(HALF))
def test_token_logprobs(rows, classes, dtype):
    from repsurf_amd import objectives
    for pad, shift in ((0, 0), (3, 1)):
        z = logits_of(rows, classes, dtype, seed=rows + classes, pad=pad, shift=shift).requires_grad_(True)
        y = targets_of(rows, classes, seed=classes, ignored=0.0 if rows == 1 else 0.2)
        ref = Ref(z, y)
        got = objectives.token_logprobs(z, y.cuda())
        ref.check_logp(got)
        up = torch.randn(rows, generator=torch.Generator().manual_seed(1))
        g, = torch.autograd.grad(got, z, up.cuda())
        want, = torch.autograd.grad(ref.logp, ref.z, up.double())
        ref.check_grad(g, want, dtype, up.double(), torch.zeros(rows, dtype=torch.float64))
        with torch.no_grad():
            assert torch.equal(objectives.token_logprobs(z, y.cuda()), got)


LENGTHS = [[5], [0, 3, 0, 7], [1, 1], [40, 0, 17, 33, 2, 64], [100, 3, 50, 51]]


def ends(lengths):
    return torch.tensor(lengths).cumsum(0).to(torch.int32).cuda()


@pytest.mark.parametrize("lengths", LENGTHS)
@pytest.mark.parametrize("classes,dtype", [(13, torch.float32), (1500, torch.bfloat16)])
@pytest.mark.parametrize("average", [False, True])
def test_sequence_logprobs(lengths, classes, dtype, average):
    from repsurf_amd import objectives
    n, rows = sum(lengths), sum(lengths) + 5
    z = logits_of(rows, classes, dtype, seed=n).requires_grad_(True)
    y = targets_of(rows, classes, seed=n)
    ref = Ref(z, y, behind=n)
    got = objectives.sequence_logprobs(z, y.cuda(), ends(lengths), average=average)
    parts, counts, bound = ref.logp.split(lengths + [5])[:-1], ref.counts.split(lengths + [5])[:-1], ref.L.split(lengths + [5])[:-1]
    k = torch.tensor([1.0 / max(1, int(c.sum())) if average else 1.0 for c in counts], dtype=torch.float64)
    want = torch.stack([p.sum() for p in parts]) * k
    tol = torch.stack([(b * c).sum() for b, c in zip(bound, counts)]) * k + U * want.detach().abs()
    assert ((got.detach().double().cpu() - want.detach()).abs() <= tol).all()
    up = torch.randn(len(lengths), generator=torch.Generator().manual_seed(2))
    g, = torch.autograd.grad(got, z, up.cuda())
    w, = torch.autograd.grad(want, ref.z, up.double())
    c = torch.cat([(up[i].double() * k[i]).expand(m) for i, m in enumerate(lengths)] + [torch.zeros(5, dtype=torch.float64)])
    ref.check_grad(g, w, dtype, c, 3 * U * c.abs())


@pytest.mark.parametrize("lengths", [[1, 1], [0, 3, 0, 7], [40, 0, 17, 33, 2, 64], [100, 3, 50, 51], [2] * 600])
@pytest.mark.parametrize("classes,dtype", [(13, torch.float32), (1500, torch.bfloat16), (20001, torch.float16)])
@pytest.mark.parametrize("smoothing,average", [(0.0, False), (0.1, True)])
def test_preference_loss(lengths, classes, dtype, smoothing, average):
    from repsurf_amd import objectives
    if classes > 2000 and sum(lengths) > 300:
        lengths = lengths[:20]
    n, rows, b, beta = sum(lengths), sum(lengths) + 3, len(lengths), 0.1
    z = logits_of(rows, classes, dtype, seed=n, pad=1).requires_grad_(True)
    y = targets_of(rows, classes, seed=n)
    ref = Ref(z, y, behind=n)
    counts = ref.counts.split(lengths + [3])[:-1]
    k = torch.tensor([1.0 / max(1, int(c.sum())) if average else 1.0 for c in counts], dtype=torch.float64)
    sums = torch.stack([p.sum() for p in ref.logp.split(lengths + [3])[:-1]]) * k
    other = (sums.detach() + torch.randn(b, generator=torch.Generator().manual_seed(4)) * 3).float()
    r = beta * (sums - other.double())
    h = r[: b // 2] - r[b // 2:]
    ls = torch.nn.functional.logsigmoid
    want = -((1 - smoothing) * ls(h) + smoothing * ls(-h)).mean()
    got = objectives.preference_loss(z, y.cuda(), ends(lengths), other.cuda(), beta=beta, label_smoothing=smoothing, average=average)
    dr = beta * torch.stack([(x * c).sum() for x, c in zip(ref.L.split(lengths + [3])[:-1], counts)]) * k       # what a reward may be off
    rewards = torch.cat([got.chosen_rewards, got.rejected_rewards]).double().cpu()
    assert ((rewards - r.detach()).abs() <= dr + U * r.detach().abs()).all()
    dh = dr[: b // 2] + dr[b // 2:]                                                    # d loss / dh is at most 1
    assert abs(float(got.loss) - float(want)) <= float(dh.mean()) + 2 * U * abs(float(want))
    scale = 3.0
    g, = torch.autograd.grad(got.loss * scale, z)
    w, = torch.autograd.grad(want * scale, ref.z, retain_graph=True)
    coef, = torch.autograd.grad(want * scale, sums)
    spread = lambda t: torch.cat([t[i].expand(m) for i, m in enumerate(lengths)] + [torch.zeros(3, dtype=torch.float64)])      # noqa: E731
    slope_off = scale * beta * 2 / b * k * torch.cat([dh, dh]) / 4                      # sigmoid's slope is at most 1 / 4
    c = spread(coef * k)
    ref.check_grad(g, w, dtype, c, spread(slope_off) + 4 * U * c.abs())
    assert got.loss.requires_grad and not got.chosen_rewards.requires_grad


RATIOS = torch.tensor([0.5, 0.79, 0.81, 0.95, 1.0, 1.1, 1.19, 1.21, 1.5, 2.5], dtype=torch.float64)      # none within 1e-3 of a border 0.8, 1.2


def policy_case(lengths, behind, classes, dtype, seed, pad=0):
    rows = sum(lengths) + behind
    g = torch.Generator().manual_seed(seed)
    z = logits_of(rows, classes, dtype, seed=seed, pad=pad).requires_grad_(True)
    y = targets_of(rows, classes, seed=seed)
    ref = Ref(z, y, behind=sum(lengths))
    ratio = RATIOS[torch.randint(0, len(RATIOS), (rows,), generator=g)]
    old = (ref.logp.detach() - ratio.log()).float()
    adv = torch.randn(rows, generator=g)
    other = (ref.logp.detach() + torch.randn(rows, generator=g) * 0.3).float()
    return z, y, ref, old, adv, other


def policy_want(ref, lengths, behind, old, adv, other, clip, kl_coef, reduction):
    rows = len(old)
    per = [c.sum().clamp_min(1) for c in ref.counts.split(lengths + [behind])]
    if reduction == "token":
        w = torch.full((rows,), 1.0 / max(1, int(ref.counts.sum())), dtype=torch.float64)
    else:
        w = torch.cat([torch.full((m,), 1.0 / float(n) / len(lengths), dtype=torch.float64) for m, n in zip(lengths + [behind], per)])
    w = w * ref.counts
    x = ref.logp.detach().clone().requires_grad_(True)
    r, a = torch.exp(x - old.double()), adv.double()
    each = -torch.minimum(r * a, r.clamp(1 - clip[0], 1 + clip[1]) * a)
    kl = torch.zeros_like(x)
    if other is not None:
        d = other.double() - x
        kl = torch.exp(d) - 1 - d
    loss = (w * (each + kl_coef * kl)).sum()
    cut = torch.where(a >= 0, r > 1 + clip[1], r < 1 - clip[0])
    c, = torch.autograd.grad(loss, x)
    sens = w * (r.detach() * a.abs() + (kl_coef * torch.exp(other.double() - x.detach()) if other is not None else 0))      # of each to log p, and of c
    return float(loss), float((w * kl).sum()), float((w * cut).sum()), c, sens


@pytest.mark.parametrize("lengths,behind", [([6], 0), ([40, 0, 17, 33, 2, 64], 7), ([300, 200], 0), ([1], 3)])
@pytest.mark.parametrize("classes,dtype", [(2, torch.float32), (13, torch.float32), (40, torch.float16), (1100, torch.bfloat16), (20001, torch.float32)])
@pytest.mark.parametrize("reduction,use_ref,clip", [("token", True, (0.2, 0.2)), ("sequence", False, (0.2, 0.4)), ("sequence", True, (0.2, 0.2))])
def test_policy_loss(lengths, behind, classes, dtype, reduction, use_ref, clip):
    from repsurf_amd import objectives
    z, y, ref, old, adv, other = policy_case(lengths, behind, classes, dtype, 3, pad=2)
    kl_coef = 0.05
    other = other if use_ref else None
    loss, kl, cut, c, sens = policy_want(ref, lengths, behind, old, adv, other, clip, kl_coef, reduction)
    args = (z, y.cuda(), old.cuda(), adv.cuda())
    kw = dict(ref_logp=None if other is None else other.cuda(), offset=ends(lengths), clip=clip, kl_coef=kl_coef, reduction=reduction)
    got = objectives.policy_loss(*args, **kw)
    ref.check_logp(got.logp)
    dl = float((sens * ref.L).sum())
    assert abs(float(got.loss) - loss) <= 1.01 * dl + U * abs(loss)
    wide = float((sens / kl_coef * ref.L).sum())
    assert abs(float(got.kl) - kl) <= 1.01 * wide + U * kl
    assert abs(float(got.clip_fraction) - cut) <= 2 * U * cut
    want, = torch.autograd.grad(ref.logp, ref.z, c, retain_graph=True)
    dc = 1.01 * sens * ref.L + U * c.abs()
    unit, = torch.autograd.grad(got.loss, z, retain_graph=True)
    ref.check_grad(unit, want, dtype, c, dc)
    again, = torch.autograd.grad(got.loss, z, retain_graph=True)           # the gradient formed with the loss was handed out: computed again
    ref.check_grad(again, want, dtype, c, dc)
    scaled, = torch.autograd.grad(got.loss * 0.3, z)
    ref.check_grad(scaled, want * 0.3, dtype, c * 0.3, 0.3 * dc + 2 * U * c.abs())
    fresh, = torch.autograd.grad(objectives.policy_loss(*args, **kw).loss * 0.3, z)
    assert torch.equal(fresh, scaled)
    with torch.no_grad():
        still = objectives.policy_loss(*args, **kw)
    assert not still.loss.requires_grad and all(torch.equal(a, b) for a, b in zip(still, got))      # the same bits, with a gradient or without


@pytest.mark.parametrize("classes", [8, 16, 31, 64, 127, 250, 512, 1023, 2047, 4095, 4097, 5119, 5121, 9215, 9217, 10239, 16384, 17409, 18433, 33000, 34816, 50001, 51201,
                                     67583, 69633, 131071, 135169])
@pytest.mark.parametrize("dtype", list(HALF))
def test_policy_loss_at_every_length_of_row(classes, dtype):
    """260 rows (more than the few that are cut over many workgroups), on both sides of the lengths where the kernels change: every
    log-probability in 64 bits on the device, the gradients of six rows as above"""
    from repsurf_amd import objectives
    rows = 260
    z = logits_of(rows, classes, dtype, seed=classes, pad=1 if classes % 2 else 0).requires_grad_(True)
    y = targets_of(rows, classes, seed=classes, ignored=0.1)
    counts = (y != IGN)
    n = int(counts.sum())
    x = z.detach().double()
    lp = torch.log_softmax(x, 1)
    want = torch.where(counts.cuda(), lp.gather(1, y.clamp_min(0).cuda()[:, None])[:, 0], 0.0)
    bound = (3 * (lp.exp() * (x - x.amax(1, keepdim=True)).abs()).sum(1) + 6) * U
    ratio = RATIOS[torch.randint(0, len(RATIOS), (rows,), generator=torch.Generator().manual_seed(1))].cuda()
    old = (want - ratio.log()).float()
    adv = torch.randn(rows, generator=torch.Generator().manual_seed(2)).cuda()
    got = objectives.policy_loss(z, y.cuda(), old, adv)
    assert ((got.logp.double() - want).abs() <= bound + U * want.abs()).all()
    r, a = torch.exp(want - old.double()), adv.double()
    each = torch.where(counts.cuda(), -torch.minimum(r * a, r.clamp(0.8, 1.2) * a), 0.0)
    assert abs(float(got.loss.detach()) - float(each.sum() / n)) <= 1.01 * float((r * a.abs() * bound * counts.cuda()).sum() / n) + 2 * U * abs(float(each.sum() / n))
    g, = torch.autograd.grad(got.loss, z)
    assert (g[~counts.cuda()] == 0).all()
    pick = [i for i in (0, 1, 2, 100, 255, 256, 258, 259) if counts[i]]
    ref = Ref(z.detach()[pick], y[pick])
    cut = torch.where(a >= 0, r > 1.2, r < 0.8)
    c = torch.where(cut, 0.0, -a * r / n)[pick].cpu()
    w, = torch.autograd.grad(ref.logp, ref.z, c)
    ref.check_grad(g[pick], w, dtype, c, 1.01 * c.abs() * ref.L + U * c.abs())
    alone = objectives.token_logprobs(z, y.cuda())
    assert ((alone.detach().double() - want).abs() <= bound + U * want.abs()).all()
    up = torch.randn(rows, generator=torch.Generator().manual_seed(3))
    g, = torch.autograd.grad(alone, z, up.cuda())
    ref = Ref(z.detach()[pick], y[pick])
    w, = torch.autograd.grad(ref.logp, ref.z, up[pick].double())
    ref.check_grad(g[pick], w, dtype, up[pick].double(), torch.zeros(len(pick), dtype=torch.float64))
    assert (g[~counts.cuda()] == 0).all()


def test_policy_advantages_per_sequence_and_unit_gradient():
    from repsurf_amd import head, objectives
    lengths = [40, 0, 17, 33]
    z, y, ref, old, _, _ = policy_case(lengths, 4, 13, torch.float32, 5)
    a = torch.randn(4, 1, generator=torch.Generator().manual_seed(8))
    rows = torch.cat([a[i].expand(m) for i, m in enumerate(lengths)] + [torch.zeros(4)])
    one = objectives.policy_loss(z, y.cuda(), old.cuda(), a.cuda(), offset=ends(lengths))
    two = objectives.policy_loss(z, y.cuda(), old.cuda(), rows.cuda(), offset=ends(lengths))
    assert torch.equal(one.loss, two.loss)
    one.loss.backward(head.unit_gradient(z.device))
    g, = torch.autograd.grad(two.loss, z)
    assert torch.equal(z.grad, g)
    loss = objectives.policy_loss(z, y.cuda(), old.cuda(), rows.cuda(), offset=ends(lengths)).loss
    loss /= 4                                                               # in place, as accumulation over micro-batches writes it
    q, = torch.autograd.grad(loss, z)
    assert torch.equal(q, g / 4)


@pytest.mark.parametrize("classes", [13, 1500])
def test_gradients_are_those_of_differences(classes):
    """(L(z + h e) - L(z - h e)) / 2 h of the losses that the kernels return, e a random direction, against <gradient, e>: off by what
    the same quotient in 64 bits is off its derivative, and by the losses' own errors over h"""
    from repsurf_amd import objectives
    lengths, h = [30, 20], 2.0 ** -6
    z, y, ref, old, adv, other = policy_case(lengths, 2, classes, torch.float32, 21)
    e = (torch.randn(z.shape, generator=torch.Generator().manual_seed(9)) / math.sqrt(classes) * 2 ** 8).round() / 2 ** 8
    pref = torch.tensor([-60.0, -50.0])

    def policy(zz):
        return objectives.policy_loss(zz, y.cuda(), old.cuda(), adv.cuda(), ref_logp=other.cuda(), offset=ends(lengths), kl_coef=0.05).loss

    def preference(zz):
        return objectives.preference_loss(zz, y.cuda(), ends(lengths), pref.cuda()).loss

    def policy64(zz):
        r = Ref(zz, y, behind=50)
        return policy_want(r, lengths, 2, old, adv, other, (0.2, 0.2), 0.05, "token")[0]

    def preference64(zz):
        s = torch.stack([x.sum() for x in Ref(zz, y, behind=50).logp.split([30, 20, 2])[:-1]])
        d = 0.1 * (s - pref.double())
        return float(-torch.nn.functional.logsigmoid(d[0] - d[1]))

    for f, f64, sens in ((policy, policy64, 3.0), (preference, preference64, 0.1 * 50)):
        g, = torch.autograd.grad(f(z), z)
        slope = float((g.double().cpu() * e).sum())
        up, down = (z.detach() + h * e.cuda()), (z.detach() - h * e.cuda())
        quotient = (float(f(up)) - float(f(down))) / (2 * h)
        exact = (f64(up) - f64(down)) / (2 * h)
        assert abs(quotient - exact) <= (sens * float(ref.L.max()) + U * abs(f64(up))) / h
        z64 = z.detach().double()
        small = 2.0 ** -16
        true = (f64(z64 + small * e.cuda()) - f64(z64 - small * e.cuda())) / (2 * small)
        assert abs(slope - quotient) <= 1.5 * abs(true - exact) + 2 * (sens * float(ref.L.max()) + U * abs(f64(up))) / h + 1e-6 * abs(true)


@pytest.mark.parametrize("classes", [13, 1500, 20001])
@pytest.mark.parametrize("dtype", list(HALF))
def test_masked_and_broken_rows_stay_with_themselves(classes, dtype):
    from repsurf_amd import head, objectives
    rows = 24
    z = logits_of(rows, classes, dtype, seed=2)
    y = targets_of(rows, classes, seed=2, ignored=0.0)
    low = torch.finfo(dtype).min
    z[1, :] = float("nan"); z[2, 3:] = float("inf"); y[1] = y[2] = IGN            # ignored rows may hold anything
    z[3, : classes // 2] = -math.inf; y[3] = classes - 1                           # a masked half
    z[4, :] = -math.inf; z[4, 1] = 2.0; y[4] = 1                                   # one class left: certainty
    z[5, : classes // 2] = low; y[5] = classes - 1                                 # masked by the type's lowest value
    z[6, :] = low                                                                  # nothing but that: uniform
    z[7, :] = torch.finfo(dtype).max
    z[8, 0] = -math.inf; y[8] = 0                                                  # an impossible target
    z[9, :] = -math.inf                                                            # nothing left
    z[10, 2] = float("nan")
    z[11, 1] = float("inf"); y[11] = 0
    y[12], y[13] = classes, -7                                                     # no classes
    z.requires_grad_(True)
    before = head.bad_label_count(z.device)
    good = [i for i in range(rows) if i not in (1, 2, 8, 9, 10, 11, 12, 13)]
    ref = Ref(z.detach()[good], y[good])
    logp = objectives.token_logprobs(z, y.cuda())
    assert head.bad_label_count(z.device) - before == 2
    ref.check_logp(logp[good])
    got = logp.detach().cpu()
    assert got[1] == 0 and got[2] == 0 and got[4] == 0 and got[8] == -math.inf and torch.isnan(got[[9, 10, 11, 12, 13]]).all()
    up = torch.randn(rows, generator=torch.Generator().manual_seed(1))
    g, = torch.autograd.grad(logp, z, up.cuda())
    w, = torch.autograd.grad(ref.logp, ref.z, up[good].double())
    ref.check_grad(g[good], w, dtype, up[good].double(), torch.zeros(len(good), dtype=torch.float64))
    gc = g.cpu().float()
    assert (gc[1] == 0).all() and (gc[2] == 0).all() and torch.isfinite(gc[8]).all() and torch.isnan(gc[[9, 10, 12, 13]]).all()
    old, adv = torch.full((rows,), -2.0), torch.ones(rows)
    y[[8, 9, 10, 11, 12, 13]] = IGN
    out = objectives.policy_loss(z, y.cuda(), old.cuda(), adv.cuda())
    p, = torch.autograd.grad(out.loss, z)
    assert torch.isfinite(out.loss) and (p.cpu()[[1, 2, 8, 9, 10, 11, 12, 13]] == 0).all() and torch.isfinite(p).all()
    y[12] = classes
    out = objectives.policy_loss(z, y.cuda(), old.cuda(), adv.cuda())
    p2, = torch.autograd.grad(out.loss, z)
    keep = [i for i in range(rows) if i != 12]
    assert torch.isnan(out.loss) and torch.isnan(p2[12]).all() and torch.isfinite(p2[keep]).all()


def test_nothing_counts():
    from repsurf_amd import objectives
    for rows in (0, 9):
        z = torch.full((rows, 13), float("nan"), device="cuda", requires_grad=True)
        y = torch.full((rows,), IGN, device="cuda")
        zero = torch.zeros(rows, device="cuda")
        off = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
        for reduction in ("token", "sequence"):
            out = objectives.policy_loss(z, y, zero, zero, ref_logp=zero, offset=off, kl_coef=0.1, reduction=reduction)
            g, = torch.autograd.grad(out.loss, z)
            assert float(out.loss) == 0 and float(out.kl) == 0 and float(out.clip_fraction) == 0 and (g == 0).all() and g.shape == z.shape
        out = objectives.preference_loss(z, y, off, torch.zeros(2, device="cuda"))
        g, = torch.autograd.grad(out.loss, z)
        assert abs(float(out.loss) - math.log(2)) <= U and (g == 0).all()
        assert (objectives.token_logprobs(z, y) == 0).all() and (objectives.sequence_logprobs(z, y, off) == 0).all()
        g, = torch.autograd.grad(objectives.token_logprobs(z, y).sum(), z)
        assert (g == 0).all() and g.shape == z.shape


def test_layouts_types_and_refusals_on_the_device():
    from repsurf_amd import objectives
    z = logits_of(50, 13, torch.float32)
    y = targets_of(50, 13).cuda()
    want = objectives.token_logprobs(z, y)
    t = z.t().contiguous().t()                                     # columns first
    assert torch.equal(objectives.token_logprobs(t, y), want)
    assert torch.equal(objectives.token_logprobs(z, y.to(torch.int32)), want)
    wide = torch.stack([y, y], 1)[:, 0]                            # strided targets
    assert torch.equal(objectives.token_logprobs(z, wide), want)
    row = z[:1].expand(50, 13)                                     # a row pitch of nothing
    assert torch.equal(objectives.token_logprobs(row, y), objectives.token_logprobs(row.contiguous(), y))
    assert torch.equal(objectives.sequence_logprobs(z, y, torch.tensor([20, 50]).cuda()), objectives.sequence_logprobs(z, y, ends([20, 30])))
    zero = torch.zeros(50, device="cuda")
    for call in (lambda: objectives.preference_loss(z, y, ends([10, 20, 20]), zero[:3]), lambda: objectives.preference_loss(z, y, ends([10, 40]), zero[:3]),
                 lambda: objectives.preference_loss(z, y, ends([10, 40]), zero[:2], label_smoothing=0.7),
                 lambda: objectives.policy_loss(z, y, zero, zero, reduction="sequence"), lambda: objectives.policy_loss(z, y, zero, zero, reduction="none"),
                 lambda: objectives.policy_loss(z, y, zero[:3], zero), lambda: objectives.policy_loss(z, y, zero, zero[:2, None]),
                 lambda: objectives.policy_loss(z, y, zero, zero, clip=(-0.1, 0.1)), lambda: objectives.policy_loss(z, y, zero, zero, ref_logp=zero[:1]),
                 lambda: objectives.policy_loss(z, y, zero.cpu(), zero), lambda: objectives.token_logprobs(z, y.cpu()),
                 lambda: objectives.policy_loss(z, y, zero, zero[:3, None], offset=ends([20, 30]))):
        with pytest.raises(ValueError):
            call()
    q = z.clone().requires_grad_(True)
    g, = torch.autograd.grad(objectives.token_logprobs(q, y).sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()                                         # differentiable once


def test_rows_whose_offsets_pass_32_bits():
    """70001 x 65536 logits in bf16: 4.6e9 elements; the first, the middle and the last rows"""
    from repsurf_amd import objectives
    rows, classes = 70001, 65536
    z = torch.empty(rows, classes, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(0))
    y = torch.randint(0, classes, (rows,), generator=torch.Generator().manual_seed(0))
    pick = torch.tensor([0, 1, 32767, 32768, 65535, 65536, rows - 1])
    up = torch.zeros(rows)
    up[pick] = torch.randn(len(pick), generator=torch.Generator().manual_seed(1))
    z.requires_grad_(True)
    logp = objectives.token_logprobs(z, y.cuda())
    g, = torch.autograd.grad(logp, z, up.cuda())
    ref = Ref(z.detach()[pick.cuda()], y[pick])
    ref.check_logp(logp[pick.cuda()])
    w, = torch.autograd.grad(ref.logp, ref.z, up[pick].double())
    ref.check_grad(g[pick.cuda()], w, torch.bfloat16, up[pick].double(), torch.zeros(len(pick), dtype=torch.float64))


@pytest.mark.parametrize("classes,dtype", [(13, torch.float32), (5003, torch.bfloat16), (40001, torch.bfloat16)])
def test_captured_replays_are_the_eager_calls(classes, dtype):
    """forward and backward of the two losses in one graph, four replays on new data with eager calls and synchronisations between them"""
    from repsurf_amd import objectives
    lengths = [30, 0, 20, 14]
    z, y, _, old, adv, other = policy_case(lengths, 3, classes, dtype, 31)
    off, y = ends(lengths), y.cuda()
    pref = torch.tensor([-30.0, 0.0, -40.0, -20.0]).cuda()
    old, adv, other = old.cuda(), adv.cuda(), other.cuda()

    def run(zz, oo, aa):
        a = objectives.policy_loss(zz, y, oo, aa, ref_logp=other, offset=off, kl_coef=0.05, reduction="sequence")
        b = objectives.preference_loss(zz, y, off, pref)
        g, = torch.autograd.grad(a.loss + 0.5 * b.loss, zz)
        return [a.loss, a.logp, a.kl, a.clip_fraction, b.loss, b.chosen_rewards, b.rejected_rewards, g]

    live = run(z, old, adv)                               # an eager result of the same leaves stays alive over the capture
    sz, so, sa = z.detach().clone().requires_grad_(True), old.clone(), adv.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            run(sz, so, sa)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(sz, so, sa)
    for k in range(4):
        with torch.no_grad():
            sz.copy_(logits_of(z.shape[0], classes, dtype, seed=50 + k))
            sa.copy_(torch.randn(len(adv), generator=torch.Generator().manual_seed(k)))
        graph.replay()
        torch.cuda.synchronize()
        eager = run(sz.detach().clone().requires_grad_(True), so, sa)
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(out, eager)):
            assert torch.equal(a, b), (k, i)
    assert torch.isfinite(live[0])


def test_saved_tensors_that_a_hook_moves():
    """the backward passes read what autograd hands back, not where the forward pass found it"""
    from repsurf_amd import objectives
    z, y, _, old, adv, _ = policy_case([30, 20], 2, 1500, torch.bfloat16, 61)
    y, old, adv, off = y.cuda(), old.cuda(), adv.cuda(), ends([30, 20])
    calls = (lambda: objectives.token_logprobs(z, y).sum(), lambda: objectives.sequence_logprobs(z, y, off, average=True).sum(),
             lambda: objectives.preference_loss(z, y, off, old[:2]).loss, lambda: objectives.policy_loss(z, y, old, adv, offset=off).loss * 0.5)
    want = [torch.autograd.grad(f(), z)[0] for f in calls]
    for f, w in zip(calls, want):
        with torch.autograd.graph.save_on_cpu():
            loss = f()
        junk = [torch.full((52, 1500), 7.0, device="cuda") for _ in range(4)]
        assert torch.equal(torch.autograd.grad(loss, z)[0], w) and len(junk) == 4


def test_two_streams_at_once():
    from repsurf_amd import objectives
    cases = [policy_case([300, 200], 5, c, torch.bfloat16, 41 + c) for c in (600, 30001)]
    dev = [[t.cuda() for t in (c[1], c[3], c[4], c[5])] for c in cases]

    def run(i):
        y, old, adv, other = dev[i]
        o = objectives.policy_loss(cases[i][0], y, old, adv, ref_logp=other, kl_coef=0.1)
        return o.loss, torch.autograd.grad(o.loss, cases[i][0])[0]

    want = [run(0), run(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        got = []
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append(run(i))
        torch.cuda.synchronize()
        for (a, b), (c, d) in zip(want, got):
            assert torch.equal(a, c) and torch.equal(b, d)


def test_a_policy_update_of_a_point_classifier():
    """Scores of the old and the reference policy, the loss through the framework's row Linear, AdamW with 8-bit moments and clipping: two
    epochs over a batch.  The first step's gradients against 64 bits -- the weight gradient is a product over 4096 rows whose factors are
    fp32 (or three bf16 parts of them): relative 2^-20 of its norm covers sums of that length -- and the run itself."""
    from repsurf_amd import mlp, objectives
    from repsurf_amd.optim import AdamW
    torch.manual_seed(0)
    rows, width, classes = 4096, 64, 13
    x = torch.randn(rows, width, device="cuda")
    lin = torch.nn.Linear(width, classes).cuda()
    y = torch.randint(0, classes, (rows,), device="cuda")
    off = ends([1000, 2000, 1000])
    with torch.no_grad():
        old = objectives.token_logprobs(mlp.row_linear(x, lin), y)
        other = objectives.token_logprobs(mlp.row_linear(x, lin) * 0.9, y)
    adv = torch.randn(3, 1, device="cuda")
    opt = AdamW(lin.parameters(), lr=1e-2, state_bits=8, max_grad_norm=1.0)
    w, b = lin.weight.detach().double().cpu().requires_grad_(True), lin.bias.detach().double().cpu().requires_grad_(True)
    losses = []
    for epoch in range(2):
        opt.zero_grad()
        out = objectives.policy_loss(mlp.row_linear(x, lin), y, old, adv, ref_logp=other, offset=off, kl_coef=0.1, reduction="sequence")
        out.loss.backward()
        if epoch == 0:
            lp = torch.log_softmax(x.double().cpu() @ w.t() + b, 1).gather(1, y.cpu()[:, None])[:, 0][:4000]
            a = adv.double().cpu().view(3).repeat_interleave(torch.tensor([1000, 2000, 1000]))
            d = other.double().cpu()[:4000] - lp
            each = -torch.exp(lp - old.double().cpu()[:4000]) * a + 0.1 * (torch.exp(d) - 1 - d)
            torch.stack([p.mean() for p in each.split([1000, 2000, 1000])]).mean().backward()
            for got, want in ((lin.weight.grad, w.grad), (lin.bias.grad, b.grad)):
                assert (got.double().cpu() - want).norm() <= 2.0 ** -20 * 64 * want.norm()
        opt.step()
        losses.append(float(out.loss.detach()))
    assert torch.isfinite(torch.tensor(losses)).all() and torch.isfinite(lin.weight).all() and float(opt.grad_norm) > 0
    assert (out.logp - old).abs().max() > 0          # the second epoch's policy is another one


def test_gradients_of_pitched_logits_are_dense():
    """|x - M| stays below 7 and D below 3 on normal numbers: (3 * 7 + 12 + 3 * 3) u = 42 u of a p below 0.9; the coefficient exp(log p + 50) adds
    the error of its exponent, (3 * 3 + 6) u, and its rounding"""
    from repsurf_amd import objectives
    whole = torch.randn(20, 40, device="cuda")
    for z in (whole[:, :13], whole[3:4, :13], whole[:, 5:6], whole[::2, :13], whole[:13, :20].t()):
        z = z.detach().requires_grad_(True)
        rows = z.shape[0]
        y = torch.zeros(rows, dtype=torch.long, device="cuda")
        zero = torch.zeros(rows, device="cuda")
        want = torch.zeros(rows, z.shape[1], dtype=torch.float64)
        want[:, 0] = 1
        want = (want - torch.softmax(z.detach().double().cpu(), 1))
        for f, scale in ((lambda: objectives.token_logprobs(z, y).sum(), 1.0), (lambda: objectives.policy_loss(z, y, zero - 50, zero + 1, clip=(1, 1e30)).loss, None)):
            g, = torch.autograd.grad(f(), z)
            assert g.shape == z.shape
            if scale:
                assert (g.double().cpu() - want).abs().max() <= 40 * U
            else:                                    # -r A averaged: every row's coefficient is -exp(log p + 50) / rows
                c = -torch.exp(torch.log_softmax(z.detach().double().cpu(), 1)[:, :1] + 50) / rows
                assert ((g.double().cpu() - c * want).abs() <= 60 * U * c.abs()).all()
