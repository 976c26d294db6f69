"""repsurf_amd.objectives where a call meets something unusual."""
import math

import pytest
import torch

from tests.test_objectives_gpu import ends, logits_of, targets_of

pytestmark = pytest.mark.gpu


def bits(t):
    return t.view(torch.int32 if t.element_size() == 4 else torch.int16)


# ---- rows behind the last sequence ------------------------------------------------------------------------------------
@pytest.mark.parametrize("classes", [13, 1500, 20001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lengths", [[40, 17], [200, 0, 100]])          # (57 rows of 20001 classes are cut over many workgroups, 300 are not)
@pytest.mark.parametrize("reduction", ["token", "sequence"])
def test_rows_behind_the_last_sequence_may_hold_anything(classes, dtype, lengths, reduction):
    """The same bits as with well-behaved padding, whatever the upstream gradient is and however often it is asked for; and zeros there."""
    from repsurf_amd import head, objectives
    n, behind = sum(lengths), 6
    z = logits_of(n + behind, classes, dtype, seed=classes)
    y = targets_of(n + behind, classes, seed=1, ignored=0.1)
    off = ends(lengths)
    g = torch.Generator().manual_seed(3)
    old, adv = (torch.randn(n + behind, generator=g) - math.log(classes)).cuda(), torch.randn(n + behind, generator=g).cuda()
    y[n:] = torch.arange(behind) % classes
    odd, yo, oo, ao = z.clone(), y.clone(), old.clone(), adv.clone()
    odd[n] = float("nan"); odd[n + 1, 1] = float("inf"); odd[n + 2] = 100.0; odd[n + 3] = torch.finfo(dtype).max; odd[n + 4, :] = -math.inf
    yo[n + 4], yo[n + 5] = -7, classes
    oo[n:], ao[n:] = float("nan"), float("inf")
    before = head.bad_label_count(z.device)

    def run(zz, yy, old_, adv_):
        zz = zz.detach().clone().requires_grad_(True)
        out = objectives.policy_loss(zz, yy.cuda(), old_, adv_, offset=off, reduction=reduction)
        grads = [torch.autograd.grad(out.loss, zz, retain_graph=True)[0] for _ in range(2)]          # handed out, then computed again
        grads.append(torch.autograd.grad(out.loss * 0.3, zz)[0])
        fresh = objectives.policy_loss(zz, yy.cuda(), old_, adv_, offset=off, reduction=reduction)
        grads.append(torch.autograd.grad(fresh.loss * 0.3, zz)[0])
        grads.append(torch.autograd.grad(objectives.sequence_logprobs(zz, yy.cuda(), off).sum(), zz)[0])
        if len(lengths) % 2 == 0:
            grads.append(torch.autograd.grad(objectives.preference_loss(zz, yy.cuda(), off, torch.zeros(len(lengths), device="cuda")).loss, zz)[0])
        return out, grads

    want, clean = run(z, y, old, adv)
    got, grads = run(odd, yo, oo, ao)
    assert head.bad_label_count(z.device) == before
    assert torch.isfinite(want.loss) and torch.equal(want.loss, got.loss) and torch.equal(want.logp, got.logp)
    for i, (a, b) in enumerate(zip(clean, grads)):
        assert (b[n:] == 0).all(), i
        assert torch.equal(bits(a[:n]), bits(b[:n])), i


# ---- an upstream gradient that does not exist -------------------------------------------------------------------------
class Drop(torch.autograd.Function):
    """hands nothing on: its input has no gradient"""

    @staticmethod
    def forward(ctx, x):
        return x.clone()

    @staticmethod
    def backward(ctx, g):
        return None


def small_case(classes=13, seed=7):
    z = logits_of(50, classes, torch.float32, seed=seed)
    y = targets_of(50, classes, seed=seed).cuda()
    g = torch.Generator().manual_seed(seed)
    return z, y, ends([30, 20]), (torch.randn(50, generator=g) - 2).cuda(), torch.randn(50, generator=g).cuda(), torch.tensor([-60.0, -50.0]).cuda()


def losses(z, y, off, old, adv, pref):
    from repsurf_amd import objectives
    return {"token": lambda: objectives.token_logprobs(z, y), "sequence": lambda: objectives.sequence_logprobs(z, y, off, average=True),
            "preference": lambda: objectives.preference_loss(z, y, off, pref).loss, "policy": lambda: objectives.policy_loss(z, y, old, adv, offset=off).loss}


@pytest.mark.parametrize("name", ["token", "sequence", "preference", "policy"])
@pytest.mark.parametrize("unit", [False, True])
def test_no_upstream_gradient_is_no_gradient(name, unit):
    from repsurf_amd import head
    z, *rest = small_case()
    z.requires_grad_(True)
    if unit:
        head.unit_gradient(z.device)
    f = losses(z, *rest)[name]
    assert torch.autograd.grad(Drop.apply(f()).sum(), z, allow_unused=True) == (None,)
    w = torch.randn(z.shape, generator=torch.Generator().manual_seed(1)).cuda()
    g, = torch.autograd.grad(Drop.apply(f()).sum() + (z * w).sum(), z)
    assert torch.equal(g, w)


# ---- data that would have a gradient --------------------------------------------------------------------------------
@pytest.mark.parametrize("frozen", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_data_has_no_gradient(frozen, dtype):
    """scores of another network taken outside no_grad, advantages of a value head: the same bits as detached, and no gradient for them"""
    from repsurf_amd import objectives
    z, y, off, old, adv, pref = small_case()
    z.requires_grad_(not frozen)
    other = logits_of(50, 13, torch.float32, seed=9).requires_grad_(True)
    score, sums = objectives.token_logprobs(other, y).to(dtype), objectives.sequence_logprobs(other, y, off).to(dtype)
    value = adv.to(dtype).requires_grad_(True)

    def policy(o, a, r):
        return objectives.policy_loss(z, y, o, a, ref_logp=r, offset=off, kl_coef=0.1)

    for got, want in ((policy(score, value, score), policy(score.detach(), value.detach(), score.detach())),
                      (objectives.preference_loss(z, y, off, sums), objectives.preference_loss(z, y, off, sums.detach()))):
        assert torch.equal(got.loss, want.loss) and got.loss.requires_grad != frozen
        if not frozen:
            a, b, c = torch.autograd.grad(got.loss, (z, other, value), allow_unused=True)
            d, = torch.autograd.grad(want.loss, z)
            assert torch.equal(a, d) and b is None and c is None


# ---- forward-mode derivatives are not offered ---------------------------------------------------------------------------
def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fw
    from repsurf_amd import objectives
    z, y, off, old, adv, pref = small_case()
    calls = [lambda t: objectives.token_logprobs(t, y), lambda t: objectives.sequence_logprobs(t, y, off), lambda t: objectives.preference_loss(t, y, off, pref),
             lambda t: objectives.policy_loss(t, y, old, adv)]
    data = [lambda t: objectives.preference_loss(z, y, off, t(pref)), lambda t: objectives.policy_loss(z, y, t(old), adv),
            lambda t: objectives.policy_loss(z, y, old, t(adv)), lambda t: objectives.policy_loss(z, y, old, adv, ref_logp=t(old), kl_coef=0.1)]
    want = [f(z) for f in calls[:2]]
    with fw.dual_level():
        for f in calls:
            for leaf in (z, z.clone().requires_grad_(True)):
                with pytest.raises(NotImplementedError):
                    f(fw.make_dual(leaf, torch.ones_like(leaf)))
        for f in data:
            with pytest.raises(NotImplementedError):
                f(lambda t: fw.make_dual(t, torch.ones_like(t)))
        assert all(torch.equal(f(z), w) for f, w in zip(calls, want))          # no tangent: nothing to refuse
    assert all(torch.equal(f(z), w) for f, w in zip(calls, want))


# ---- a reference that masks the taken class -----------------------------------------------------------------------------
@pytest.mark.parametrize("classes", [13, 1500, 20001])
@pytest.mark.parametrize("rows", [24, 300])
def test_a_reference_that_masks_the_taken_class(classes, rows):
    """exp(d) - 1 - d is infinite there, its slope exp(d) - 1 is -1; the rows beside it keep theirs.  Tolerances as in the policy tests: of a
    coefficient what the log-probability moves it by, and its rounding."""
    from repsurf_amd import objectives
    from tests.test_objectives_gpu import U, Ref
    z, y = logits_of(rows, classes, torch.float32, seed=4).requires_grad_(True), targets_of(rows, classes, seed=4)
    y[2], y[5] = 1, 2
    ref = Ref(z, y)
    g = torch.Generator().manual_seed(6)
    x = ref.logp.detach()
    old, adv, other = (x - 0.05).float(), torch.randn(rows, generator=g), (x + torch.randn(rows, generator=g)).float()
    other[2], other[5], kl = -math.inf, -1e30, 0.05
    out = objectives.policy_loss(z, y.cuda(), old.cuda(), adv.cuda(), ref_logp=other.cuda(), kl_coef=kl)
    assert float(out.loss) == math.inf and float(out.kl) == math.inf
    w = ref.counts / int(ref.counts.sum())
    r, d, a = torch.exp(x - old.double()), other.double() - x, adv.double()
    c = w * (-a * r - kl * torch.expm1(d))
    sens = w * (r * a.abs() + kl * torch.exp(d))
    want, = torch.autograd.grad(ref.logp, ref.z, c, retain_graph=True)
    for factor in (1.0, 0.5):
        got, = torch.autograd.grad(out.loss * factor, z, retain_graph=True)
        assert torch.isfinite(got).all()
        ref.check_grad(got, want * factor, torch.float32, c * factor, factor * (1.01 * sens * ref.L + 3 * U * c.abs()))


# ---- pairs that are far apart -------------------------------------------------------------------------------------------
@pytest.mark.parametrize("smoothing", [0.0, 0.1])
@pytest.mark.parametrize("apart", [0.0, 4.0, 30.0, 50.0, 80.0, -30.0, -50.0, -80.0])
def test_the_slope_of_pairs_that_are_far_apart(apart, smoothing):
    """h = `apart` and its neighbours.  d loss / dh = smoothing - sigmoid(-h); sigmoid(-h) moves by at most itself times dh, so what the sums
    are off (beta L) is what it is off relatively; the coefficient adds the roundings of itself and of its two factors."""
    from repsurf_amd import objectives
    from tests.test_objectives_gpu import U, Ref
    lengths, beta = [30, 11, 7, 19], 0.1
    n = sum(lengths)
    z, y = logits_of(n, 13, torch.float32, seed=8).requires_grad_(True), targets_of(n, 13, seed=8)
    ref = Ref(z, y)
    sums = torch.stack([p.sum() for p in ref.logp.split(lengths)])
    other = sums.detach().clone()
    other[0] -= apart / beta
    other[1] -= (apart + 0.7) / beta
    other = other.float()
    r = beta * (sums - other.double())
    h = r[:2] - r[2:]
    ls = torch.nn.functional.logsigmoid
    want = -((1 - smoothing) * ls(h) + smoothing * ls(-h)).mean()
    got = objectives.preference_loss(z, y.cuda(), ends(lengths), other.cuda(), beta=beta, label_smoothing=smoothing)
    dr = beta * torch.stack([x.sum() for x in (ref.L * ref.counts).split(lengths)])
    dh = dr[:2] + dr[2:]
    low = torch.sigmoid(-h.detach())
    slope = smoothing - low                                    # d loss / dh, and what it may be off
    off = low * torch.expm1(dh) + 2.0 ** -50 * (smoothing + low)
    assert abs(float(got.loss) - float(want)) <= float(dh.mean()) + 2 * U * abs(float(want))
    g, = torch.autograd.grad(got.loss, z)
    spread = lambda t: torch.cat([t[i].expand(m) for i, m in enumerate(lengths)])      # noqa: E731
    c = spread(torch.cat([slope, -slope]) * beta / 2)
    w, = torch.autograd.grad(ref.logp, ref.z, c)
    ref.check_grad(g, w, torch.float32, c, spread(torch.cat([off, off]) * beta / 2) + 4 * U * c.abs())
    assert (g != 0).any()


# ---- saved logits in another layout -----------------------------------------------------------------------------------
@pytest.mark.parametrize("classes", [13, 5003])
def test_pitched_logits_that_come_back_dense(classes):
    """unpacked where they lay, but without their pitch; and by columns"""
    z, y, off, old, adv, pref = small_case(classes)
    room = torch.zeros(50 * (classes + 30), device="cuda")
    pitched = room.view(50, classes + 30)[:, :classes]
    for name in ("token", "sequence", "preference", "policy"):
        leaf = z.clone().requires_grad_(True)
        up = 0.5 * torch.ones_like(losses(leaf, y, off, old, adv, pref)[name]())
        want, = torch.autograd.grad(losses(leaf, y, off, old, adv, pref)[name](), leaf, up)
        for dense in (True, False):
            with torch.no_grad():
                pitched.copy_(z)
            leaf = pitched.detach().requires_grad_(True)

            def unpack(t):
                if t.dim() != 2:
                    return t
                out = room[:50 * classes].view(50, classes) if dense else torch.empty(classes, 50, device="cuda").t()
                with torch.no_grad():
                    out.copy_(z)
                return out

            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
                loss = losses(leaf, y, off, old, adv, pref)[name]()
            got, = torch.autograd.grad(loss, leaf, up)
            assert torch.equal(got, want), (name, dense)


# ---- a backward pass captured without its forward pass --------------------------------------------------------------------
@pytest.mark.parametrize("name", ["token", "sequence", "preference", "policy"])
@pytest.mark.parametrize("classes", [13, 5003])
def test_a_captured_backward_pass_of_an_eager_forward_pass(name, classes):
    """Replays with upstream gradients of 0.5, 1, 2 and 1 again, each against an eager pass; what a replay returned may be overwritten in
    between.  The logits are no leaf: nothing is accumulated in the graph."""
    z, y, off, old, adv, pref = small_case(classes)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x = z.clone().requires_grad_(True) * 1.0
        f = losses(x, y, off, old, adv, pref)[name]
        warm = f()
        up = torch.ones_like(warm)
        torch.autograd.grad(warm, x, up, retain_graph=True)
        out = f()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        g, = torch.autograd.grad(out, x, up, retain_graph=True)
    for k in (0.5, 1.0, 2.0, 1.0):
        with torch.cuda.stream(side):
            up.fill_(k)
            graph.replay()
            got = g.clone()
            g.zero_()
            want, = torch.autograd.grad(warm, x, up, retain_graph=True)
        torch.cuda.synchronize()
        assert torch.equal(got, want), k


@pytest.mark.parametrize("classes", [13, 5003])
def test_forward_and_backward_passes_in_graphs_of_their_own(classes):
    """the second graph twice for each replay of the first, on new logits"""
    z, y, off, old, adv, pref = small_case(classes)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x = z.clone().requires_grad_(True)
        w = x * 1.0
        f = losses(w, y, off, old, adv, pref)["policy"]
        up = torch.ones_like(f())
        torch.autograd.grad(f(), w, up)
    torch.cuda.synchronize()
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(first, stream=side):
        out = f()
    with torch.cuda.graph(second, stream=side, pool=first.pool()):
        g, = torch.autograd.grad(out, w, up, retain_graph=True)
    for k in range(3):
        with torch.cuda.stream(side):
            with torch.no_grad():
                w.copy_(logits_of(50, classes, torch.float32, seed=20 + k))
            first.replay()
            again = w.detach().clone().requires_grad_(True)
            for factor in (0.5, 1.0, 2.0):
                up.fill_(factor)
                second.replay()
                got = g.clone()
                g.zero_()
                loss = losses(again, y, off, old, adv, pref)["policy"]()
                want, = torch.autograd.grad(loss, again, up)
                assert torch.equal(out, loss) and torch.equal(got, want), (k, factor)
        torch.cuda.synchronize()
