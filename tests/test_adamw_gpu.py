"""repsurf_amd.optim.AdamW (csrc/adamw.hip) against its formulas in 64 bits.

Tolerances.  u = 2^-24, half a step of fp32.  One update rounds m four times (the constant 1 - b1, difference, product, sum) and v six times
(two constants, three products, the sum; all but three of them on the small term), each by at most u of the largest term; the moments contract, so over k steps |dm| <= 4 k u max|m, g|, and
|dv| <= 5 k u max(v, g^2).  The update's ratio is then off by at most (4 + 2.5 + 9) k u relative -- the square root halves v's error; the device's
root and reciprocal (2 u each), the sum, the product, the step size and the bias corrections add nine -- and p by k (3 u |p| + 16 k u lr r), r the largest
ratio seen: the constant 1 - lr wd, its product with p and the sum are three roundings of at most u |p| each."""
import copy

import numpy as np
import pytest
import torch

from tests import adamw_oracle as O

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
SHAPES = [(64, 10, 1, 1), (1,), (3,), (255,), (256,), (257,), (513, 129), (2049,), (1, 7), (40, 1024)]
HYPER = dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2)


def make(shapes, dtype=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter(torch.randn(s, generator=g).to(dtype).cuda()) for s in shapes]


def give(ps, seed, scale=0.1):
    g = torch.Generator().manual_seed(1000 + seed)
    for p in ps:
        p.grad = (torch.randn(p.shape, generator=g) * scale).to(p.dtype).to(p.device)


def np64(t):
    return t.detach().double().cpu().numpy()


class Twin:
    """the same steps in 64 bits"""

    def __init__(self, ps, hyper):
        self.h = hyper
        self.p = [np64(p) for p in ps]
        self.m, self.v, self.t = [np.zeros_like(p) for p in self.p], [np.zeros_like(p) for p in self.p], [0] * len(ps)
        self.ratio, self.big, self.gbig = 0.0, [0.0] * len(ps), [0.0] * len(ps)

    def step(self, grads, clip=1.0):
        for i, g in enumerate(grads):
            if g is None:
                continue
            self.t[i] += 1
            b1, b2 = self.h["betas"]
            old = self.p[i]
            self.p[i], self.m[i], self.v[i] = O.step(old, g, self.m[i], self.v[i], self.t[i], self.h["lr"], b1, b2, self.h["eps"], self.h["weight_decay"], clip)
            if g.size:
                self.ratio = max(self.ratio, np.abs(self.p[i] - old * (1 - self.h["lr"] * self.h["weight_decay"])).max() / max(self.h["lr"], 1e-30))
                self.gbig[i] = max(self.gbig[i], np.abs(g * clip).max(), np.abs(self.m[i]).max())

    def check(self, ps, opt, moments=True):
        for i, p in enumerate(ps):
            if p.numel() == 0:
                continue
            k = max(1, self.t[i])
            tol = k * (3 * U * np.abs(self.p[i]) + 16 * k * U * self.h["lr"] * self.ratio)
            assert (np.abs(np64(p) - self.p[i]) <= tol).all(), i
            if moments:
                s = opt.state[p]
                assert (np.abs(np64(s["exp_avg"]) - self.m[i]) <= 4 * k * U * self.gbig[i]).all(), i
                assert (np.abs(np64(s["exp_avg_sq"]) - self.v[i]) <= 5 * k * U * self.gbig[i] ** 2).all(), i


@pytest.mark.parametrize("hyper", [HYPER, dict(HYPER, weight_decay=0.0), dict(HYPER, betas=(0.0, 0.9)), dict(HYPER, betas=(0.8, 0.99), lr=0.1, eps=1e-3)])
def test_32_bits_over_more_tensors_than_one_launch_takes(hyper):
    from repsurf_amd.optim import AdamW
    ps, hyper = make(SHAPES * 9), dict(hyper)                   # 90 tensors
    opt, twin = AdamW(ps, **hyper), Twin(ps, hyper)
    for it in range(4):
        give(ps, it)
        if it == 2:
            hyper["lr"] *= 0.5
            opt.param_groups[0]["lr"] = hyper["lr"]
        opt.step()
        twin.step([np64(p.grad) for p in ps])
    hyper["lr"] *= 2                        # the bound is that of the larger rate
    twin.check(ps, opt)


def test_strided_grads_odd_addresses_missing_grads_and_groups():
    from repsurf_amd.optim import AdamW
    flat = torch.randn(5000, device="cuda")
    ps = [torch.nn.Parameter(flat[1:1 + 700].view(70, 10)), torch.nn.Parameter(flat[1003:1003 + 33 * 65].view(33, 65)),
          torch.nn.Parameter(torch.zeros(0, 4, device="cuda")), torch.nn.Parameter(torch.randn(300, device="cuda"))]
    opt = AdamW([{"params": ps[:2]}, {"params": ps[2:], "lr": 3e-3, "weight_decay": 0.0}], **HYPER)
    twins = [Twin(ps[:2], HYPER), Twin(ps[2:], dict(HYPER, lr=3e-3, weight_decay=0.0))]
    for it in range(5):
        give(ps, it)
        ps[0].grad = ps[0].grad.t().contiguous().t()           # the transpose's strides
        big = torch.zeros(33 * 65 + 3, device="cuda")
        big[3:].copy_(ps[1].grad.view(-1))
        ps[1].grad = big[3:].view(33, 65)                      # four bytes off every larger alignment
        if it in (1, 2):
            ps[0].grad = None                                  # its step count and bias correction wait
        if it == 3:
            ps[3].grad = None
        opt.step()
        for tw, part in zip(twins, (ps[:2], ps[2:])):
            tw.step([None if p.grad is None else np64(p.grad) for p in part])
    for tw, part in zip(twins, (ps[:2], ps[2:])):
        tw.check(part, opt)
    sd = opt.state_dict()
    assert [float(sd["state"][i]["step"]) for i in range(4)] == [3.0, 5.0, 0.0, 4.0]
    assert float(flat[0]) == float(flat[0]) and torch.isfinite(flat).all()


def test_neighbours_of_a_parameter_stay_as_they_are():
    from repsurf_amd.optim import AdamW
    for dtype, bits in ((torch.float32, 32), (torch.bfloat16, 32), (torch.float32, 8), (torch.bfloat16, 8)):
        flat = torch.randn(4000, device="cuda").to(dtype)
        before = flat.clone()
        spans = [(1, 258), (301, 302), (399, 399 + 1027), (1501, 1501 + 2051)]
        ps = [torch.nn.Parameter(flat[a:b]) for a, b in spans]
        give(ps, 0)
        AdamW(ps, state_bits=bits, **HYPER).step()
        same = torch.ones(4000, dtype=torch.bool)
        for a, b in spans:
            same[a:b] = False
        assert torch.equal(flat.cpu()[same], before.cpu()[same])
        assert (flat.cpu()[~same] != before.cpu()[~same]).float().mean() > 0.3


def test_it_resumes_from_torch_and_torch_from_it():
    from repsurf_amd.optim import AdamW
    a, b = make(SHAPES), make(SHAPES)
    ref = torch.optim.AdamW(b, **HYPER)
    for it in range(3):
        give(b, it)
        ref.step()
    with torch.no_grad():
        for x, y in zip(a, b):
            x.copy_(y)
    opt = AdamW(a, lr=1.0)
    opt.load_state_dict(copy.deepcopy(ref.state_dict()))
    assert opt.param_groups[0]["lr"] == HYPER["lr"]
    twin = Twin(a, HYPER)
    twin.m, twin.v, twin.t = [np64(ref.state[p]["exp_avg"]) for p in b], [np64(ref.state[p]["exp_avg_sq"]) for p in b], [3] * len(b)
    for it in range(3, 5):
        give(a, it)
        opt.step()
        twin.step([np64(p.grad) for p in a])
    twin.check(a, opt)
    back = torch.optim.AdamW(make(SHAPES), lr=1.0)
    back.load_state_dict(opt.state_dict())
    for p, q in zip(back.param_groups[0]["params"], a):
        assert torch.equal(back.state[p]["exp_avg"], opt.state[q]["exp_avg"]) and float(back.state[p]["step"]) == 5.0


def test_it_loads_from_the_cpu_and_from_bf16_moments(tmp_path):
    """a checkpoint mapped to the CPU; torch's own for bf16 parameters, whose moments are bf16"""
    from repsurf_amd.optim import AdamW
    a = make(SHAPES, torch.bfloat16)
    for bits in (32, 8):
        first = AdamW(a, state_bits=bits, seed=2, **HYPER)
        give(a, 1)
        first.step()
        torch.save(first.state_dict(), tmp_path / "o.pt")
        b = make(SHAPES, torch.bfloat16)
        second = AdamW(b, state_bits=bits, seed=2, **HYPER)
        second.load_state_dict(torch.load(tmp_path / "o.pt", map_location="cpu", weights_only=True))
        for k, x in first.flat_state().items():
            assert torch.equal(x, second.flat_state()[k])
    b = make(SHAPES, torch.bfloat16)
    ref = torch.optim.AdamW(b, **HYPER)
    give(b, 1)
    ref.step()
    opt = AdamW(b, **HYPER)
    opt.load_state_dict(ref.state_dict())
    for p in b:
        assert torch.equal(opt.state[p]["exp_avg"], ref.state[p]["exp_avg"].float())
    assert int(opt._dev[0]["step"][0]) == 1


def test_a_master_is_what_the_parameter_was_and_what_it_cut_off():
    """the halves of words at the borders of the format: ties, the largest numbers, denormals, NaNs with a payload"""
    from repsurf_amd.optim import AdamW
    words = torch.tensor([0, 0x7FFF, 0x8000, 0x8001, 0xFFFF, 0x10000, 0x3F808000, 0x3F80FFFF, 0x3F818000, 0x7F7FFFFF, 0x7F7F8000, 0x7F800000, 0x1, 0x00800000], dtype=torch.int64)
    words = torch.cat([words, words + 0x80000000])
    x = torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32).view(torch.float32)
    p = torch.nn.Parameter(torch.zeros(len(x), dtype=torch.bfloat16, device="cuda"))
    p.grad = torch.zeros_like(p)
    opt = AdamW([p], lr=0.0, weight_decay=0.0)
    opt.step()
    bits = words + 0x8000
    with torch.no_grad():                                   # as a step would have left them
        up = (bits >> 16) & 0xFFFF
        p.view(torch.int16).copy_(torch.where(up >= 1 << 15, up - (1 << 16), up).to(torch.int16))
        low = words & 0xFFFF
        opt.flat_state()["low"][:len(x)] = torch.where(low >= 1 << 15, low - (1 << 16), low).to(torch.int16).cuda()
    master = opt.unpack_state()["master"][:len(x)].cpu()
    assert torch.equal(master.view(torch.int32), x.view(torch.int32))
    opt.step()                                              # a rate of nothing: the same words again
    again = opt.unpack_state()["master"][:len(x)].cpu()
    finite = torch.isfinite(x)
    assert torch.equal(again.view(torch.int32)[finite], x.view(torch.int32)[finite]) and torch.isinf(again[~finite]).sum() + torch.isnan(again[~finite]).sum() == (~finite).sum()


def test_bf16_parameters_keep_their_masters():
    """200 steps of 1e-4 each on values near 1: bf16's spacing there is 2^-7, so without a master nothing would move"""
    from repsurf_amd.optim import AdamW
    ps = make(SHAPES, torch.bfloat16)
    h = dict(HYPER, lr=1e-4)
    opt, twin = AdamW(ps, **h), Twin(ps, h)
    for it in range(200):
        give(ps, 5)
        opt.step()
        twin.step([np64(p.grad) for p in ps])
    assert twin.ratio < 10
    master = opt.unpack_state()["master"].cpu()
    at = 0
    for p, want, t in zip(ps, twin.p, twin.t):
        got = np64(master[at:at + p.numel()]).reshape(want.shape)
        tol = t * (3 * U * (np.abs(want) + t * h["lr"] * twin.ratio) + 16 * U * h["lr"] * twin.ratio * 10)         # the ratio is off by a bounded part: the moments contract
        assert (np.abs(got - want) <= tol).all()
        assert (np.abs(np64(p) - got) <= 2.0 ** -8 * np.abs(got)).all()             # half a step of bf16
        at += -(-p.numel() // 256) * 256
    with torch.no_grad():                                                           # written from outside, zero and infinity among it
        for p in ps:
            p.zero_()
            p.view(-1)[0] = float("inf")
    master = opt.unpack_state()["master"]
    at = 0
    for p in ps:
        part = master[at:at + p.numel()]
        assert torch.isinf(part[0]) or part[0] > 3e38
        assert (part[1:].abs() < 1e-38).all()
        at += -(-p.numel() // 256) * 256


def run8(dtype, shapes, steps, seed, scale=0.1):
    from repsurf_amd.optim import AdamW
    ps = make(shapes, dtype)
    opt = AdamW(ps, state_bits=8, seed=seed, **HYPER)
    return ps, opt


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_8_bits_against_the_format_in_64_bits(dtype):
    """Every step from the values that the device holds.  m and v are off by a few u before they are rounded, so an element goes to the
    other neighbour only where the dither comes within that of its border: 8 u / 2^-4 of them at most, the grid's step being 2^-4 of
    the value at least; 3 of them in 10^5 elements are allowed for, and each by one step of the grid."""
    ps, opt = run8(dtype, SHAPES, 4, seed=11)
    b1, b2 = HYPER["betas"]
    sizes = [p.numel() for p in ps]
    starts = np.concatenate([[0], np.cumsum([-(-n // 256) * 256 for n in sizes])])
    state = {"exp_avg": np.zeros(starts[-1]), "exp_avg_sq": np.zeros(starts[-1])}
    masters = [np64(p) for p in ps]
    for t in range(1, 5):
        give(ps, t, scale=10.0 ** -t)
        opt.step()
        got = {k: np64(x) for k, x in opt.unpack_state().items()}
        off = 0
        for i, p in enumerate(ps):
            a, b, n = starts[i], starts[i + 1], sizes[i]
            new, m, v = O.step(masters[i].reshape(-1), np64(p.grad).reshape(-1), state["exp_avg"][a:a + n], state["exp_avg_sq"][a:a + n], t,
                               HYPER["lr"], b1, b2, HYPER["eps"], HYPER["weight_decay"])
            dm, dv = O.dither(11, t, a // 256, (b - a) // 256)
            for name, x, d in (("exp_avg", m, dm), ("exp_avg_sq", v, dv)):
                q, step = O.quantise(O.blocks_of(x), name == "exp_avg", d)
                diff = np.abs(got[name][a:b].reshape(-1, 256) - q)
                assert (diff <= step * 1.01).all(), (name, i, t)
                off += int((diff > 0).sum())
            held = got["master"][a:a + n] if dtype == torch.bfloat16 else np64(p).reshape(-1)
            assert (np.abs(held - new) <= 3 * U * np.abs(new) + 16 * U * HYPER["lr"] * 12).all(), (i, t)
            masters[i] = held
            assert np.all(got["exp_avg"][a + n:b] == 0) and np.all(got["exp_avg_sq"][a + n:b] == 0)
        assert off <= 3 + 1e-4 * starts[-1], off
        state = got


@pytest.mark.parametrize("clip", [None, 0.05])
def test_8_bit_moments_are_those_of_the_elementary_operations(clip):
    """Two steps against torch's own fp32 operations and the rounding in 64 bits, on a million elements: no moment differs.  Both sides
    round the same values the same way but in the grid's linear part, where the kernel's word has 20 bits below a step: one element in 2^20
    of those there, none expected here."""
    from repsurf_amd.optim import AdamW
    n = 1 << 20
    g = torch.Generator().manual_seed(7)
    p = torch.nn.Parameter(torch.randn(n, generator=g).cuda())
    opt = AdamW([p], state_bits=8, seed=4, max_grad_norm=clip, **HYPER)
    m, v = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    for t in (1, 2, 3):
        p.grad = (torch.randn(n, generator=g) * 1e-3).cuda()
        x = p.grad
        if clip:
            norm = x.double().square().sum().sqrt().float()
            x = x * torch.clamp(clip / (norm + 1e-6), max=1.0)
        m = m + (x - m) * (1 - 0.9)
        v = v * 0.999 + (1 - 0.999) * x * x
        opt.step()
        dm, dv = O.dither(4, t, 0, n // 256)
        m, v = (torch.from_numpy(O.quantise(np64(y).reshape(-1, 256), s, d)[0].reshape(-1)).float().cuda() for y, s, d in ((m, True, dm), (v, False, dv)))
        got = opt.unpack_state()
        assert int((got["exp_avg"] != m).sum()) == 0 and int((got["exp_avg_sq"] != v).sum()) == 0, t
        if clip:
            assert torch.equal(opt.grad_norm, norm)


def test_8_bits_decay_a_second_moment():
    """one large gradient, then none: rounded to nearest, b2 v would stay v for ever"""
    from repsurf_amd.optim import AdamW
    p = torch.nn.Parameter(torch.zeros(4096, device="cuda"))
    opt = AdamW([p], state_bits=8, lr=0.0)
    for it in range(500):
        p.grad = torch.full_like(p, 1.0 if it == 0 else 0.0)
        opt.step()
    v = np64(opt.unpack_state()["exp_avg_sq"])
    want = 1e-3 * 0.999 ** 499
    # the deviation of a step's rounding is below 0.3 steps of 2^-3 v, 500 of them and 4096 elements: 0.3 / 8 * sqrt(500 / 4096) = 1.3 %
    assert abs(v.mean() / want - 1) < 5 * 0.013


def test_8_bits_extremes():
    """A NaN, an infinity, denormals and a range wider than the grid's leave their block's other elements as they would be"""
    from repsurf_amd.optim import AdamW
    p = torch.nn.Parameter(torch.zeros(1024, device="cuda"))
    q = torch.nn.Parameter(torch.zeros(1024, device="cuda"))
    g = torch.randn(1024, generator=torch.Generator().manual_seed(3)).cuda()
    g[300] = 1e-12                           # far below its block's range
    g[512:768] = 1e-30 * g[512:768]          # squares below fp32's smallest numbers
    g[768:] = 0
    bad = g.clone()
    bad[7], bad[100] = float("nan"), float("inf")
    a, b = AdamW([p], state_bits=8), AdamW([q], state_bits=8)
    for it in range(3):
        p.grad, q.grad = g.clone(), bad.clone()
        a.step(); b.step()
    keep = torch.ones(1024, dtype=torch.bool)
    keep[[7, 100]] = False
    x, y = a.unpack_state(), b.unpack_state()
    for k in ("exp_avg", "exp_avg_sq"):
        if k == "exp_avg":
            assert torch.isnan(y[k][7]) and torch.isnan(y[k][100])
        else:
            assert torch.isinf(y[k][7]) and torch.isinf(y[k][100])
        assert torch.isfinite(x[k]).all() and torch.equal(x[k].cpu()[keep], y[k].cpu()[keep])
    assert torch.equal(p.detach().cpu()[keep], q.detach().cpu()[keep]) and torch.isnan(q[7]) and torch.isnan(q[100])
    assert (x["exp_avg_sq"][300] > 0) and p[300].abs() < 1e-2          # a second moment never vanishes under its gradient
    assert (p[768:] == 0).all() and torch.isfinite(p).all()


def test_8_bit_state_dicts(tmp_path):
    from repsurf_amd.optim import AdamW
    ps, opt = run8(torch.bfloat16, SHAPES, 0, seed=5)
    for it in range(2):
        give(ps, it)
        opt.step()
    torch.save(opt.state_dict(), tmp_path / "o.pt")
    qs = make(SHAPES, torch.bfloat16)
    with torch.no_grad():
        for x, y in zip(qs, ps):
            x.copy_(y)
    other = AdamW(qs, state_bits=8, seed=5, lr=9.0)
    other.load_state_dict(torch.load(tmp_path / "o.pt", weights_only=True))
    for k, x in opt.flat_state().items():
        assert torch.equal(x, other.flat_state()[k])
    for it in range(2, 4):
        give(ps, it); give(qs, it)
        opt.step(); other.step()
    for x, y in zip(ps, qs):
        assert torch.equal(x, y)
    # 32-bit moments are rounded to nearest: at most half a step, 2^-4 of the value, above the linear range
    wide = AdamW(make(SHAPES), **HYPER)
    give(wide.param_groups[0]["params"], 1)
    wide.step()
    packed = AdamW(make(SHAPES), state_bits=8)
    packed.load_state_dict(wide.state_dict())
    assert packed.state_dict()["state"][0]["step"] == 1
    for k, octaves in (("exp_avg", 14), ("exp_avg_sq", 30)):
        x, y = np64(wide.flat_state()[k]).reshape(-1, 256), np64(packed.unpack_state()[k]).reshape(-1, 256)
        least = np.exp2(O.exponent(x).max(1, keepdims=True) - octaves + 1 - 3) / 2
        assert (np.abs(x - y) <= np.maximum(np.abs(x) * 2.0 ** -4, np.where(k == "exp_avg", 1, 2) * least)).all()
    with pytest.raises(ValueError, match="8-bit"):
        wide.load_state_dict(packed.state_dict())


@pytest.mark.parametrize("bits,dtype", [(32, torch.float32), (8, torch.bfloat16)])
@pytest.mark.parametrize("bound", [1.0, 1e6])
def test_clipping_by_the_common_norm(bits, dtype, bound):
    """The norm is summed in fp64 and rounded once."""
    from repsurf_amd.optim import AdamW
    ps = make(SHAPES * 9, dtype)
    give(ps, 3)
    want = np.sqrt(sum((np64(p.grad) ** 2).sum() for p in ps))
    clipped, plain = AdamW(ps, state_bits=bits, max_grad_norm=bound, **HYPER), None
    before = [p.detach().clone() for p in ps]
    grads = [p.grad.clone() for p in ps]
    clipped.step()
    assert abs(float(clipped.grad_norm) / want - 1) <= 1.001 * U
    assert all(torch.equal(p.grad, g) for p, g in zip(ps, grads))
    m = np64(clipped.unpack_state()["exp_avg"])
    at, c = 0, min(1.0, bound / (want + 1e-6))
    for p in ps:
        x = 0.1 * c * np64(p.grad).reshape(-1)
        tol = np.abs(x) * (12 * U if bits == 32 else 2.0 ** -3) + (0 if bits == 32 else np.abs(x).max() * 2.0 ** -16)
        assert (np.abs(m[at:at + x.size] - x) <= tol).all()
        at += -(-x.size // 256) * 256
    ps[4].grad[0] = float("nan")
    clipped.step()
    assert torch.isnan(clipped.grad_norm) and all(torch.isnan(p).all() for p in ps if p.numel())      # as torch's clipping leaves it


@pytest.mark.parametrize("bits,dtype,bound", [(32, torch.float32, None), (8, torch.float32, 0.5), (8, torch.bfloat16, None), (32, torch.bfloat16, 0.5)])
def test_captured_steps_are_the_eager_ones_bit_for_bit(bits, dtype, bound):
    from repsurf_amd.optim import AdamW
    a, b = make(SHAPES, dtype), make(SHAPES, dtype)
    kw = dict(HYPER, state_bits=bits, max_grad_norm=bound, seed=9)
    ours, eager = AdamW(a, **kw), AdamW(b, **kw)
    give(a, 0); give(b, 0)
    static = [p.grad for p in a]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ours.step()
    torch.cuda.current_stream().wait_stream(side)
    eager.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ours.step()
    for it in range(1, 5):
        give(b, it)
        for g, p in zip(static, b):
            g.copy_(p.grad)
        for opt in (ours, eager):
            opt.param_groups[0]["lr"] = 1e-3 / it
        ours.sync_hyper()
        graph.replay()
        eager.step()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(a, b)), it
    for k, x in ours.flat_state().items():
        assert torch.equal(x, eager.flat_state()[k])
    if bound:
        assert torch.equal(ours.grad_norm, eager.grad_norm)
    assert [int(t) for t in ours._dev[0]["step"]] == [5] * len(a)
    ours.load_state_dict(eager.state_dict())              # in place: the graph's addresses still hold
    give(b, 9)
    for g, p in zip(static, b):
        g.copy_(p.grad)
    ours.sync_hyper()
    graph.replay()
    eager.step()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_refusals_on_the_device():
    from repsurf_amd import _lib
    from repsurf_amd.optim import AdamW
    p = torch.nn.Parameter(torch.zeros(4, 6, device="cuda").t())
    p.grad = torch.zeros(4, 6, device="cuda").t()
    with pytest.raises(_lib.RepSurfHipError, match="contiguous"):
        AdamW([p]).step()
    h = torch.nn.Parameter(torch.zeros(4, device="cuda", dtype=torch.float16))
    h.grad = torch.zeros_like(h)
    with pytest.raises(_lib.RepSurfHipError, match="fp32 or bf16"):
        AdamW([h]).step()
    buf = torch.zeros(8, device="cuda")
    two = [torch.nn.Parameter(buf), torch.nn.Parameter(buf)]
    for q in two:
        q.grad = torch.zeros(8, device="cuda")
    with pytest.raises(_lib.RepSurfHipError, match="share"):
        AdamW(two).step()
    q = torch.nn.Parameter(torch.zeros(8, device="cuda"))
    q.grad = torch.zeros(8, device="cuda")
    opt = AdamW([q])
    opt.step()
    room = torch.zeros(600, device="cuda")
    q.data = room                                            # larger than the state that was made for it
    with pytest.raises(_lib.RepSurfHipError, match="another size"):
        opt.step()
    q.grad = None
    q.grad = torch.zeros(600, device="cuda")
    with pytest.raises(_lib.RepSurfHipError, match="another size"):
        opt.step()
    q.data = room[:8]
    q.grad = None
    q.grad = torch.zeros(8, device="cuda")
    opt.step()
    opt.param_groups[0]["params"] = [torch.nn.Parameter(torch.zeros(8, device="cuda"))]
    opt.param_groups[0]["params"][0].grad = torch.zeros(8, device="cuda")
    with pytest.raises(_lib.RepSurfHipError, match="changed"):
        opt.step()


def test_a_tensor_whose_offsets_pass_32_bits():
    """2^32 + 300 bf16 parameters with 8-bit moments: the last elements against the formula"""
    from repsurf_amd.optim import AdamW
    n = (1 << 32) + 300
    p = torch.nn.Parameter(torch.full((n,), 0.5, dtype=torch.bfloat16, device="cuda"))
    p.grad = torch.full((n,), 0.25, dtype=torch.bfloat16, device="cuda")
    opt = AdamW([p], state_bits=8, **HYPER)
    opt.step()
    want = 0.5 * (1 - 1e-5) - 1e-3 * 0.25 / (0.25 + 1e-8)
    for part in (p[:1000], p[(1 << 31) - 500:(1 << 31) + 500], p[n - 600:]):
        x = np64(part)
        assert (np.abs(x - want) <= 2.0 ** -8 * want).all()
    low = opt.flat_state()["low"]
    assert low.numel() == n // 256 * 256 + 256 and (low[n:] == 0).all()
    for a in (0, n - 100):
        bits = (p[a:a + 100].detach().view(torch.int16).int() << 16) + low[a:a + 100].int()
        assert (np.abs(np64(bits.view(torch.float32)) - want) <= 3 * U * want + 16 * U * 1e-3).all()
    codes = opt.flat_state()["exp_avg"]
    assert (codes[n:] == 0).all() and (codes[n - 300:n] != 0).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_the_training_loop_step_takes_it(bits):
    """graph.TrainLoopStep with this optimizer: forward, loss, backward, norm and update as one replay are the eager loop.  The bounds
    are those of the same comparison with Adam (test_graph_gpu.py); 8-bit moments may lie one step of their grid, an eighth, apart."""
    from models.repsurf.repsurf_ssg_umb import Model
    from repsurf_amd.graph import TrainLoopStep
    from repsurf_amd.optim import AdamW
    from tests import torch_executor
    from tests.test_graph_gpu import cloud, disable_dropout, name_seeded_init, ref_args
    from util.utils import SmoothClsLoss
    torch_executor.set_backend("hip")
    crit = SmoothClsLoss()
    batches = [(torch.from_numpy(cloud(20 + i, b, 1024)).cuda().permute(0, 2, 1).contiguous(), (torch.arange(b).cuda() * (i + 1)) % 15)
               for i, b in enumerate((8, 8, 5))]

    def fresh():
        m = Model(ref_args())
        name_seeded_init(m)
        disable_dropout(m)
        m = m.cuda().train()
        return m, AdamW(m.parameters(), state_bits=bits, max_grad_norm=1.0, seed=3, **HYPER)

    eager, eopt = fresh()
    torch.manual_seed(77)
    want = []
    for pts, lab in batches:
        eopt.zero_grad()
        loss = crit(eager(pts), lab.long())
        loss.backward()
        eopt.step()
        want.append((loss.item(), float(eopt.grad_norm)))
    graphed, gopt = fresh()
    step = TrainLoopStep(graphed, crit, gopt)
    torch.manual_seed(77)
    for (pts, lab), (lw, nw) in zip(batches, want):
        _, loss = step(pts, lab.long())
        assert abs(loss.item() - lw) <= 1e-4 and abs(float(gopt.grad_norm) / nw - 1) <= 1e-2
    a, b = torch.cat([p.detach().flatten() for p in graphed.parameters()]), torch.cat([p.detach().flatten() for p in eager.parameters()])
    assert torch.isfinite(a).all() and (a - b).norm() / b.norm() < 1e-3
    assert [int(t) for t in gopt._dev[0]["step"]] == [3] * len(list(graphed.parameters()))
    for k, x in gopt.unpack_state().items():
        y = eopt.unpack_state()[k]
        assert (x - y).norm() / y.norm() < (1e-2 if bits == 32 else 0.125), k
    step.close()


@pytest.mark.parametrize("bits", [32, 8])
def test_the_ragged_segmentation_step_takes_it(bits):
    """graph.RaggedSegStep, two network graphs that share the optimizer's state, clipped: against the same step launched eagerly.  The
    first loss is the eager one bit for bit, the second to what the gradients' atomics leave of one update (the bound of the same
    comparison with Adam, test_seg_gpu.py)."""
    from repsurf_amd.graph import RaggedSegStep
    from repsurf_amd.head import CrossEntropyLoss
    from repsurf_amd.optim import AdamW
    from tests.test_seg_gpu import _ragged_batches, _seg_model, subproject
    _, batches, labels = _ragged_batches()
    crit = CrossEntropyLoss(ignore_index=255)
    with subproject("segmentation"):
        base = _seg_model()
        base.surface_constructor.random_inv = False
        runs = []
        for capture in (True, False):
            model = copy.deepcopy(base)
            opt = AdamW(model.parameters(), state_bits=bits, max_grad_norm=1.0, seed=2, **HYPER)
            step = RaggedSegStep(model, crit, opt, batches[0], labels[0], capacity=4 * 1024, capture=capture)
            losses, norms = [], []
            for s in range(4):
                losses.append(step(batches[(s + 1) % 4], labels[(s + 1) % 4]).item())
                torch.cuda.synchronize()
                norms.append(float(opt.grad_norm))
            assert [int(t) for t in opt._dev[0]["step"]] == [4] * len(opt.param_groups[0]["params"])
            step.close()
            runs.append((losses, norms))
        (l1, n1), (l0, n0) = runs
        assert l1[0] == l0[0] and abs(l1[1] - l0[1]) <= 1e-5 and np.isfinite(l1).all(), (l1, l0)
        assert abs(n1[0] / n0[0] - 1) <= 1e-4 and np.isfinite(n1).all()


def test_a_policy_step_of_the_segmentation_network_as_one_graph():
    """scores by the acting network, then network, policy loss, backward, norm and update captured by graph.RaggedSegStep with the loss as its
    criterion; padding rows carry the ignored label.  Against the eager loop of the same calls."""
    from repsurf_amd import objectives
    from repsurf_amd.graph import RaggedSegStep
    from repsurf_amd.optim import AdamW
    from tests.test_seg_gpu import _ragged_batches, _seg_model, subproject
    _, batches, labels = _ragged_batches()
    with subproject("segmentation"):
        base = _seg_model()
        base.surface_constructor.random_inv = False
        runs = []
        for capture in (True, False):
            model = copy.deepcopy(base)
            old = torch.full((4 * 1024,), -2.5, device="cuda")
            adv = torch.randn(4 * 1024, generator=torch.Generator().manual_seed(1)).cuda()

            def crit(pred, target):
                rows = pred.shape[0]
                return objectives.policy_loss(pred, target, old[:rows], adv[:rows], kl_coef=0.1, ref_logp=old[:rows], ignore_index=255).loss

            opt = AdamW(model.parameters(), max_grad_norm=1.0, **HYPER)
            step = RaggedSegStep(model, crit, opt, batches[0], labels[0], capacity=4 * 1024, capture=capture, ignore_index=255)
            runs.append([step(batches[(s + 1) % 4], labels[(s + 1) % 4]).item() for s in range(4)])
            step.close()
        assert runs[0][0] == runs[1][0] and abs(runs[0][1] - runs[1][1]) <= 1e-4 * max(1.0, abs(runs[1][1])) and np.isfinite(runs[0]).all(), runs
