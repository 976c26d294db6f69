"""repsurf_amd.optim.AdamW where a call meets something unusual."""
import copy

import pytest
import torch

from tests.test_adamw_gpu import HYPER, give, make

pytestmark = pytest.mark.gpu
SHAPES = [(64, 10, 1, 1), (1,), (255,), (256,), (257,), (513, 129), (1, 7)]


def words(t):
    return t.detach().clone().view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.element_size()])


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("kinds", [(torch.float32,), (torch.bfloat16,), (torch.float32, torch.bfloat16)])
def test_it_takes_its_own_state_back(bits, kinds):
    """opt.load_state_dict(opt.state_dict()) changes nothing but what the program changed in it: every word of the state, and the step after it"""
    from repsurf_amd.optim import AdamW
    ps = [p for k in kinds for p in make(SHAPES, k, seed=1)]
    twins = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    opt = AdamW([{"params": ps[:4]}, {"params": ps[4:], "lr": 2e-3}], state_bits=bits, **HYPER)
    other = AdamW([{"params": twins[:4]}, {"params": twins[4:], "lr": 2e-3}], state_bits=bits, **HYPER)
    for it in range(3):
        for o, q in ((opt, ps), (other, twins)):
            give(q, it)
            if it == 1:
                q[2].grad = None
            o.step()
    before = [{k: words(v) for k, v in opt.flat_state(g).items()} for g in (0, 1)]
    for sd in (opt.state_dict(), copy.deepcopy(opt.state_dict()), copy.copy(opt.state_dict())):
        sd["param_groups"][0]["lr"] = 5e-4
        opt.load_state_dict(sd)
        assert opt.param_groups[0]["lr"] == 5e-4
        for g in (0, 1):
            for k, v in opt.flat_state(g).items():
                assert torch.equal(words(v), before[g][k]), (g, k)
        assert [float(opt.state_dict()["state"][i]["step"]) for i in range(4)] == [3.0, 3.0, 2.0, 3.0]
    other.param_groups[0]["lr"] = 5e-4
    for o, q in ((opt, ps), (other, twins)):
        give(q, 9)
        o.step()
    for a, b in zip(ps, twins):
        assert torch.equal(words(a), words(b))
    for g in (0, 1):
        for (k, a), b in zip(opt.flat_state(g).items(), other.flat_state(g).values()):
            assert torch.equal(words(a), words(b)), k


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("groups", [1, 2])
def test_its_own_state_in_another_order(bits, groups):
    """states exchanged between two parameters of one shape, one of a third left out: read whole before anything is written"""
    from repsurf_amd.optim import AdamW
    ps = make([(300, 5), (300, 5), (700,)])
    opt = AdamW([{"params": ps[:1]}, {"params": ps[1:]}] if groups == 2 else ps, state_bits=bits, **HYPER)
    for it in range(2):
        give(ps, it)
        opt.step()
    names = ("exp_avg", "exp_avg_sq") + (("exp_avg_exponent", "exp_avg_sq_exponent") if bits == 8 else ())
    want = [{k: opt.state[p][k].clone() for k in names} for p in ps]
    sd = opt.state_dict()
    opt.load_state_dict({"state": {0: sd["state"][1], 1: sd["state"][0]}, "param_groups": sd["param_groups"]})
    for k in names:
        assert torch.equal(opt.state[ps[0]][k], want[1][k]) and torch.equal(opt.state[ps[1]][k], want[0][k])
        assert (opt.state[ps[2]][k] == 0).all()
    assert [float(opt.state_dict()["state"][i]["step"]) for i in range(3)] == [2.0, 2.0, 0.0]


@pytest.mark.parametrize("eps", [0.0, 1e-20, 1e-12])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_small_eps_beside_small_gradients(eps, dtype):
    """Second moments down to fp32's smallest numbers, each rounded by at most 2^-150 there (half its spacing), three times a step: the ratio is
    off by dv / 2 v relatively, beside the bound of the other tests.  A gradient of 0 moves nothing but the decay."""
    import numpy as np
    from repsurf_amd.optim import AdamW
    from tests.test_adamw_gpu import U, Twin, np64
    hyper = dict(HYPER, eps=eps)
    n, k = 2100, 3
    p = torch.nn.Parameter(torch.zeros(n, dtype=dtype, device="cuda"))
    size = torch.logspace(-20.5, -3, n, dtype=torch.float64) * torch.where(torch.arange(n) % 2 == 0, 1.0, -1.0)
    size[7], size[n - 1] = 0.0, 0.0
    p.grad = size.to(dtype).cuda()
    opt, twin = AdamW([p], **hyper), Twin([p], hyper)
    with np.errstate(invalid="ignore", divide="ignore"):
        for _ in range(k):
            opt.step()
            twin.step([np64(p.grad)])
    got = opt.unpack_state()["master"][:n].double().cpu().numpy() if dtype == torch.bfloat16 else np64(p)
    v = twin.v[0]
    live = np64(p.grad) != 0
    want = twin.p[0]
    dv = 3 * k * 2.0 ** -150
    tol = k * (3 * U * np.abs(want) + hyper["lr"] * (16 * k * U + dv / np.where(live, v, 1.0)))
    assert (got[~live] == 0).all() and np.isfinite(got).all()
    assert (v[live].min() < 1e-43) and (np.abs(got - want) <= tol)[live].all()
