"""repsurf_amd.optim.AdamW without a device, where a call meets something unusual: its host side over buffers on the CPU."""
import pytest
import torch

from repsurf_amd import optim


@pytest.fixture
def on_the_cpu(monkeypatch):
    """the host side alone: parameters may lie on the CPU, and nothing is launched"""
    monkeypatch.setattr(optim.AdamW, "_check_param", staticmethod(lambda p, device: None))


def made(bits, *shapes, dtype=torch.float32):
    """an optimizer whose state holds numbers that are its elements' own"""
    ps = [torch.nn.Parameter(torch.zeros(s, dtype=dtype)) for s in shapes]
    opt = optim.AdamW(ps, state_bits=bits)
    st = opt._group_state(0, opt.param_groups[0], torch.device("cpu"))
    for k, buf in enumerate(st["flat"].values()):
        buf.copy_((torch.arange(buf.numel()) * 7 + 3 + k) % 120)
    st["step"].copy_(torch.arange(len(shapes)) + 100)
    return opt, st


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_it_takes_its_own_state_back(on_the_cpu, bits, dtype):
    opt, st = made(bits, (300, 5), (256,), (1, 7), dtype=dtype)
    sd = opt.state_dict()
    want = {i: {k: v.clone() for k, v in s.items()} for i, s in sd["state"].items()}
    sd["param_groups"][0]["lr"] = 0.5
    opt.load_state_dict(sd)
    got = opt.state_dict()
    assert opt.param_groups[0]["lr"] == 0.5 and st["step"].tolist() == [100, 101, 102]
    for i, s in want.items():
        assert s.keys() == got["state"][i].keys()
        for k, v in s.items():
            assert torch.equal(v, got["state"][i][k]), (i, k)


def tables_of(opt, st):
    tables, _ = opt._tables(st, opt.param_groups[0]["params"])
    return [(bf16, list(t.p), list(t.n)) for bf16, t in tables]


def test_lists_follow_the_parameters_types(on_the_cpu):
    """parameters and gradients whose memory stays where it is while its type changes: another list, or a refusal"""
    opt, st = made(32, (40,), (30,))
    a, b = opt.param_groups[0]["params"]
    words, grads = [p.detach().clone() for p in (a, b)], [torch.zeros(40), torch.zeros(30)]

    def give(kinds):
        for p, w, g, kind in zip((a, b), words, grads, kinds):
            p.grad = None
            p.data = w.view(kind)[:w.numel()]
            p.grad = g.view(kind)[:w.numel()]

    f, h = torch.float32, torch.bfloat16
    give((f, f))
    first = tables_of(opt, st)
    assert first == [(0, [a.data_ptr(), b.data_ptr()], [40, 30])] and tables_of(opt, st) == first
    give((f, h))
    with pytest.raises(optim._lib.RepSurfHipError, match="became bf16"):
        opt._tables(st, [a, b])
    give((f, f))
    assert tables_of(opt, st) == first
    opt = optim.AdamW([torch.nn.Parameter(torch.zeros(40, dtype=h)), torch.nn.Parameter(torch.zeros(30))])
    a, b = opt.param_groups[0]["params"]
    st = opt._group_state(0, opt.param_groups[0], torch.device("cpu"))
    give((h, f))
    assert tables_of(opt, st) == [(0, [b.data_ptr()], [30]), (1, [a.data_ptr()], [40])]
    give((f, f))
    assert tables_of(opt, st) == [(0, [a.data_ptr(), b.data_ptr()], [40, 30])]
    give((h, f))
    assert tables_of(opt, st) == [(0, [b.data_ptr()], [30]), (1, [a.data_ptr()], [40])]


def test_a_gradient_of_another_type_is_refused(on_the_cpu):
    opt, st = made(32, (40,))
    p, g = opt.param_groups[0]["params"][0], torch.zeros(40)
    p.grad = g
    tables_of(opt, st)
    if not hasattr(p, "grad_dtype"):
        pytest.skip("gradients have their parameter's type here")
    p.grad = None
    p.grad_dtype = torch.bfloat16
    p.grad = g.view(torch.bfloat16)[:40]
    assert p.grad.data_ptr() == g.data_ptr()
    with pytest.raises(optim._lib.RepSurfHipError, match="parameter's type"):
        opt._tables(st, [p])


def test_state_that_does_not_fit_is_refused_before_anything_is_written(on_the_cpu):
    opt, st = made(8, (300, 5), (256,))
    good = opt.state_dict()
    before = {k: v.clone() for k, v in st["flat"].items()}

    def spoiled(i, **kw):
        state = {k: dict(v) for k, v in good["state"].items()}
        for k, v in kw.items():
            if v is None:
                del state[i][k]
            else:
                state[i][k] = v
        return {"state": state, "param_groups": [dict(good["param_groups"][0], lr=0.5)]}

    byte = lambda *n: torch.zeros(n, dtype=torch.uint8)      # noqa: E731
    for bad, text in ((spoiled(0, exp_avg_exponent=byte(1)), "exponent"), (spoiled(0, exp_avg_sq_exponent=byte(7)), "exponent"),
                      (spoiled(1, exp_avg_exponent=byte(2)), "exponent"), (spoiled(1, exp_avg_exponent=torch.tensor(3, dtype=torch.uint8)), "exponent"),
                      (spoiled(1, exp_avg_sq=None, exp_avg_sq_exponent=None), "without the other"), (spoiled(0, exp_avg=None), "without the other")):
        with pytest.raises(ValueError, match=text):
            opt.load_state_dict(bad)
        assert opt.param_groups[0]["lr"] == good["param_groups"][0]["lr"] and st["step"].tolist() == [100, 101]
        assert all(torch.equal(v, before[k]) for k, v in st["flat"].items())


def test_a_sparse_gradient_is_refused(on_the_cpu):
    opt, st = made(32, (4, 3), (5,))
    a, b = opt.param_groups[0]["params"]
    a.grad, b.grad = torch.sparse_coo_tensor([[0], [1]], [1.0], (4, 3)), torch.zeros(5)
    for other in (b.grad, None):
        b.grad = other
        with pytest.raises(optim._lib.RepSurfHipError, match="dense"):
            opt._tables(st, [a, b])
