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
