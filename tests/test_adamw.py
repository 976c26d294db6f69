"""repsurf_amd.optim.AdamW without a device: refusals, the binding's structs, the dither's statistics, the format's arithmetic."""
import ctypes
import os
import subprocess

import numpy as np
import pytest
import torch

from repsurf_amd import _lib, optim
from tests import adamw_oracle as O
from tests.util import ROOT


def params(*shapes, dtype=torch.float32):
    return [torch.nn.Parameter(torch.zeros(s, dtype=dtype)) for s in shapes]


@pytest.mark.parametrize("kw", [dict(lr=-1.0), dict(eps=-1e-8), dict(weight_decay=-1.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)),
                                dict(state_bits=16), dict(max_grad_norm=0.0), dict(max_grad_norm=-1.0), dict(max_grad_norm=float("nan"))])
def test_bad_arguments_are_refused(kw):
    with pytest.raises(ValueError):
        optim.AdamW(params((3,)), **kw)


def test_a_parameter_twice_in_a_group_is_refused():
    p = params((3,))[0]
    with pytest.raises(ValueError):
        optim.AdamW([p, p])


def test_it_is_an_adam_for_the_graphed_steps():
    assert issubclass(optim.AdamW, optim.Adam)


def test_a_step_on_the_cpu_is_refused():
    p = params((3,))[0]
    p.grad = torch.ones(3)
    with pytest.raises(_lib.RepSurfHipError, match="HIP device"):
        optim.AdamW([p]).step()
    assert optim.AdamW(params((3,))).step() is None          # no gradients: nothing to do
    with pytest.raises(_lib.RepSurfHipError, match="no state"):
        optim.AdamW(params((3,))).flat_state()


def test_foreign_state_is_refused():
    opt = optim.AdamW(params((3,)))
    sd = torch.optim.AdamW(params((3,))).state_dict()
    groups = sd["param_groups"]
    with pytest.raises(ValueError, match="amsgrad"):
        opt.load_state_dict({"state": {}, "param_groups": [dict(groups[0], amsgrad=True)]})
    with pytest.raises(ValueError, match="shape"):
        opt.load_state_dict({"state": {0: {"step": 1.0, "exp_avg": torch.zeros(4), "exp_avg_sq": torch.zeros(4)}}, "param_groups": groups})
    with pytest.raises(ValueError, match="8-bit"):
        opt.load_state_dict({"state": {0: {"step": 1.0, "exp_avg": torch.zeros(3, dtype=torch.uint8), "exp_avg_sq": torch.zeros(3, dtype=torch.uint8)}},
                             "param_groups": groups})
    with pytest.raises(ValueError, match="exponents"):
        optim.AdamW(params((3,)), state_bits=8).load_state_dict(
            {"state": {0: {"step": 1.0, "exp_avg": torch.zeros(3, dtype=torch.uint8), "exp_avg_sq": torch.zeros(3, dtype=torch.uint8)}},
             "param_groups": groups})
    opt.load_state_dict({"state": {}, "param_groups": groups})          # a fresh torch optimizer's state dict
    assert opt.param_groups[0]["lr"] == groups[0]["lr"]


def test_entry_points_report_bad_arguments():
    one = (ctypes.c_void_p * 1)(256)
    sizes, at, slot = (ctypes.c_longlong * 1)(4), (ctypes.c_longlong * 1)(0), (ctypes.c_int * 1)(0)
    cast = lambda a: ctypes.cast(a, ctypes.c_void_p)      # noqa: E731

    def listed(**kw):
        d = dict(count=1, p=cast(one), g=cast(one), n=cast(sizes), at=cast(at), slot=cast(slot))
        d.update(kw)
        return ctypes.byref(optim.AdamWList(*[d[k] for k, _ in optim.AdamWList._fields_]))

    def args(**kw):
        d = dict(bits=32, exp_avg=256, exp_avg_sq=256, step=256, done=256)
        d.update(kw)
        return ctypes.byref(optim.AdamWArgs(**d))

    for a, text in [(dict(bits=16), "bits"), (dict(bits=8), "bits"), (dict(bf16=1), "low"), (dict(exp_avg=None), "null"), (dict(done=None), "null")]:
        with pytest.raises(_lib.RepSurfHipError, match=text):
            _lib.call("rs_adamw_step", listed(), args(**a), None)
    with pytest.raises(_lib.RepSurfHipError, match="null pointer"):
        _lib.call("rs_adamw_step", listed(p=None), args(), None)
    for bad in ((ctypes.c_longlong * 1)(0), (ctypes.c_longlong * 1)(-5)):
        with pytest.raises(_lib.RepSurfHipError, match="tensor 0"):
            _lib.call("rs_adamw_step", listed(n=cast(bad)), args(), None)
    huge = (ctypes.c_longlong * 1)(1 << 36)
    with pytest.raises(_lib.RepSurfHipError, match="at most"):
        _lib.call("rs_adamw_step", listed(n=cast(huge)), args(), None)
    odd = (ctypes.c_longlong * 1)(128)
    with pytest.raises(_lib.RepSurfHipError, match="multiple of 256"):
        _lib.call("rs_adamw_step", listed(at=cast(odd)), args(), None)
    used = ctypes.c_int()
    with pytest.raises(_lib.RepSurfHipError, match="room"):
        _lib.call("rs_grad_square_sums", listed(), 0, 256, 0, ctypes.byref(used), None)
    for a in ((0, 256, 1.0, 256), (1, None, 1.0, 256), (1, 256, 0.0, 256), (1, 256, 1.0, None)):
        with pytest.raises(_lib.RepSurfHipError, match="rs_grad_norm"):
            _lib.call("rs_grad_norm", *a, None)
    with pytest.raises(_lib.RepSurfHipError, match="null"):
        _lib.call("rs_adamw_masters", listed(), None, None, None)
    for name, a in (("rs_adamw_pack", (100,) + (256,) * 6), ("rs_adamw_unpack", (100,) + (256,) * 4 + (0, 256, 256))):
        with pytest.raises(_lib.RepSurfHipError, match="multiple"):
            _lib.call(name, *a, None)
    _lib.call("rs_adamw_pack", 0, *(None,) * 7)
    _lib.call("rs_adamw_step", listed(count=0), args(), None)          # nothing to update


def test_structs_match_the_header(tmp_path):
    pairs = {"rs_adamw_list": optim.AdamWList, "rs_adamw_args": optim.AdamWArgs}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "repsurf_hip.h"', 'int main(void) {',
             'if (RS_GRAD_SQUARE_SUMS != %d || RS_ADAMW_DONE != %d) return 1;' % (optim.GRAD_SQUARE_SUMS, optim.DONE)]
    for c, cls in pairs.items():
        lines.append(f'printf("{c} size %zu\\n", sizeof({c}));')
        lines += [f'printf("{c} {f} %zu\\n", offsetof({c}, {f}));' for f, _ in cls._fields_]
    (tmp_path / "l.c").write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(tmp_path / "l.c"), "-o", str(tmp_path / "l")], check=True)
    out = subprocess.run([str(tmp_path / "l")], check=True, capture_output=True, text=True).stdout.split("\n")
    for line in filter(None, out):
        c, f, v = line.split()
        assert int(v) == (ctypes.sizeof(pairs[c]) if f == "size" else getattr(pairs[c], f).offset), line


def test_the_dither_is_uniform_and_uncorrelated():
    """2^19 pairs: a mean of n uniform numbers is within 5 / sqrt(12 n) of one half, a correlation within 5 / sqrt(n) of nothing"""
    n = 0
    parts = []
    for t in (1, 2, 1000, 123457):
        a, b = O.dither(7, t, 0, 512)
        parts.append(np.stack([a.reshape(-1), b.reshape(-1)]) / 65536)
        n += a.size
    x = np.concatenate(parts, 1)
    bound = 5 / np.sqrt(n)
    assert np.abs(x.mean(1) - 0.5).max() < 0.29 * bound
    z = (x - 0.5) * np.sqrt(12)
    assert abs((z[0] * z[1]).mean()) < bound                                       # the two of a pair
    for lag in (1, 2, 4, 64, 256):                                                 # neighbours, lanes, blocks
        assert np.abs((z[:, lag:] * z[:, :-lag]).mean(1)).max() < bound
    m = n // 4
    assert np.abs((z[:, :m] * z[:, m:2 * m]).mean(1)).max() < 5 / np.sqrt(m)       # the same element, one step later
    counts = np.histogram(x[0], 256, (0, 1))[0]
    assert ((counts - n / 256) ** 2 / (n / 256)).sum() < 255 + 5 * np.sqrt(2 * 255)


def test_the_rounding_has_the_mean_of_its_input():
    rng = np.random.RandomState(0)
    x = rng.randn(1, 256) * np.exp2(rng.randint(-14, 1, (1, 256)))
    got = np.zeros_like(x)
    for k in range(4000):
        q, step = O.quantise(x, True, rng.randint(0, 65536, x.shape))
        got += q
    # a rounding between two values `step` apart has a deviation of at most step / 2
    assert (np.abs(got / 4000 - x) <= 5 * step / 2 / np.sqrt(4000)).all()
