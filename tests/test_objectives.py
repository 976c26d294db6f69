"""repsurf_amd.objectives without a device: refusals and the binding's structs."""
import ctypes
import os
import subprocess

import pytest
import torch

from repsurf_amd import _lib, objectives as O
from tests.util import ROOT

Z, Y, OFF = torch.zeros(6, 5), torch.zeros(6, dtype=torch.long), torch.tensor([3, 6], dtype=torch.int32)
A = torch.zeros(6)


@pytest.mark.parametrize("call,error", [
    (lambda: O.token_logprobs(Z[0], Y), ValueError),
    (lambda: O.token_logprobs(Z.double(), Y), TypeError),
    (lambda: O.token_logprobs(Z, Y[:5]), ValueError),
    (lambda: O.token_logprobs(Z, Y.float()), ValueError),
    (lambda: O.token_logprobs(Z[:, :0], Y), ValueError),
    (lambda: O.token_logprobs(Z, Y), _lib.RepSurfHipError),
    (lambda: O.sequence_logprobs(Z, Y, OFF[:0]), ValueError),
    (lambda: O.sequence_logprobs(Z, Y, OFF.float()), ValueError),
    (lambda: O.sequence_logprobs(Z, Y, OFF), _lib.RepSurfHipError),
    (lambda: O.preference_loss(Z, Y, OFF, A[:2]), _lib.RepSurfHipError),
    (lambda: O.policy_loss(Z, Y, A, A), _lib.RepSurfHipError),
])
def test_refusals(call, error):
    with pytest.raises(error):
        call()


def test_entry_points_report_bad_arguments():
    def rows(**kw):
        d = dict(logits=256, rows=4, ld=8, classes=8, type=0, target=256)
        d.update(kw)
        return ctypes.byref(O.LogitsDesc(**d))

    for bad in (dict(rows=-1), dict(classes=0), dict(ld=7), dict(type=3), dict(offset=256), dict(sequences=2), dict(logits=None), dict(target=None),
                dict(classes=(1 << 30) + 1, ld=1 << 31), dict(rows=1 << 31, offset=256, sequences=1), dict(rows=1 << 31)):
        with pytest.raises(_lib.RepSurfHipError, match="rs_token_logprobs"):
            _lib.call("rs_token_logprobs", rows(**bad), 256, None, None, None, None)
        with pytest.raises(_lib.RepSurfHipError):
            _lib.call("rs_token_logprobs_backward", rows(**bad), 256, 256, None, 0, 256, None)
    with pytest.raises(_lib.RepSurfHipError, match="null"):
        _lib.call("rs_token_logprobs", rows(), None, None, None, None, None)
    with pytest.raises(_lib.RepSurfHipError, match="null"):
        _lib.call("rs_token_logprobs_backward", rows(), None, 256, None, 0, 256, None)
    with pytest.raises(_lib.RepSurfHipError, match="null"):
        _lib.call("rs_sequence_sums", rows(), 256, 0, 256, None, None, None)
    for a in ((0, 256, 256, 256, 0.1, 0.0), (1, None, 256, 256, 0.1, 0.0), (1, 256, 256, 256, 0.1, 0.6), (1, 256, 256, 256, 0.1, -0.1)):
        with pytest.raises(_lib.RepSurfHipError, match="rs_preference_pairs"):
            _lib.call("rs_preference_pairs", *a, 256, 256, 256, None)

    def policy(**kw):
        d = dict(old_logp=256, advantages=256, token_mean=1, low=0.8, high=1.2, counts=256, counts_room=64, partial=256, partial_room=6144, loss=256, stats=256)
        d.update(kw)
        return ctypes.byref(O.PolicyDesc(**d))

    for bad in (dict(loss=None), dict(stats=None), dict(partial=None), dict(counts=None), dict(old_logp=None), dict(advantages=None), dict(dlogits=256),
                dict(coef=256), dict(token_mean=0), dict(advantages_per_sequence=1), dict(counts_room=0), dict(partial_room=11)):
        with pytest.raises(_lib.RepSurfHipError, match="rs_policy_loss"):
            _lib.call("rs_policy_loss", rows(), policy(**bad), None)
    _lib.call("rs_token_logprobs", rows(rows=0), 256, None, None, None, None)          # nothing to do
    _lib.call("rs_token_logprobs_backward", rows(rows=0), 256, 256, None, 0, 256, None)


def test_structs_match_the_header(tmp_path):
    pairs = {"rs_logits": O.LogitsDesc, "rs_policy": O.PolicyDesc}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "repsurf_hip.h"', 'int main(void) {',
             f'if (RS_POLICY_COUNTS != {O.POLICY_COUNTS} || RS_POLICY_GROUPS != {O.POLICY_GROUPS} || RS_LOGITS_FEW_ROWS != {O.FEW_ROWS} || RS_LOGITS_PARTS != {O.PARTS}) return 1;']
    for c, cls in pairs.items():
        lines.append(f'printf("{c} size %zu\\n", sizeof({c}));')
        lines += [f'printf("{c} {f} %zu\\n", offsetof({c}, {f}));' for f, _ in cls._fields_]
    (tmp_path / "l.c").write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(tmp_path / "l.c"), "-o", str(tmp_path / "l")], check=True)
    for line in subprocess.run([str(tmp_path / "l")], check=True, capture_output=True, text=True).stdout.splitlines():
        c, f, v = line.split()
        assert int(v) == (ctypes.sizeof(pairs[c]) if f == "size" else getattr(pairs[c], f).offset), line
