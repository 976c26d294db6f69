"""repsurf_amd.objectives without a device, where a call meets something unusual: its autograd code with a recorder in the kernels' place."""
import pytest
import torch

from repsurf_amd import objectives as O

ROWS, CLASSES = 6, 5


@pytest.fixture
def calls(monkeypatch):
    """the ABI calls that would be made: (name, arguments); descriptors as dicts of what stood in them"""
    made = []

    def record(device, name, *args):
        made.append((name, [{f: getattr(a._obj, f) for f, _ in a._obj._fields_} if hasattr(a, "_obj") else a for a in args]))

    monkeypatch.setattr(O, "_call", record)
    monkeypatch.setitem(O._bad, None, 0)
    monkeypatch.setattr(O, "_capture", lambda device: 0)
    return made


def leaf():
    return torch.randn(ROWS, CLASSES, generator=torch.Generator().manual_seed(0)).requires_grad_(True)


def functions(z):
    y, off, one = torch.zeros(ROWS, dtype=torch.long), torch.tensor([2, 5], dtype=torch.int32), torch.ones(ROWS)
    return {"token": lambda: O._TokenLogprobs.apply(z, y, -100, True), "sequence": lambda: O._SequenceLogprobs.apply(z, y, off, -100, False, True),
            "preference": lambda: O._Preference.apply(z, y, off, torch.zeros(2), 0.1, 0.0, False, -100, True)[0],
            "policy": lambda: O._Policy.apply(z, y, one, one, None, off, 0.8, 1.2, 0.0, True, -100, True)[0]}


NAMES = ["token", "sequence", "preference", "policy"]


class Drop(torch.autograd.Function):
    """hands nothing on: its input has no gradient"""

    @staticmethod
    def forward(ctx, x):
        return x.clone()

    @staticmethod
    def backward(ctx, g):
        return None


@pytest.mark.parametrize("name", NAMES)
def test_no_upstream_gradient_is_no_gradient(calls, name):
    z = leaf()
    out = functions(z)[name]()
    assert torch.autograd.grad(Drop.apply(out).sum(), z, allow_unused=True) == (None,)
    assert not any(n.endswith("backward") for n, _ in calls)
    torch.autograd.grad(functions(z)[name]().sum(), z)
    assert sum(n.endswith("backward") for n, _ in calls) == 1


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_data_is_taken_out_of_its_graph(dtype):
    t = torch.ones(ROWS, dtype=dtype, requires_grad=True)
    for data in (t, t * 2, t[::1], t.detach()):
        got = O._values("data", data, (ROWS,), leaf())
        assert got.dtype is torch.float32 and not got.requires_grad and torch.equal(got, data.detach().float())
    plain = torch.ones(ROWS)
    assert O._values("data", plain, (ROWS,), leaf()) is plain


def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fw
    y, off, one, two = torch.zeros(ROWS, dtype=torch.long), torch.tensor([2, 5], dtype=torch.int32), torch.ones(ROWS), torch.zeros(2)
    with fw.dual_level():
        for z in (leaf().detach(), leaf()):
            dual = fw.make_dual(z, torch.ones_like(z))
            for call in (lambda: O.token_logprobs(dual, y), lambda: O.sequence_logprobs(dual, y, off), lambda: O.preference_loss(dual, y, off, two),
                         lambda: O.policy_loss(dual, y, one, one)):
                with pytest.raises(NotImplementedError):
                    call()
        z, dual, two_dual = leaf(), fw.make_dual(one, one), fw.make_dual(two, two)
        for call in (lambda: O.policy_loss(z, y, dual, one), lambda: O.policy_loss(z, y, one, dual), lambda: O.policy_loss(z, y, one, one, ref_logp=dual),
                     lambda: O.preference_loss(z, y, off, two_dual)):
            with pytest.raises(NotImplementedError):
                call()
        with pytest.raises(O._lib.RepSurfHipError, match="HIP device"):          # no tangent: it goes on as far as it can on the CPU
            O.policy_loss(z, y, one, one)


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("kind", ["dense", "columns", "pitched"])
def test_saved_logits_that_come_back_in_another_layout(calls, name, kind):
    """a hook that packs pitched logits and unpacks them at the very address where they lay, dense (as a freed buffer is handed out again):
    what the backward pass is told about them is what came back"""
    room = torch.zeros(ROWS * 16)
    z = room.view(ROWS, 16)[:, :CLASSES].requires_grad_(True)
    values, seen = torch.randn(ROWS, CLASSES), []

    def pack(t):
        return (t, t.dim() == 2)

    def unpack(packed):
        t, logits = packed
        if not logits:
            return t
        if kind == "dense":
            out = room[:ROWS * CLASSES].view(ROWS, CLASSES)
        elif kind == "columns":
            out = torch.zeros(CLASSES, ROWS).t()
        else:
            out = torch.zeros(ROWS, 9)[:, :CLASSES]
        with torch.no_grad():
            out.copy_(values)
        seen.append(out)
        return out

    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        out = functions(z)[name]()
    forward = next(a[0] for n, a in calls if n in ("rs_token_logprobs", "rs_policy_loss"))
    assert forward["ld"] == 16 and forward["logits"] == z.data_ptr()
    torch.autograd.grad(out.sum(), z)
    desc = next(a[0] for n, a in calls if n.endswith("backward"))
    assert desc["ld"] == (9 if kind == "pitched" else CLASSES)
    if kind != "columns":
        assert desc["logits"] == seen[-1].data_ptr()
    else:
        assert desc["logits"] != seen[-1].data_ptr()          # a copy whose rows lie dense


def test_saved_logits_that_come_back_as_something_else_are_refused(calls):
    for other in (torch.zeros(ROWS, CLASSES, dtype=torch.bfloat16), torch.zeros(ROWS - 1, CLASSES), torch.zeros(ROWS, CLASSES + 1), torch.zeros(ROWS)):
        z = leaf()
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: other if t.dim() == 2 else t):
            out = functions(z)["policy"]()
        with pytest.raises(O._lib.RepSurfHipError, match="saved logits"):
            torch.autograd.grad(out.sum(), z)


def test_sequences_need_their_offset():
    y = torch.zeros(ROWS, dtype=torch.long)
    for call in (lambda: O.sequence_logprobs(leaf(), y, None), lambda: O.preference_loss(leaf(), y, None, torch.zeros(2))):
        with pytest.raises(ValueError, match="offset"):
            call()
