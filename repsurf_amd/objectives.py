"""Objectives on the log-probabilities of taken classes, on the kernels of csrc/logits.hip.

Beside head.CrossEntropyLoss, which fits a model to labels, these fit it to what a label or an answer was WORTH: a reward per row, or a
preference between two labelings.  Logits are (rows, classes) in fp32, bf16 or fp16, a row per point or token, with any row pitch; packed
batches hand over `offset` (B,) int32, the running row ends of their clouds (the collate format of the segmentation path), and rows behind
the last end do not count.  Neither do rows whose target is `ignore_index`: their logits are not read, their gradient is zero.  A target
outside [0, classes) makes its row NaN and is counted by head.bad_label_count, as the cross entropy does it.

    token_logprobs       log softmax(logits)[target] of every row, without the (rows, classes) log-softmax
    sequence_logprobs    their sum (or mean) over every sequence: what preference_loss takes of the reference model
    preference_loss      -log sigmoid(beta * difference of two sequences' log ratios), chosen sequences first
    policy_loss          clipped policy objective with a KL term against a reference policy

A row's statistics are collected in fp64; gradients are rounded once, to the logits' type.  The losses are differentiable in `logits` alone
(once, by backward passes; forward-mode tangents are refused); the other tensors are data.  The calls allocate through torch and can be
captured into a graph once they ran eagerly."""
import ctypes
from collections import namedtuple

import torch
from torch.autograd import Function, forward_ad
from torch.autograd.function import once_differentiable

from . import _lib, head

P, c_int, c_ll, c_double = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_double
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
POLICY_COUNTS, POLICY_GROUPS = 64, 8192          # RS_POLICY_COUNTS, RS_POLICY_GROUPS
FEW_ROWS, PARTS = 256, 64                         # RS_LOGITS_FEW_ROWS, RS_LOGITS_PARTS
SKIP_UNIT, ROW_COEF = 1, 2                        # RS_BACKWARD_SKIP_UNIT, RS_BACKWARD_ROW_COEF

PolicyLoss = namedtuple("PolicyLoss", "loss logp kl clip_fraction")
PreferenceLoss = namedtuple("PreferenceLoss", "loss chosen_rewards rejected_rewards")


class LogitsDesc(ctypes.Structure):          # rs_logits
    _fields_ = [("logits", P), ("rows", c_ll), ("ld", c_ll), ("classes", c_int), ("type", c_int), ("target", P), ("ignore_index", c_ll),
                ("offset", P), ("sequences", c_int), ("bad_labels", P)]


class PolicyDesc(ctypes.Structure):          # rs_policy
    _fields_ = [("old_logp", P), ("advantages", P), ("ref_logp", P), ("advantages_per_sequence", c_int), ("token_mean", c_int), ("low", c_double),
                ("high", c_double), ("kl_coef", c_double), ("counts", P), ("counts_room", c_int), ("partial", P), ("partial_room", c_int),
                ("loss", P), ("stats", P), ("logp", P), ("dlogits", P), ("coef", P), ("stat", P), ("scratch", P)]


def _no_tangent(*tensors):
    """forward-mode derivatives are refused: nothing here would carry a tangent on"""
    if getattr(forward_ad, "_current_level", 0) >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError("objectives: forward-mode derivatives are not offered")          # (a level below 0: none is entered)


def _logits(logits, target, offset, *data):
    """checks, and the tensors as the kernels take them"""
    _no_tangent(logits, *data)
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError(f"objectives: logits must be (rows, classes), got {tuple(logits.shape)}")
    if logits.dtype not in _TYPES:
        raise TypeError(f"objectives: logits must be fp32, bf16 or fp16, got {logits.dtype}")
    if target.dim() != 1 or target.shape[0] != logits.shape[0] or target.is_floating_point():
        raise ValueError(f"objectives: target must hold one class index per row, got {tuple(target.shape)} {target.dtype}")
    if offset is not None and (offset.dim() != 1 or offset.numel() < 1 or offset.is_floating_point()):
        raise ValueError("objectives: offset must be the (B,) running row ends")
    device = logits.device
    if target.device != device or (offset is not None and offset.device != device):
        raise ValueError("objectives: all tensors must be on the logits' device")
    if device.type != "cuda":
        raise _lib.RepSurfHipError("repsurf_amd.objectives run on the HIP device only (got a CPU tensor); there is no CPU fallback")
    return _pitched(logits)[0], _as(target, torch.int64), None if offset is None else _as(offset, torch.int32)


def _pitched(logits):
    """logits as the kernels take them (rows that lie dense, in order and apart), and the elements from one row to the next"""
    classes = logits.shape[1]
    if logits.is_contiguous():
        return logits, classes
    ld = logits.stride(0)
    return (logits, ld) if logits.stride(1) == 1 and ld >= classes else (logits.contiguous(), classes)


def _as(t, dtype):
    """data (not differentiated) as a dense tensor of a type"""
    if t.dtype is dtype and t.is_contiguous():
        return t.detach() if t.requires_grad else t
    return t.detach().to(dtype).contiguous()


def _values(name, t, shape, logits):
    if t.shape != shape:
        raise ValueError(f"objectives: {name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.device != logits.device:
        raise ValueError("objectives: all tensors must be on the logits' device")
    return _as(t, torch.float32)


_bad = {}


def _desc(logits, target, ignore_index, offset):
    rows, classes = logits.shape
    device = logits.device
    bad = _bad.get(device.index)
    if bad is None:
        bad = _bad[device.index] = head._bad_counter(device).data_ptr()        # (lives as long as the process)
    return LogitsDesc(logits.data_ptr(), rows, max(logits.stride(0), classes), classes, _TYPES[logits.dtype], target.data_ptr(), ignore_index,
                      None if offset is None else offset.data_ptr(), 0 if offset is None else offset.numel(), bad)


_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _call(device, name, *args):
    """an ABI call on the current stream of the tensors' device"""
    if device.index == _current_device():
        _lib.call(name, *args, _lib.current_stream())
    else:
        with torch.cuda.device(device):
            _lib.call(name, *args, _lib.current_stream())


def _capture(device):
    """the number of the capture that the current stream of a device is part of; 0: of none"""
    if device.index != _current_device():
        with torch.cuda.device(device):
            return _capture(device)
    if not torch.cuda.is_current_stream_capturing():
        return 0
    number = ctypes.c_ulonglong()
    _lib.call("rs_capture_id", ctypes.byref(number), _lib.current_stream())
    return number.value


def _backward(ctx, logits, target, offset, work, coef, gout, flags=0, out=None):
    """from the tensors as autograd hands them back (a hook may have moved them, to another pitch too); the rows' stat lies in `work`, ctx.stat
    floats from its start; coef: an address in it, or of a tensor that the caller holds.  (Autograd runs this on a thread of its own, whose every
    line costs twice what it costs elsewhere.)"""
    desc = ctx.desc
    rows, classes = logits.shape if logits.dim() == 2 else (-1, -1)
    if rows != desc.rows or classes != desc.classes or _TYPES.get(logits.dtype) != desc.type:
        raise _lib.RepSurfHipError("objectives: the saved logits came back with another shape or type")
    logits, desc.ld = _pitched(logits)
    if out is None:
        out = torch.empty_like(logits)          # (contiguous also where the logits have a pitch)
    desc.logits, desc.target = logits.data_ptr(), target.data_ptr()
    if offset is not None:
        desc.offset = offset.data_ptr()
    if gout is not None:
        gout = (gout if gout.dtype is torch.float32 else gout.to(torch.float32)).data_ptr()
    _call(logits.device, "rs_token_logprobs_backward", ctx.ref, work.data_ptr() + 4 * ctx.stat, coef, gout, flags, out.data_ptr())
    return out


def _once(inputs):
    """a backward pass over so many inputs that can be differentiated no further; the wrapper that says so is entered only where somebody
    builds its graph.  Where nothing came down to the first output (the only one that is differentiable) there is no gradient."""
    def wrap(fn):
        careful, none = once_differentiable(fn), (None,) * inputs
        return lambda ctx, g, *rest: none if g is None else careful(ctx, g, *rest) if torch.is_grad_enabled() else fn(ctx, g, *rest)
    return wrap


def _keep(ctx, desc, stat, *tensors):
    ctx.set_materialize_grads(False)          # (no zeros for the outputs that have no gradient)
    ctx.save_for_backward(*tensors)
    ctx.desc, ctx.ref, ctx.stat = desc, ctypes.byref(desc), stat


def _wanted(logits):
    return logits.requires_grad and torch.is_grad_enabled()


def _run(function, logits, *args):
    """a Function whose last argument says whether a gradient is wanted; scoring goes past autograd"""
    if _wanted(logits):
        return function.apply(logits, *args, True)
    return function.forward(None, logits.detach(), *args, False)


def _new(logits, *shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device=logits.device)


def _scratch_floats(logits):
    """room (a multiple of 8 bytes) for the pieces of a few long rows"""
    rows, classes = logits.shape
    return 0 if rows > FEW_ROWS or classes <= 8192 else 3 * PARTS * rows


class _TokenLogprobs(Function):
    @staticmethod
    def forward(ctx, logits, target, ignore_index, grad):
        rows = logits.shape[0]
        room = _scratch_floats(logits)
        logp = _new(logits, rows)
        work = _new(logits, room + (2 * rows if grad else 0)) if room or grad else None          # scratch, then stat
        desc = _desc(logits, target, ignore_index, None)
        _call(logits.device, "rs_token_logprobs", ctypes.byref(desc), logp.data_ptr(), None, work.data_ptr() + 4 * room if grad else None,
              work.data_ptr() if room else None)
        if grad:
            _keep(ctx, desc, room, logits, target, work)
        return logp

    @staticmethod
    @_once(4)
    def backward(ctx, g):
        logits, target, work = ctx.saved_tensors
        g = _as(g, torch.float32)
        return _backward(ctx, logits, target, None, work, g.data_ptr(), None), None, None, None


def token_logprobs(logits, target, ignore_index=-100):
    """logits (rows, classes), target (rows,) -> (rows,) fp32: log softmax(logits)[target], 0 for rows that do not count.  Reads the logits once;
    differentiable in them."""
    logits, target, _ = _logits(logits, target, None)
    return _run(_TokenLogprobs, logits, target, ignore_index)


def _sequences(logits, target, offset, ignore_index, average, extra=0):
    """-> (desc, out fp32, buffer, places): what the sequences of a packed batch add up to.  One buffer holds the rows' fp64
    log-probabilities, the sequences' fp64 sums, scratch, the rows' stat, and the sequences' factors, at these places (in floats)."""
    rows, n, room = logits.shape[0], offset.numel(), _scratch_floats(logits)
    sizes = dict(logp=2 * rows, sums=2 * n, scratch=room, stat=2 * rows, each=n, extra=extra)
    buf, out = _new(logits, sum(sizes.values())), _new(logits, n)
    places, at, start = {}, 0, buf.data_ptr()
    for k, v in sizes.items():
        places[k] = at
        at += v
    of = {k: start + 4 * v for k, v in places.items()}
    desc = _desc(logits, target, ignore_index, offset)
    _call(logits.device, "rs_token_logprobs", ctypes.byref(desc), None, of["logp"], of["stat"], of["scratch"] if room else None)
    _call(logits.device, "rs_sequence_sums", ctypes.byref(desc), of["logp"], int(average), of["sums"], out.data_ptr(), of["each"])
    return desc, out, buf, places


class _SequenceLogprobs(Function):
    @staticmethod
    def forward(ctx, logits, target, offset, ignore_index, average, grad):
        desc, out, buf, places = _sequences(logits, target, offset, ignore_index, average)
        if grad:
            _keep(ctx, desc, places["stat"], logits, target, offset, buf)
        return out

    @staticmethod
    @_once(6)
    def backward(ctx, g):
        logits, target, offset, buf = ctx.saved_tensors
        coef = _as(g, torch.float32) * buf[buf.numel() - offset.numel():]
        return (_backward(ctx, logits, target, offset, buf, coef.data_ptr(), None),) + (None,) * 5


def sequence_logprobs(logits, target, offset, ignore_index=-100, average=False):
    """(B,) fp32: the sum of token_logprobs over every sequence of a packed batch, or (average) their mean over the rows that count; 0 for
    a sequence without any.  Differentiable in the logits."""
    if offset is None:
        raise ValueError("sequence_logprobs: needs offset, the (B,) running row ends")
    logits, target, offset = _logits(logits, target, offset)
    return _run(_SequenceLogprobs, logits, target, offset, ignore_index, average)


class _Preference(Function):
    @staticmethod
    def forward(ctx, logits, target, offset, ref, beta, smoothing, average, ignore_index, grad):
        n = offset.numel()
        desc, rewards, buf, places = _sequences(logits, target, offset, ignore_index, average, extra=n)
        loss, start = _new(logits), buf.data_ptr()
        _call(logits.device, "rs_preference_pairs", n // 2, start + 4 * places["sums"], start + 4 * places["each"], ref.data_ptr(), beta, smoothing,
              loss.data_ptr(), rewards.data_ptr(), start + 4 * places["extra"])
        if grad:
            _keep(ctx, desc, places["stat"], logits, target, offset, buf)
            ctx.coef = places["extra"]
        ctx.mark_non_differentiable(rewards)
        return loss, rewards

    @staticmethod
    @_once(9)
    def backward(ctx, g, _):
        logits, target, offset, buf = ctx.saved_tensors
        return (_backward(ctx, logits, target, offset, buf, buf.data_ptr() + 4 * ctx.coef, g),) + (None,) * 8


def preference_loss(logits, target, offset, ref_logps, beta=0.1, label_smoothing=0.0, average=False, ignore_index=-100):
    """Paired log ratios.  The packed batch holds 2 P sequences, the P chosen ones first: sequence i is preferred to sequence P + i.  With
    r = beta * (sequence_logprobs(logits) - ref_logps) and h = r[i] - r[P + i],
        loss = mean of -(1 - label_smoothing) log sigmoid(h) - label_smoothing log sigmoid(-h).
    ref_logps (2 P,): sequence_logprobs of the reference model's logits (same `average`).
    -> PreferenceLoss(loss, chosen_rewards, rejected_rewards); the rewards (P,) are r, detached."""
    if offset is None:
        raise ValueError("preference_loss: needs offset, the (B,) running row ends")
    logits, target, offset = _logits(logits, target, offset, ref_logps)
    n = offset.numel()
    if n % 2:
        raise ValueError(f"preference_loss: {n} sequences are no pairs")
    if not 0.0 <= label_smoothing <= 0.5:
        raise ValueError("preference_loss: label_smoothing must lie in [0, 0.5]")
    ref = _values("ref_logps", ref_logps, (n,), logits)
    loss, rewards = _Preference.apply(logits, target, offset, ref, float(beta), float(label_smoothing), average, ignore_index, _wanted(logits))
    return PreferenceLoss(loss, rewards[: n // 2], rewards[n // 2:])


class _Policy(Function):
    @staticmethod
    def forward(ctx, logits, target, old, adv, ref, offset, low, high, kl_coef, token_mean, ignore_index, grad):
        rows = logits.shape[0]
        loss, stats, logp = old.new_empty(()), old.new_empty(2), old.new_empty(rows)
        partial = 3 * min(rows, POLICY_GROUPS)
        room, counts = _scratch_floats(logits), POLICY_COUNTS * (1 if token_mean else offset.numel())
        # one buffer: partial sums (fp64), scratch, counts, then the rows' stat (pairs: at an even place) and coef
        work = old.new_empty(2 * partial + room + counts + (3 * rows if grad else 0))
        at = work.data_ptr()
        scratch = at + 8 * partial
        count_at = scratch + 4 * room
        stat = count_at + 4 * counts
        coef = stat + 8 * rows
        d = torch.empty_like(logits) if grad else None
        held = grad and rows > 0
        desc = _desc(logits, target, ignore_index, offset)
        p = PolicyDesc(old.data_ptr(), adv.data_ptr(), None if ref is None else ref.data_ptr(), int(adv.dim() == 2), int(token_mean), low, high, kl_coef,
                       count_at, counts, at, partial, loss.data_ptr(), stats.data_ptr(), logp.data_ptr(), d.data_ptr() if held else None,
                       coef if held else None, stat if held else None, scratch if room else None)
        _call(logits.device, "rs_policy_loss", ctypes.byref(desc), ctypes.byref(p))
        if grad:
            _keep(ctx, desc, (stat - at) // 4, logits, target, work, offset)
            ctx.d, ctx.capture = d, _capture(logits.device)
        ctx.mark_non_differentiable(logp, stats)
        return loss, logp, stats

    @staticmethod
    @_once(12)
    def backward(ctx, g, *_):
        logits, target, work, offset = ctx.saved_tensors
        d = ctx.d
        ctx.d = None                       # handed out once: a second pass over a retained graph computes it again
        if d is not None and ctx.capture != _capture(logits.device):
            d = None                       # so does one that is replayed apart from the forward pass, which is each time a pass of its own
        first = d is not None
        if first and head._unit:
            one = head._unit.get(str(logits.device))
            if one is not None and g.data_ptr() == one.data_ptr():          # loss.backward(unit_gradient(device))
                return (d,) + (None,) * 11
        coef = work.data_ptr() + 4 * (ctx.stat + 2 * logits.shape[0])
        return (_backward(ctx, logits, target, offset, work, coef, g, ROW_COEF | (SKIP_UNIT if first else 0), d),) + (None,) * 11


def policy_loss(logits, target, old_logp, advantages, ref_logp=None, offset=None, clip=(0.2, 0.2), kl_coef=0.0, reduction="token", ignore_index=-100):
    """Clipped policy objective.  Per row that counts, with x = log softmax(logits)[target], r = exp(x - old_logp), A = advantages, d = ref_logp - x:
        -min(r A, clamp(r, 1 - clip[0], 1 + clip[1]) A) + kl_coef * (exp(d) - 1 - d)
    old_logp (rows,): token_logprobs of the policy that acted.  advantages: (rows,), or (B, 1): one per sequence of the packed batch.
    ref_logp (rows,): token_logprobs of the reference policy (None: no KL term).
    reduction "token": mean over the rows that count; "sequence": over every sequence's rows, then over the B sequences (one without any row
    that counts adds 0).  Nothing that counts: the loss is 0, its gradient too.
    -> PolicyLoss(loss, logp (rows,), kl, clip_fraction); the last three are detached: x, the mean of exp(d) - 1 - d and the share of rows
    whose ratio was cut off, both weighted like the loss.
    One pass over the logits: the gradient is formed with the loss, and `loss.backward()` hands it out (a pass with another upstream
    gradient than 1, a second one, and one captured without its forward pass compute it again from the logits, with one rounding)."""
    logits, target, offset = _logits(logits, target, offset, old_logp, advantages, ref_logp)
    rows = logits.shape[0]
    if reduction not in ("token", "sequence"):
        raise ValueError(f"policy_loss: reduction={reduction!r} ('token' or 'sequence')")
    if reduction == "sequence" and offset is None:
        raise ValueError("policy_loss: reduction='sequence' needs offset")
    low, high = 1.0 - float(clip[0]), 1.0 + float(clip[1])
    if not (low <= 1.0 <= high):
        raise ValueError("policy_loss: clip must not be negative")
    if advantages.dim() == 2 and offset is None:
        raise ValueError("policy_loss: advantages per sequence need offset")
    adv = _values("advantages", advantages, (rows,) if advantages.dim() != 2 else (offset.numel(), 1), logits)
    old = _values("old_logp", old_logp, (rows,), logits)
    ref = None if ref_logp is None else _values("ref_logp", ref_logp, (rows,), logits)
    loss, logp, stats = _Policy.apply(logits, target, old, adv, ref, offset, low, high, float(kl_coef), reduction == "token", ignore_index,
                                      _wanted(logits))
    return PolicyLoss(loss, logp, *stats.unbind())
