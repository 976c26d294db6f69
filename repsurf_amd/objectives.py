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
(once); the other tensors are data.  The calls allocate through torch and can be captured into a graph once they ran eagerly."""
import ctypes
from collections import namedtuple

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import _lib, head

P, c_int, c_ll, c_double = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_double
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
POLICY_COUNTS, POLICY_PARTIAL = 64, 6144          # RS_POLICY_COUNTS, RS_POLICY_PARTIAL
FEW_ROWS, PARTS = 256, 64                         # RS_LOGITS_FEW_ROWS, RS_LOGITS_PARTS

PolicyLoss = namedtuple("PolicyLoss", "loss logp kl clip_fraction")
PreferenceLoss = namedtuple("PreferenceLoss", "loss chosen_rewards rejected_rewards")


class LogitsDesc(ctypes.Structure):          # rs_logits
    _fields_ = [("logits", P), ("rows", c_ll), ("ld", c_ll), ("classes", c_int), ("type", c_int), ("target", P), ("ignore_index", c_ll),
                ("offset", P), ("sequences", c_int), ("bad_labels", P)]


class PolicyDesc(ctypes.Structure):          # rs_policy
    _fields_ = [("old_logp", P), ("advantages", P), ("ref_logp", P), ("advantages_per_sequence", c_int), ("token_mean", c_int), ("low", c_double),
                ("high", c_double), ("kl_coef", c_double), ("counts", P), ("counts_room", c_int), ("partial", P), ("partial_room", c_int),
                ("loss", P), ("stats", P), ("logp", P), ("dlogits", P), ("coef", P), ("stat", P), ("scratch", P)]


def _logits(logits, target, offset):
    """checks, and the tensors as the kernels take them"""
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError(f"objectives: logits must be (rows, classes), got {tuple(logits.shape)}")
    if logits.dtype not in _TYPES:
        raise TypeError(f"objectives: logits must be fp32, bf16 or fp16, got {logits.dtype}")
    if target.shape != logits.shape[:1] or target.is_floating_point():
        raise ValueError(f"objectives: target must hold one class index per row, got {tuple(target.shape)} {target.dtype}")
    if offset is not None and (offset.dim() != 1 or offset.numel() < 1 or offset.is_floating_point()):
        raise ValueError("objectives: offset must be the (B,) running row ends")
    for t in (logits, target, offset):
        if t is not None and t.device != logits.device:
            raise ValueError("objectives: all tensors must be on the logits' device")
    if not logits.is_cuda:
        raise _lib.RepSurfHipError("repsurf_amd.objectives run on the HIP device only (got a CPU tensor); there is no CPU fallback")
    if logits.shape[0] and (logits.stride(1) != 1 or logits.stride(0) < logits.shape[1]):
        logits = logits.contiguous()
    target = target.to(torch.int64).contiguous()
    if offset is not None:
        offset = offset.to(torch.int32).contiguous()
    return logits, target, offset


def _values(name, t, shape, logits):
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"objectives: {name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.device != logits.device:
        raise ValueError("objectives: all tensors must be on the logits' device")
    return t.detach().to(torch.float32).contiguous()


def _desc(logits, target, ignore_index, offset):
    rows, classes = logits.shape
    return LogitsDesc(logits=logits.data_ptr(), rows=rows, ld=max(logits.stride(0), classes), classes=classes, type=_TYPES[logits.dtype],
                      target=target.data_ptr(), ignore_index=int(ignore_index), offset=None if offset is None else offset.data_ptr(),
                      sequences=0 if offset is None else offset.numel(), bad_labels=head._bad_counter(logits.device).data_ptr())


def _backward(desc, logits, stat, coef, gout, skip_unit, out):
    _lib.call("rs_token_logprobs_backward", ctypes.byref(desc), stat.data_ptr(), coef.data_ptr(), None if gout is None else gout.data_ptr(),
              skip_unit, out.data_ptr(), _lib.current_stream())
    return out


def _wanted(logits):
    return logits.requires_grad and torch.is_grad_enabled()


def _new(logits, *shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device=logits.device)


def _scratch(logits):
    """room for the pieces of a few long rows, or None"""
    rows, classes = logits.shape
    return None if rows > FEW_ROWS or classes <= 8192 else _new(logits, 3 * PARTS * rows)


class _TokenLogprobs(Function):
    @staticmethod
    def forward(ctx, logits, target, ignore_index, grad):
        rows = logits.shape[0]
        logp = _new(logits, rows)
        stat, scratch = _new(logits, rows, 2) if grad else None, _scratch(logits)
        with torch.cuda.device(logits.device):
            _lib.call("rs_token_logprobs", ctypes.byref(_desc(logits, target, ignore_index, None)), logp.data_ptr(), None,
                      None if stat is None else stat.data_ptr(), None if scratch is None else scratch.data_ptr(), _lib.current_stream())
        if stat is not None:
            ctx.save_for_backward(logits, target, stat)
            ctx.ignore_index = ignore_index
        return logp

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        logits, target, stat = ctx.saved_tensors
        with torch.cuda.device(logits.device):
            d = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
            return _backward(_desc(logits, target, ctx.ignore_index, None), logits, stat, g.to(torch.float32).contiguous(), None, 0, d), None, None, None


def token_logprobs(logits, target, ignore_index=-100):
    """logits (rows, classes), target (rows,) -> (rows,) fp32: log softmax(logits)[target], 0 for rows that do not count.  Reads the logits once;
    differentiable in them."""
    logits, target, _ = _logits(logits, target, None)
    return _TokenLogprobs.apply(logits, target, ignore_index, _wanted(logits))


def _sequences(logits, target, offset, ignore_index, average, stat):
    """-> (desc, sums fp64, sums fp32, each): a row's factor in its sequence's sum"""
    n = offset.numel()
    logp, sums = _new(logits, logits.shape[0], dtype=torch.float64), _new(logits, n, dtype=torch.float64)
    out, each = _new(logits, n), _new(logits, n)
    desc = _desc(logits, target, ignore_index, offset)
    scratch = _scratch(logits)
    _lib.call("rs_token_logprobs", ctypes.byref(desc), None, logp.data_ptr(), None if stat is None else stat.data_ptr(),
              None if scratch is None else scratch.data_ptr(), _lib.current_stream())
    _lib.call("rs_sequence_sums", ctypes.byref(desc), logp.data_ptr(), int(average), sums.data_ptr(), out.data_ptr(), each.data_ptr(),
              _lib.current_stream())
    return desc, sums, out, each


class _SequenceLogprobs(Function):
    @staticmethod
    def forward(ctx, logits, target, offset, ignore_index, average, grad):
        stat = _new(logits, logits.shape[0], 2) if grad else None
        with torch.cuda.device(logits.device):
            _, _, out, each = _sequences(logits, target, offset, ignore_index, average, stat)
        if stat is not None:
            ctx.save_for_backward(logits, target, offset, stat, each)
            ctx.ignore_index = ignore_index
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        logits, target, offset, stat, each = ctx.saved_tensors
        with torch.cuda.device(logits.device):
            d = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
            d = _backward(_desc(logits, target, ctx.ignore_index, offset), logits, stat, g.to(torch.float32) * each, None, 0, d)
        return d, None, None, None, None, None


def sequence_logprobs(logits, target, offset, ignore_index=-100, average=False):
    """(B,) fp32: the sum of token_logprobs over every sequence of a packed batch, or (average) their mean over the rows that count; 0 for
    a sequence without any.  Differentiable in the logits."""
    logits, target, offset = _logits(logits, target, offset)
    return _SequenceLogprobs.apply(logits, target, offset, ignore_index, average, _wanted(logits))


class _Preference(Function):
    @staticmethod
    def forward(ctx, logits, target, offset, ref, beta, smoothing, average, ignore_index, grad):
        n = offset.numel()
        stat = _new(logits, logits.shape[0], 2) if grad else None
        loss, rewards, coef = _new(logits), _new(logits, n), _new(logits, n)
        with torch.cuda.device(logits.device):
            _, sums, _, each = _sequences(logits, target, offset, ignore_index, average, stat)
            _lib.call("rs_preference_pairs", n // 2, sums.data_ptr(), each.data_ptr(), ref.data_ptr(), float(beta), float(smoothing), loss.data_ptr(),
                      rewards.data_ptr(), coef.data_ptr(), _lib.current_stream())
        if stat is not None:
            ctx.save_for_backward(logits, target, offset, stat, coef)
            ctx.ignore_index = ignore_index
        ctx.mark_non_differentiable(rewards)
        return loss, rewards

    @staticmethod
    @once_differentiable
    def backward(ctx, g, _):
        logits, target, offset, stat, coef = ctx.saved_tensors
        with torch.cuda.device(logits.device):
            d = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
            d = _backward(_desc(logits, target, ctx.ignore_index, offset), logits, stat, coef, g.to(torch.float32).contiguous(), 0, d)
        return (d,) + (None,) * 8


def preference_loss(logits, target, offset, ref_logps, beta=0.1, label_smoothing=0.0, average=False, ignore_index=-100):
    """Paired log ratios.  The packed batch holds 2 P sequences, the P chosen ones first: sequence i is preferred to sequence P + i.  With
    r = beta * (sequence_logprobs(logits) - ref_logps) and h = r[i] - r[P + i],
        loss = mean of -(1 - label_smoothing) log sigmoid(h) - label_smoothing log sigmoid(-h).
    ref_logps (2 P,): sequence_logprobs of the reference model's logits (same `average`).
    -> PreferenceLoss(loss, chosen_rewards, rejected_rewards); the rewards (P,) are r, detached."""
    logits, target, offset = _logits(logits, target, offset)
    n = offset.numel()
    if n % 2:
        raise ValueError(f"preference_loss: {n} sequences are no pairs")
    if not 0.0 <= label_smoothing <= 0.5:
        raise ValueError("preference_loss: label_smoothing must lie in [0, 0.5]")
    ref = _values("ref_logps", ref_logps, (n,), logits)
    loss, rewards = _Preference.apply(logits, target, offset, ref, beta, label_smoothing, average, ignore_index, _wanted(logits))
    return PreferenceLoss(loss, rewards[: n // 2], rewards[n // 2:])


class _Policy(Function):
    @staticmethod
    def forward(ctx, logits, target, old, adv, ref, offset, low, high, kl_coef, token_mean, ignore_index, grad):
        rows = logits.shape[0]
        loss, stats, logp = _new(logits), _new(logits, 2), _new(logits, rows)
        d = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device) if grad else None
        row = _new(logits, rows, 3) if grad else None                # coef, and stat behind it
        room = POLICY_COUNTS * (1 if token_mean else offset.numel())
        counts, partial = _new(logits, room, dtype=torch.int32), _new(logits, POLICY_PARTIAL, dtype=torch.float64)
        desc = _desc(logits, target, ignore_index, offset)
        p = PolicyDesc(old_logp=old.data_ptr(), advantages=adv.data_ptr(), ref_logp=None if ref is None else ref.data_ptr(),
                       advantages_per_sequence=int(adv.dim() == 2), token_mean=int(token_mean), low=low, high=high, kl_coef=kl_coef,
                       counts=counts.data_ptr(), counts_room=room, partial=partial.data_ptr(), partial_room=POLICY_PARTIAL, loss=loss.data_ptr(),
                       stats=stats.data_ptr(), logp=logp.data_ptr())
        scratch = _scratch(logits)
        if scratch is not None:
            p.scratch = scratch.data_ptr()
        if grad and rows:
            p.dlogits, p.coef, p.stat = d.data_ptr(), row.data_ptr(), row.data_ptr() + 4 * rows
        with torch.cuda.device(logits.device):
            _lib.call("rs_policy_loss", ctypes.byref(desc), ctypes.byref(p), _lib.current_stream())
        if grad:
            ctx.save_for_backward(logits, target, offset, row)
            ctx.d, ctx.ignore_index = d, ignore_index
        ctx.mark_non_differentiable(logp, stats)
        return loss, logp, stats

    @staticmethod
    @once_differentiable
    def backward(ctx, g, *_):
        logits, target, offset, row = ctx.saved_tensors
        d, first = ctx.d, ctx.d is not None
        ctx.d = None                       # handed out once: a second pass over a retained graph computes it again
        one = head._unit.get(str(logits.device))
        if first and ((one is not None and g.data_ptr() == one.data_ptr()) or logits.shape[0] == 0):      # loss.backward(unit_gradient(device))
            return (d,) + (None,) * 11
        with torch.cuda.device(logits.device):
            if not first:
                d = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
            if logits.shape[0]:
                # per-row coefficients: the offsets were taken into account when they were made
                _lib.call("rs_token_logprobs_backward", ctypes.byref(_desc(logits, target, ctx.ignore_index, None)), row.data_ptr() + 4 * logits.shape[0],
                          row.data_ptr(), g.to(torch.float32).contiguous().data_ptr(), int(first), d.data_ptr(), _lib.current_stream())
        return (d,) + (None,) * 11


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
    gradient than 1 computes it again from the logits, with one rounding)."""
    logits, target, offset = _logits(logits, target, offset)
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
    return PolicyLoss(loss, logp, stats[0], stats[1])
