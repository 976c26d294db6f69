"""Adam on the HIP kernel of csrc/adam.hip: the optimizer of the reference's training tools.

`Adam(params, lr, betas, eps, weight_decay)` has torch.optim.Adam's update rule, defaults, `param_groups` (LR schedulers
work on it) and state-dict layout (`step`, `exp_avg`, `exp_avg_sq` per parameter; classification/tool/
train_cls_scanobjectnn.py:179-185 builds it, :166-170 / :261-271 resume from / save its state dict).  The ~70 parameter
tensors of a RepSurf-U classifier are updated by one launch (rs_adam_step takes 80 tensors per launch) instead of the
framework's chunked multi-tensor kernels; learning rate and step count are read from device memory, so a captured step
(graph.GraphedStep) follows a scheduler -- call `sync_hyper()` before each replay, GraphedStep does.
"""
import ctypes
import math

import torch

from . import _lib, mlp_hip

P, c_int, c_ll = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong
MAX_TENSORS = 80          # RS_ADAM_MAX


class AdamTable(ctypes.Structure):           # rs_adam_table
    _fields_ = [("p", P * MAX_TENSORS), ("g", P * MAX_TENSORS), ("m", P * MAX_TENSORS), ("v", P * MAX_TENSORS),
                ("n", c_int * MAX_TENSORS), ("count", c_int)]


class Adam(torch.optim.Optimizer):
    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0):
        if lr < 0.0 or eps < 0.0 or weight_decay < 0.0 or not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
            raise ValueError("Adam: invalid hyper-parameter")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))
        self._dev = {}        # group index -> dict(hyper=device floats, host=last values, step, done)

    # ---- device-side hyper-parameters / counters ---------------------------------------------------------------
    def _group_state(self, gi, group, device):
        st = self._dev.get(gi)
        if st is None:
            st = dict(hyper=torch.zeros(10, dtype=torch.float64, device=device), host=None,      # [5..9]: the kernel's (include/repsurf_hip.h)
                      step=torch.zeros(1, dtype=torch.int32, device=device),
                      done=torch.zeros(1, dtype=torch.int32, device=device))
            self._dev[gi] = st
        return st

    @staticmethod
    def _hyper_values(group):
        return (float(group["lr"]), float(group["betas"][0]), float(group["betas"][1]), float(group["eps"]),
                float(group["weight_decay"]))

    def sync_hyper(self):
        """push changed learning rates etc. to the device (host-side; not capturable -- call it before a replay)"""
        for gi, group in enumerate(self.param_groups):
            st = self._dev.get(gi)
            if st is None:
                continue
            vals = self._hyper_values(group)
            if st["host"] != vals:
                st["hyper"][:5].copy_(torch.tensor(vals, dtype=torch.float64))
                st["host"] = vals

    # ---- state dict in torch.optim.Adam's layout ------------------------------------------------------------------
    def state_dict(self):
        for gi, group in enumerate(self.param_groups):
            st = self._dev.get(gi)
            if st is None:
                continue
            step = float(st["step"].item())
            for p in group["params"]:
                if p in self.state:
                    self.state[p]["step"] = torch.tensor(step, dtype=torch.float32)
        return super().state_dict()

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        for gi, group in enumerate(self.param_groups):
            steps = [float(self.state[p]["step"]) for p in group["params"] if p in self.state and "step" in self.state[p]]
            if steps:
                dev = next(p.device for p in group["params"])
                self._group_state(gi, group, dev)["step"].fill_(int(steps[0]))
        self._dev_reset_host()

    def _dev_reset_host(self):
        for st in self._dev.values():
            st["host"] = None

    # ---- the update -------------------------------------------------------------------------------------------------
    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for gi, group in enumerate(self.param_groups):
            ps = [p for p in group["params"] if p.grad is not None]
            if not ps:
                continue
            dev = ps[0].device
            if dev.type != "cuda":
                raise _lib.RepSurfHipError("repsurf_amd.optim.Adam runs on the HIP device only")
            st = self._group_state(gi, group, dev)
            if st["host"] is None:
                if torch.cuda.is_current_stream_capturing():
                    raise _lib.RepSurfHipError("repsurf_amd.optim.Adam: run one eager step (or sync_hyper()) before capture")
                self.sync_hyper()
            stream = _lib.current_stream()
            keep = []
            for c0 in range(0, len(ps), MAX_TENSORS):
                chunk = ps[c0:c0 + MAX_TENSORS]
                tab = AdamTable()
                for i, p in enumerate(chunk):
                    if p.dtype != torch.float32 or not p.is_contiguous():
                        raise _lib.RepSurfHipError("repsurf_amd.optim.Adam: parameters must be contiguous fp32")
                    s = self.state[p]
                    if "exp_avg" not in s:
                        s["exp_avg"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                        s["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                        s["step"] = torch.tensor(0.0)
                    g = p.grad if p.grad.is_contiguous() else p.grad.contiguous()
                    keep.append(g)
                    tab.p[i], tab.g[i], tab.m[i], tab.v[i] = p.data_ptr(), g.data_ptr(), s["exp_avg"].data_ptr(), \
                        s["exp_avg_sq"].data_ptr()
                    tab.n[i] = p.numel()
                tab.count = len(chunk)
                last = c0 + MAX_TENSORS >= len(ps)
                _lib.call("rs_adam_step", ctypes.byref(tab), st["hyper"].data_ptr(), st["step"].data_ptr(),
                          st["done"].data_ptr(), 1 if last else 0, stream)
        mlp_hip.weights_changed()       # raw-pointer update: tensor._version does not move (mlp_hip._prepacked)
        return loss


# ---------------------------------------------------------------------------------------------------------------- AdamW
BLOCK = 256               # tensors start at multiples of it in the flat moment buffers; elements that share an 8-bit exponent
GRAD_SQUARE_SUMS, DONE = 1024, 528      # RS_GRAD_SQUARE_SUMS, RS_ADAMW_DONE


class AdamWList(ctypes.Structure):           # rs_adamw_list
    _fields_ = [("count", c_int), ("p", P), ("g", P), ("n", P), ("at", P), ("slot", P)]


class AdamWArgs(ctypes.Structure):           # rs_adamw_args
    _fields_ = [("bits", c_int), ("bf16", c_int), ("exp_avg", P), ("exp_avg_sq", P), ("exp_avg_exponent", P), ("exp_avg_sq_exponent", P),
                ("low", P), ("step", P), ("done", P), ("hyper_dev", P), ("hyper", ctypes.c_double * 7), ("clip", P), ("seed", ctypes.c_uint)]


_address, _dense, _size, _type = torch.Tensor.data_ptr, torch.Tensor.is_contiguous, torch.Tensor.numel, torch.Tensor.dtype.__get__
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


class _Table:
    """The host arrays of one rs_adamw_list: tensors of one type in one group."""

    def __init__(self, rows):
        n = len(rows)
        self.p, self.g = (P * n)(*[r[0] for r in rows]), (P * n)(*[r[1] for r in rows])
        self.n, self.at = (c_ll * n)(*[r[2] for r in rows]), (c_ll * n)(*[r[3] for r in rows])
        self.slot = (c_int * n)(*[r[4] for r in rows])
        self.count = n
        self.list = AdamWList(n, *[ctypes.cast(a, P) for a in (self.p, self.g, self.n, self.at, self.slot)])
        self.ref = ctypes.byref(self.list)
        self.args = self.vals = None         # the rs_adamw_args of these tensors' launches, and the hyper-parameters in it


class AdamW(Adam):
    """torch.optim.AdamW's update (decoupled weight decay), arguments, `param_groups` and state-dict layout over many tensors at once, on
    csrc/adamw.hip: the optimizer that the reference's segmentation loop builds (segmentation/tool/train.py).

    Parameters are contiguous tensors in fp32, or in bf16 -- these keep, beside the moments, the 16 bits that their fp32 master has below
    them (`low`), so a step smaller than bf16's spacing is not lost; a parameter that is written from outside moves its master with it.  Such a
    parameter is its master rounded to nearest, halves away from zero (torch: to even): 16 signed bits hold what is below it.
    state_bits=8 holds both moments in one byte per element and one exponent per 256 (include/repsurf_hip.h has the format): 4 bytes
    of state traffic per parameter instead of 16.  Values are rounded stochastically by a fixed function of (seed, step, element): the
    same run gives the same bits.  max_grad_norm=x multiplies every gradient by min(1, x / (norm + 1e-6)), norm being that of all
    gradients of the step (torch.nn.utils.clip_grad_norm_ with its update fused into the step: p.grad stays as it is);
    `grad_norm` is that norm, a device scalar that the next step overwrites.

    Every parameter counts its own steps, on the device: one without a gradient is left out and its bias correction waits, and a
    captured step (graph.GraphedStep, graph.TrainLoopStep) counts its replays.  Hyper-parameters ride in an eager step's launch; a
    captured one reads them from device memory -- `sync_hyper()` before a replay, as the graphed steps do (max_grad_norm, the seed and
    whether gradients are clipped at all stay what they were at the capture).

    The moments of a group are slices of flat buffers (`flat_state`), every tensor at a multiple of 256 elements; `state_dict()` brings
    `state[p]["step"]` up to date from the device's counters."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, state_bits=32, max_grad_norm=None, seed=0):
        if state_bits not in (8, 32):
            raise ValueError(f"AdamW: state_bits={state_bits} (32 or 8)")
        if max_grad_norm is not None and not max_grad_norm > 0.0:
            raise ValueError("AdamW: max_grad_norm must be positive")
        super().__init__(params, lr=lr, betas=betas, eps=eps, weight_decay=weight_decay)
        self.state_bits, self.max_grad_norm, self.seed = state_bits, max_grad_norm, int(seed) & 0xFFFFFFFF
        self._norm, self._partial = None, []          # (the newest buffer of partial sums last: a captured step may hold an older one)

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        ids = [id(p) for p in self.param_groups[-1]["params"]]
        if len(set(ids)) != len(ids):
            self.param_groups.pop()
            raise ValueError("AdamW: a parameter appears twice in a group")

    @property
    def grad_norm(self):
        """norm of the last step's gradients (device scalar); None without max_grad_norm"""
        return self._norm

    # ---- state ------------------------------------------------------------------------------------------------------
    def _group_state(self, gi, group, device):
        st = self._dev.get(gi)
        params = group["params"]
        if st is None:
            if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
                raise _lib.RepSurfHipError("repsurf_amd.optim.AdamW: run one eager step before capture")
            at, end = [], 0
            for p in params:
                self._check_param(p, device)
                at.append(end)
                end += (p.numel() + BLOCK - 1) // BLOCK * BLOCK
            new = lambda n, dtype: torch.zeros((n,), dtype=dtype, device=device)      # noqa: E731
            kind = torch.float32 if self.state_bits == 32 else torch.uint8
            flat = {"exp_avg": new(end, kind), "exp_avg_sq": new(end, kind)}
            if self.state_bits == 8:
                flat.update(exp_avg_exponent=new(end // BLOCK, torch.uint8), exp_avg_sq_exponent=new(end // BLOCK, torch.uint8))
            if any(p.dtype == torch.bfloat16 for p in params):
                flat["low"] = new(end, torch.int16)
            st = dict(hyper=new(7, torch.float64), host=None, step=new(len(params), torch.int32), done=new(DONE, torch.int32),
                      flat=flat, at=at, end=end, sizes=[p.numel() for p in params], ids=[id(p) for p in params], plan=None, tables=None, key=None, vals=None)
            self._dev[gi] = st
            for p, a in zip(params, at):
                self._views(st, p, a)
        elif st["ids"] != list(map(id, params)):
            raise _lib.RepSurfHipError("repsurf_amd.optim.AdamW: the parameters of a group changed after its state was made")
        return st

    def _views(self, st, p, a):
        s, n = self.state[p], p.numel()
        s["step"] = torch.tensor(0.0)
        for k, buf in st["flat"].items():
            if k.endswith("exponent"):
                s[k] = buf[a // BLOCK:(a + n + BLOCK - 1) // BLOCK]
            elif k != "low" or p.dtype == torch.bfloat16:
                s[k] = buf[a:a + n].view(p.shape)

    @staticmethod
    def _check_param(p, device):
        if p.device != device or device.type != "cuda":
            raise _lib.RepSurfHipError("repsurf_amd.optim.AdamW runs on the HIP device only, a group on one device")
        if p.dtype not in (torch.float32, torch.bfloat16) or p.layout != torch.strided or not p.is_contiguous():
            raise _lib.RepSurfHipError("repsurf_amd.optim.AdamW: parameters must be contiguous fp32 or bf16")

    @staticmethod
    def _hyper_values(group):
        lr, (b1, b2), eps, wd = float(group["lr"]), group["betas"], float(group["eps"]), float(group["weight_decay"])
        ln = lambda b: math.log(b) if b > 0.0 else -math.inf      # noqa: E731
        return (lr, float(b1), float(b2), eps, wd, ln(float(b1)), ln(float(b2)))

    def sync_hyper(self):
        """push changed learning rates etc. to the device, for captured steps (host-side; not capturable -- call it before a replay)"""
        for gi, group in enumerate(self.param_groups):
            st = self._dev.get(gi)
            if st is None:
                continue
            vals = self._hyper_values(group)
            if st["host"] != vals:
                st["hyper"].copy_(torch.tensor(vals, dtype=torch.float64))
                st["host"] = vals

    def flat_state(self, group=0):
        """the buffers that hold a group's moments: {"exp_avg", "exp_avg_sq"} and, where they exist, {"exp_avg_exponent",
        "exp_avg_sq_exponent", "low"}; tensor i starts at the sum of the sizes before it, each rounded up to 256"""
        if group not in self._dev:
            raise _lib.RepSurfHipError("repsurf_amd.optim.AdamW: no state yet (it is made by the first step, or by load_state_dict)")
        return dict(self._dev[group]["flat"])

    @torch.no_grad()
    def unpack_state(self, group=0, dtype=torch.float32):
        """a group's moments as flat values in `dtype` (fp32, or bf16), laid out like `flat_state`; with bf16 parameters also "master", their
        fp32 masters.  32-bit moments asked for in fp32 are the buffers themselves."""
        flat = self.flat_state(group)
        st, params = self._dev[group], self.param_groups[group]["params"]
        if dtype not in (torch.float32, torch.bfloat16):
            raise ValueError(f"AdamW.unpack_state: {dtype} (fp32 or bf16)")
        dev = st["step"].device
        with torch.cuda.device(dev):
            if self.state_bits == 32:
                out = {k: flat[k].to(dtype) for k in ("exp_avg", "exp_avg_sq")}
            else:
                out = {k: torch.empty((st["end"],), dtype=dtype, device=dev) for k in ("exp_avg", "exp_avg_sq")}
                _lib.call("rs_adamw_unpack", st["end"], flat["exp_avg"].data_ptr(), flat["exp_avg_sq"].data_ptr(),
                          flat["exp_avg_exponent"].data_ptr(), flat["exp_avg_sq_exponent"].data_ptr(), int(dtype == torch.bfloat16),
                          out["exp_avg"].data_ptr(), out["exp_avg_sq"].data_ptr(), _lib.current_stream())
            if "low" in flat:
                rows = [(p.data_ptr(), p.data_ptr(), p.numel(), a, i) for i, (p, a) in enumerate(zip(params, st["at"]))
                        if p.dtype == torch.bfloat16 and p.numel()]
                all_bf16 = len(rows) == sum(p.numel() > 0 for p in params)          # (the call writes its tensors' room whole)
                out["master"] = (torch.empty if all_bf16 else torch.zeros)((st["end"],), dtype=torch.float32, device=dev)
                if rows:
                    _lib.call("rs_adamw_masters", _Table(rows).ref, flat["low"].data_ptr(), out["master"].data_ptr(), _lib.current_stream())
        return out

    # ---- state dict: torch.optim.AdamW's keys; 8-bit states and masters' low halves under keys of their own ---------------
    def state_dict(self):
        for gi, group in enumerate(self.param_groups):
            st = self._dev.get(gi)
            if st is not None:
                for p, t in zip(group["params"], st["step"].tolist()):
                    self.state[p]["step"] = torch.tensor(float(t), dtype=torch.float32)
        return torch.optim.Optimizer.state_dict(self)

    @torch.no_grad()
    def load_state_dict(self, state_dict):
        """Takes its own state dicts and torch.optim.AdamW's; fp32 moments are rounded to 8 bits (to nearest) where state_bits is 8, and
        8-bit ones are refused where it is 32.  The values are copied; a parameter without any starts anew."""
        bits = {32 if v["exp_avg"].is_floating_point() else 8 for v in state_dict["state"].values() if "exp_avg" in v}
        if len(bits) > 1 or (bits == {8} and self.state_bits == 32):
            raise ValueError("AdamW.load_state_dict: 8-bit moments need state_bits=8 (and all of them)")
        if any(k in v and k + "_exponent" not in v for v in state_dict["state"].values() for k in ("exp_avg", "exp_avg_sq") if 8 in bits):
            raise ValueError("AdamW.load_state_dict: 8-bit moments without their exponents")
        if any(sg.get("amsgrad") or sg.get("maximize") for sg in state_dict["param_groups"]):
            raise ValueError("AdamW.load_state_dict: amsgrad and maximize are not offered")
        order = [list(sg["params"]) for sg in state_dict["param_groups"]]
        for sg, group in zip(order, self.param_groups):
            for k, p in zip(sg, group["params"]):
                saved = state_dict["state"].get(k, {})
                for name, v in saved.items():
                    if name in ("exp_avg", "exp_avg_sq", "low") and tuple(v.shape) != tuple(p.shape):
                        raise ValueError(f"AdamW.load_state_dict: {name} of parameter {k} has shape {tuple(v.shape)}, the parameter {tuple(p.shape)}")
                    if name.endswith("_exponent") and tuple(v.shape) != ((p.numel() + BLOCK - 1) // BLOCK,):
                        raise ValueError(f"AdamW.load_state_dict: {name} of parameter {k} has shape {tuple(v.shape)}, one per {BLOCK} elements are needed")
                if ("exp_avg" in saved) != ("exp_avg_sq" in saved):
                    raise ValueError(f"AdamW.load_state_dict: parameter {k} has one moment without the other")
        # state_dict() hands out views of the buffers that are written below: such values are read whole before anything is
        own = {buf.untyped_storage().data_ptr() for st in self._dev.values() for buf in st["flat"].values()}
        kept = lambda v: v.clone() if torch.is_tensor(v) and v.untyped_storage().data_ptr() in own else v      # noqa: E731
        state = {k: {name: kept(v) for name, v in s.items()} for k, s in state_dict["state"].items()}
        super(Adam, self).load_state_dict({"state": {}, "param_groups": state_dict["param_groups"]})
        for gi, (keys, group) in enumerate(zip(order, self.param_groups)):
            saved = [state.get(k, {}) for k in keys]
            if gi not in self._dev and not any("exp_avg" in s for s in saved):
                continue
            dev = group["params"][0].device
            st = self._group_state(gi, group, dev)          # (what is there is written in place: a captured step keeps its addresses)
            for buf in st["flat"].values():
                buf.zero_()
            for p, a in zip(group["params"], st["at"]):
                self._views(st, p, a)
            wide = None
            if self.state_bits == 8 and bits == {32}:
                wide = {k: torch.zeros((st["end"],), dtype=torch.float32, device=dev) for k in ("exp_avg", "exp_avg_sq")}
            to, of = [], []
            for p, a, s in zip(group["params"], st["at"], saved):
                for name, v in s.items():
                    if wide is not None and name in wide:
                        to.append(wide[name][a:a + p.numel()])
                        of.append(v.reshape(-1))
                    elif name != "step" and name in self.state[p]:
                        to.append(self.state[p][name])
                        of.append(v)
            if to:
                torch._foreach_copy_(to, of)
            if wide is not None:
                f = st["flat"]
                with torch.cuda.device(dev):
                    _lib.call("rs_adamw_pack", st["end"], wide["exp_avg"].data_ptr(), wide["exp_avg_sq"].data_ptr(), f["exp_avg"].data_ptr(),
                              f["exp_avg_sq"].data_ptr(), f["exp_avg_exponent"].data_ptr(), f["exp_avg_sq_exponent"].data_ptr(), _lib.current_stream())
            steps = [int(float(s.get("step", 0))) for s in saved]
            st["step"].copy_(torch.tensor(steps, dtype=torch.int32))

    # ---- the update ---------------------------------------------------------------------------------------------------
    def _tables(self, st, params):
        """the group's lists (fp32, bf16), rebuilt when an address, a size or a type changed since the last step"""
        grads = [p.grad for p in params]
        try:
            at, some = list(map(_address, grads)), grads
        except (TypeError, RuntimeError):          # (None among them, or one without an address)
            some = [g for g in grads if g is not None]
            if any(g.layout is not torch.strided for g in some):
                raise _lib.RepSurfHipError("repsurf_amd.optim.AdamW: gradients must be dense and of their parameter's type")
            at = list(map(_address, some)) + [g is None for g in grads]
        # (a gradient has its parameter's shape)
        plan = (list(map(_address, params)), list(map(_size, params)), list(map(_type, params)), at, list(map(_type, some)))
        if plan == st["plan"] and all(map(_dense, some)) and all(map(_dense, params)):
            return st["tables"], None
        rows, keep, seen = ([], []), [], set()
        for i, (p, g) in enumerate(zip(params, grads)):
            if g is None or p.numel() == 0:
                continue
            self._check_param(p, st["step"].device)
            if p.dtype == torch.bfloat16 and "low" not in st["flat"]:
                raise _lib.RepSurfHipError("repsurf_amd.optim.AdamW: a parameter became bf16 after its state was made, without a master's low half")
            if p.numel() != st["sizes"][i] or g.shape != p.shape:
                raise _lib.RepSurfHipError("repsurf_amd.optim.AdamW: a parameter has another size than its state or its gradient")
            if g.layout != torch.strided or g.dtype != p.dtype:
                raise _lib.RepSurfHipError("repsurf_amd.optim.AdamW: gradients must be dense and of their parameter's type")
            if p.data_ptr() in seen:
                raise _lib.RepSurfHipError("repsurf_amd.optim.AdamW: two parameters of a group share their memory")
            seen.add(p.data_ptr())
            if not g.is_contiguous():
                g = g.detach().contiguous()
                keep.append(g)
            rows[p.dtype == torch.bfloat16].append((p.data_ptr(), g.data_ptr(), p.numel(), st["at"][i], i))
        tables = [(bf16, _Table(r)) for bf16, r in enumerate(rows) if r]
        st["plan"], st["tables"] = (None, None) if keep else (plan, tables)
        return tables, keep

    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        work, dev = [], None
        for gi, group in enumerate(self.param_groups):
            params = group["params"]
            first = next((p for p in params if p.grad is not None), None)
            if first is None:
                continue
            if dev is not None and first.device != dev:
                raise _lib.RepSurfHipError("repsurf_amd.optim.AdamW: all groups must be on one device")
            dev = first.device
            st = self._group_state(gi, group, dev)
            work.append((gi, group, st) + self._tables(st, params))
        if not work:
            return loss
        if dev.index != _current_device():
            with torch.cuda.device(dev):
                self._launch(work, dev)
        else:
            self._launch(work, dev)
        mlp_hip.weights_changed()       # raw-pointer update: tensor._version does not move (mlp_hip._prepacked)
        return loss

    def _launch(self, work, dev):
        stream, capturing = _lib.current_stream(), torch.cuda.is_current_stream_capturing()
        clip = None
        if self.max_grad_norm is not None:
            launches = lambda ps: (len(ps) + MAX_TENSORS - 1) // MAX_TENSORS + 1      # noqa: E731   (fp32 and bf16 ones apart)
            room = GRAD_SQUARE_SUMS * sum(launches(g["params"]) for g in self.param_groups)
            if not self._partial or self._partial[-1].numel() < room:
                if capturing:
                    raise _lib.RepSurfHipError("repsurf_amd.optim.AdamW: run one eager step before capture")
                if self._norm is None:
                    self._factors = torch.zeros((2,), dtype=torch.float32, device=dev)          # the norm, and what the gradients are multiplied by
                    self._norm = self._factors[0]
                self._partial.append(torch.empty((room,), dtype=torch.float64, device=dev))
            partial = self._partial[-1].data_ptr()
            n, used = c_int(), 0
            for w in work:
                for bf16, t in w[3]:
                    _lib.call("rs_grad_square_sums", t.ref, bf16, partial + 8 * used, room - used, ctypes.byref(n), stream)
                    used += n.value
            if used:
                _lib.call("rs_grad_norm", used, partial, self.max_grad_norm, self._factors.data_ptr(), stream)
                clip = self._factors.data_ptr() + 4
        for gi, group, st, tables, _ in work:
            key = (float(group["lr"]), tuple(group["betas"]), group["eps"], group["weight_decay"])
            if st["key"] != key:
                st["key"], st["vals"] = key, self._hyper_values(group)
            if st["host"] is None:
                if capturing:
                    raise _lib.RepSurfHipError("repsurf_amd.optim.AdamW: run one eager step (or sync_hyper()) before capture")
                self.sync_hyper()
            for bf16, t in tables:
                a = t.args
                if a is None:
                    a = t.args = self._args(gi, st, bf16)
                if t.vals is not st["vals"]:
                    a.hyper[:], t.vals = st["vals"], st["vals"]
                a.hyper_dev = st["hyper"].data_ptr() if capturing else None
                a.clip = clip
                _lib.call("rs_adamw_step", t.ref, ctypes.byref(a), stream)

    def _args(self, gi, st, bf16):
        ptr = lambda k: st["flat"][k].data_ptr() if k in st["flat"] else None      # noqa: E731
        return AdamWArgs(bits=self.state_bits, bf16=bf16, exp_avg=ptr("exp_avg"), exp_avg_sq=ptr("exp_avg_sq"),
                         exp_avg_exponent=ptr("exp_avg_exponent"), exp_avg_sq_exponent=ptr("exp_avg_sq_exponent"), low=ptr("low"),
                         step=st["step"].data_ptr(), done=st["done"].data_ptr(), seed=(self.seed + gi * 0x3C6EF372) & 0xFFFFFFFF)
