"""Trainer-side glue of the hot path: the reference trains with torch.optim.Adam over ~90 small parameter
tensors per GCPInteractions layer (configs/model/gcpnet_nms.yaml:8-12, gcpnet_lba.yaml); FusedAdam applies the same update to all
of them in one HIP launch per 96 tensors (gcpnet_adam_step) instead of several launches per tensor."""
from __future__ import annotations

import ctypes as C
import itertools
import operator
from typing import Iterable, Optional

import torch

from . import _lib, ops
from ._lib import AdamTensor, AdamWTensor, check


class FusedAdam(torch.optim.Optimizer):
    """torch.optim.Adam(params, lr, betas, eps, weight_decay) semantics (amsgrad=False, maximize=False, L2 weight decay added to
    the gradient), state keys `step`, `exp_avg`, `exp_avg_sq` as in torch (state_dicts interchange).  fp32 CUDA parameters."""

    def __init__(self, params: Iterable, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.0,
                 capturable: bool = False):
        """capturable: the step count lives in device memory (one int64 per parameter group, advanced by the update itself:
        gcpnet_adam_step_dev), state["step"] is that tensor as in torch.optim.Adam(capturable=True), and step() may be captured
        into a hipGraph (gcpnet_amd.graphs.GraphedStep(step_fn, optimizer=...)).  lr / betas / eps / weight_decay are frozen into
        a capture; every parameter of a group must take part from the first step on."""
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, capturable=capturable))
        # capturable groups: the device step counter and the parameters that take part, by group index.  NOT in param_groups:
        # torch serialises every key of a group, and a counter that came back from torch.load(map_location="cpu") would hand a
        # host pointer to the kernel; load_state_dict drops them and the next step rebuilds them from state["step"]
        self._step_dev = {}
        self._members = {}

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        self._step_dev, self._members = {}, {}

    def __setstate__(self, state):
        super().__setstate__(state)
        self._step_dev, self._members = {}, {}
        for g in self.param_groups:
            g.pop("_step_dev", None)  # (pickles of the earlier layout)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        capturing = torch.cuda.is_available() and torch.cuda.is_current_stream_capturing()
        lib = _lib.load()
        for gi, group in enumerate(self.param_groups):
            if group.get("capturable"):
                self._step_capturable(lib, group, gi)
                continue
            if capturing:
                # the step count and the bias corrections derived from it are host values passed as kernel arguments: a captured
                # step() would replay the capture-time corrections for ever and state["step"] would stop advancing
                raise RuntimeError("FusedAdam.step() with a host-side step count cannot be captured into a hipGraph: construct the "
                                   "optimizer with capturable=True, or call it eagerly after GraphedStep's replay")
            items, step = [], None
            for p in group["params"]:
                if p.grad is None:
                    continue
                if not p.is_cuda or p.dtype != torch.float32:
                    raise _lib.GcpnetHipError("FusedAdam: fp32 parameters on the GPU only (gcpnet_amd has no CPU path)")
                st = self.state[p]
                if not st:
                    st["step"] = 0
                    st["exp_avg"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
                    st["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
                st["step"] = int(st["step"]) + 1
                if step is None:
                    step = st["step"]
                if st["step"] != step:  # (parameters that joined later: their own launch)
                    self._launch(lib, group, [(p, st)], st["step"])
                    continue
                items.append((p, st))
            if items:
                self._launch(lib, group, items, step)
        ops.invalidate_packs()  # (p.data was written through a raw pointer: the packed-weight caches must not outlive it)
        return loss

    def _step_capturable(self, lib, group, gi):
        """One update of a capturable group: the step count is read and advanced on the device."""
        ps = [p for p in group["params"] if p.grad is not None]
        if not ps:
            return
        # one counter per group: a parameter that skipped a step would get the bias corrections of the wrong step count
        # (torch.optim.Adam counts per parameter), so the set that takes part is fixed by the first step
        members = tuple(id(p) for p in ps)
        if self._members.setdefault(gi, members) != members:
            raise RuntimeError("FusedAdam(capturable=True): the parameters with a gradient changed between two steps of a group "
                               "(one device step counter per group: every parameter must take part in every step)")
        dev_step = self._step_dev.get(gi)
        if dev_step is None or dev_step.device != ps[0].device:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("FusedAdam(capturable=True): run at least one eager step before capturing (state is created there)")
            known = [self.state[p]["step"] for p in ps if self.state.get(p) and "step" in self.state[p]]  # (a loaded state_dict: per-parameter values)
            start = int(round(float(known[0].item() if torch.is_tensor(known[0]) else known[0]))) if known else 0
            dev_step = self._step_dev[gi] = torch.full((1,), start, dtype=torch.int64, device=ps[0].device)
        items = []
        for p in ps:
            if not p.is_cuda or p.dtype != torch.float32:
                raise _lib.GcpnetHipError("FusedAdam: fp32 parameters on the GPU only (gcpnet_amd has no CPU path)")
            st = self.state[p]
            if "exp_avg" not in st:
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("FusedAdam(capturable=True): a parameter without state inside a capture")
                st["exp_avg"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
                st["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
            st["step"] = dev_step  # (one counter per group: every parameter takes part in every step)
            items.append((p, st))
        arr, keep = self._tensors(items)
        b1, b2 = group["betas"]
        check(lib.gcpnet_adam_step_dev(len(items), arr, float(group["lr"]), float(b1), float(b2), float(group["eps"]),
                                       float(group["weight_decay"]), C.c_void_p(dev_step.data_ptr()),
                                       C.c_void_p(torch.cuda.current_stream().cuda_stream)), "adam_step_dev")
        del keep

    @staticmethod
    def _tensors(items):
        arr = (AdamTensor * len(items))()
        keep = []
        for k, (p, st) in enumerate(items):
            g = p.grad if p.grad.is_contiguous() else p.grad.contiguous()
            keep.append(g)
            arr[k].param, arr[k].grad = p.data_ptr(), g.data_ptr()
            arr[k].exp_avg, arr[k].exp_avg_sq, arr[k].n = st["exp_avg"].data_ptr(), st["exp_avg_sq"].data_ptr(), p.numel()
        return arr, keep

    @staticmethod
    def _launch(lib, group, items, step):
        arr = (AdamTensor * len(items))()
        keep = []
        for k, (p, st) in enumerate(items):
            g = p.grad if p.grad.is_contiguous() else p.grad.contiguous()
            keep.append(g)
            arr[k].param, arr[k].grad = p.data_ptr(), g.data_ptr()
            arr[k].exp_avg, arr[k].exp_avg_sq, arr[k].n = st["exp_avg"].data_ptr(), st["exp_avg_sq"].data_ptr(), p.numel()
        b1, b2 = group["betas"]
        check(lib.gcpnet_adam_step(len(items), arr, float(group["lr"]), float(b1), float(b2), float(group["eps"]),
                                   float(group["weight_decay"]), int(step), C.c_void_p(torch.cuda.current_stream().cuda_stream)),
              "adam_step")


_address, _numel, _contiguous = torch.Tensor.data_ptr, torch.Tensor.numel, torch.Tensor.is_contiguous
_grad, _dtype = operator.attrgetter("grad"), operator.attrgetter("dtype")


class _Part:
    """The tensors of one parameter group that share a device and a type, as the launches take them."""

    def __init__(self, device, dtype, items, bits):
        self.device, self.dtype = device, dtype
        self.type = _lib.TYPE_F32 if dtype == torch.float32 else _lib.TYPE_BF16
        self.params = [p for p, _, _, _ in items]
        self.arr = (AdamWTensor * len(items))()
        self.copies = []
        # what the next step compares with (the tensors of the state are kept alive, so that their addresses stay theirs); a permuted parameter
        # or a state that holds something else than tensors never matches: such a table is built anew every step
        self.states = [st for _, _, st, _ in items]
        self.held = [v for st in self.states for v in st.values()]
        self.where = [v.data_ptr() for v in self.held] if all(map(torch.is_tensor, self.held)) else None
        self.live, self.order = [id(p) for p in self.params], [ordinal for _, _, _, ordinal in items]
        self.addresses = [p.data_ptr() if p.is_contiguous() else None for p in self.params]
        self.sizes = [p.numel() for p in self.params]
        for t, (p, g, st, ordinal) in zip(self.arr, items):
            if g.stride() != p.stride() and not (g.is_contiguous() and p.is_contiguous()):
                g = torch.empty_like(p, memory_format=torch.preserve_format).copy_(g)
                self.copies.append(g)  # (alive until the launches are enqueued)
            t.param, t.grad, t.n, t.ordinal = p.data_ptr(), g.data_ptr(), p.numel(), ordinal
            t.exp_avg, t.exp_avg_sq, t.step = st["exp_avg"].data_ptr(), st["exp_avg_sq"].data_ptr(), st["step"].data_ptr()
            if bits == 8:
                t.exp_avg_scale, t.exp_avg_sq_scale = st["exp_avg_scale"].data_ptr(), st["exp_avg_sq_scale"].data_ptr()
            if dtype == torch.bfloat16:
                t.master = st["master"].data_ptr()
        self.grads = [t.grad for t in self.arr]


class FusedAdamW(torch.optim.Optimizer):
    """torch.optim.AdamW(params, lr, betas, eps, weight_decay) semantics (decoupled weight decay, amsgrad=False, maximize=False) over all
    tensors of a group in a few HIP launches, for fp32 and bf16 parameters on the GPU.

    state_bits (32 or 8, per group): the moments `exp_avg`, `exp_avg_sq` in fp32, or as float8_e4m3fn codes with a power-of-two scale for
    every 256 elements (`exp_avg_scale`, `exp_avg_sq_scale`): 2 bytes of state per element instead of 8.  exp_avg is rounded to nearest,
    exp_avg_sq stochastically (unbiased; to nearest it would freeze), with a hash of (seed, position of the parameter, step, element):
    the same run gives the same bits.  bf16 parameters keep an fp32 `master` copy in the state; a parameter whose value is not the
    rounding of its master copy (loaded or edited since) is taken as it is.

    max_grad_norm: every step scales the gradients (not their tensors: `p.grad` stays as it is) by min(1, max_grad_norm / (norm + 1e-6)) of
    the norm over all groups, which `grad_norm` holds afterwards, on the device.

    Nothing of a step depends on a host value that changes: `step` is a device tensor per parameter, and step() may be captured into a
    hipGraph (GraphedStep(step_fn, optimizer=...)) once an eager step has created the state; lr, betas, eps and weight_decay are frozen
    into a capture.  With state_bits=32 and fp32 parameters, state_dicts interchange with torch.optim.AdamW; its groups with maximize, amsgrad or
    differentiable, and torch.optim.Adam's with a weight decay, are refused."""

    def __init__(self, params: Iterable, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2, *,
                 state_bits: int = 32, max_grad_norm: Optional[float] = None, seed: int = 0):
        if max_grad_norm is not None and not max_grad_norm > 0:
            raise ValueError(f"max_grad_norm must be positive, got {max_grad_norm}")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits, seed=seed))
        self.max_grad_norm = max_grad_norm
        self.grad_norm = None
        self._parts, self._state_ids = {}, []

    def add_param_group(self, group):
        super().add_param_group(group)
        g = self.param_groups[-1]
        try:
            self._check_group(g)
        except Exception:
            self.param_groups.pop()
            raise

    @staticmethod
    def _check_options(g):
        if isinstance(g["lr"], torch.Tensor):
            raise TypeError("FusedAdamW: lr is a number (a tensor would be read back in every step)")
        if not g["lr"] >= 0 or not g["eps"] >= 0 or not g["weight_decay"] >= 0:
            raise ValueError("FusedAdamW: lr, eps and weight_decay must not be negative")
        if not all(0 <= b < 1 for b in g["betas"]):
            raise ValueError(f"FusedAdamW: betas must lie in [0, 1), got {g['betas']}")
        if g["state_bits"] not in (8, 32):
            raise ValueError(f"FusedAdamW: state_bits is 8 or 32, got {g['state_bits']}")
        for key in ("maximize", "amsgrad", "differentiable"):  # (a group that torch.optim.AdamW wrote has them)
            if g.get(key):
                raise ValueError(f"FusedAdamW: {key}=True is another update than this one")
        if not g.get("decoupled_weight_decay", True) and g["weight_decay"]:
            raise ValueError("FusedAdamW: weight decay is decoupled from the gradient (the group is torch.optim.Adam's, with decoupled_weight_decay=False)")

    @classmethod
    def _check_group(cls, g):
        cls._check_options(g)
        if len(set(map(id, g["params"]))) != len(g["params"]):
            raise ValueError("FusedAdamW: a parameter twice in one group (both updates would run at once)")
        for p in g["params"]:
            if p.dtype not in (torch.float32, torch.bfloat16):
                raise TypeError(f"FusedAdamW: fp32 and bf16 parameters only, got {p.dtype}")

    def __setstate__(self, state):
        super().__setstate__(state)
        self.__dict__.setdefault("max_grad_norm", None)
        self.__dict__.setdefault("grad_norm", None)
        self._parts, self._state_ids = {}, []
        states, lacking = self.__dict__.get("_fitted") or ({}, [])  # (of a load)
        for g, more in zip(self.param_groups, lacking):
            g.update(more)
        self.state.update(states)

    def __getstate__(self):
        return {**super().__getstate__(), "max_grad_norm": self.max_grad_norm}

    def load_state_dict(self, state_dict):
        """torch's loader converts every state tensor to its parameter's type: here the moments, scales and master copies keep theirs.  Options come
        from the saved groups, state_bits and seed too; groups that have none of these (torch.optim.AdamW's) leave a group its own.  Moments of another
        kind than a group's state_bits (fp32 for 8, or the reverse) are refused, and so are 8-bit moments that were saved in another memory order than
        the parameter's (their scales go by it).  A refused load changes nothing."""
        # (behind all other hooks: what is checked is what is loaded, and nothing of this optimizer has been touched yet)
        hook = self.register_load_state_dict_pre_hook(lambda _, saved: self.__dict__.__setitem__("_fitted", self._fit(saved)))
        try:
            super().load_state_dict(state_dict)
        finally:
            hook.remove()
            self.__dict__.pop("_fitted", None)

    def _fit(self, state_dict):
        """The states of a state_dict as this optimizer's parameters take them, and the options that its groups lack; everything checked."""
        groups = state_dict["param_groups"]
        if [len(g["params"]) for g in groups] != [len(g["params"]) for g in self.param_groups]:
            return {}, []  # (torch's loader refuses these)
        lacking = [{k: own[k] for k in ("state_bits", "seed") if k not in g} for own, g in zip(self.param_groups, groups)]
        states = {}
        for own, g, more in zip(self.param_groups, groups, lacking):
            options = {**g, **more}
            self._check_options(options)
            for p, i in zip(own["params"], g["params"]):
                if state_dict["state"].get(i):
                    states[p] = self._fit_state(p, state_dict["state"][i], options["state_bits"])
        return states, lacking

    @classmethod
    def _fit_state(cls, p, st, bits):
        new = {}
        for key, v in st.items():
            if key == "step":
                new[key] = torch.as_tensor(v).detach().to(device=p.device, dtype=torch.float32).reshape(()).clone()
            elif not torch.is_tensor(v):
                new[key] = v
            elif key in ("master", "exp_avg", "exp_avg_sq") and v.shape == p.shape:
                if bits == 8 and key != "master" and not cls._same_order(v, p):
                    raise _lib.GcpnetHipError(f"FusedAdamW: the 8-bit state {key!r} was saved in another memory order than its parameter has now "
                                              "(its scales go by that order): give the parameter the saved layout first")
                new[key] = torch.empty_like(p, dtype=v.dtype, memory_format=torch.preserve_format).copy_(v)
            else:
                new[key] = v.detach().to(p.device).clone()
        if p.dtype == torch.bfloat16 and bits == 32:  # (torch keeps the moments of bf16 parameters in bf16)
            for key in ("exp_avg", "exp_avg_sq"):
                if torch.is_tensor(new.get(key)) and new[key].dtype == torch.bfloat16:
                    new[key] = new[key].float()
        if p.dtype == torch.bfloat16 and "master" not in new:
            new["master"] = p.detach().float()
        cls._check_state(p, new, bits)
        return new

    @staticmethod
    def _same_order(codes, p) -> bool:
        """Whether 256 consecutive elements in memory are the same elements of both."""
        return p.numel() <= 256 or all(a == b for a, b, n in zip(codes.stride(), p.stride(), p.shape) if n != 1)

    @staticmethod
    def _check_state(p, st, bits):
        blocks = -(-p.numel() // 256)
        want = {"exp_avg": torch.float32, "exp_avg_sq": torch.float32}
        if bits == 8:
            want = {"exp_avg": torch.float8_e4m3fn, "exp_avg_sq": torch.float8_e4m3fn, "exp_avg_scale": None, "exp_avg_sq_scale": None}
        if p.dtype == torch.bfloat16:
            want["master"] = torch.float32
        for key, dtype in want.items():
            t = st.get(key)
            if t is None or not torch.is_tensor(t) or t.device != p.device or t.dtype != (dtype or torch.float32):
                raise _lib.GcpnetHipError(f"FusedAdamW: state {key!r} is missing, on another device or of another type than state_bits={bits} needs")
            if dtype is None:
                if t.numel() != blocks or not t.is_contiguous():
                    raise _lib.GcpnetHipError(f"FusedAdamW: state {key!r} must hold {blocks} contiguous scales")
            elif t.shape != p.shape or (t.stride() != p.stride() and not (t.is_contiguous() and p.is_contiguous())):
                raise _lib.GcpnetHipError(f"FusedAdamW: state {key!r} must have its parameter's shape and strides")
        step = st.get("step")
        if not torch.is_tensor(step) or step.device != p.device or step.dtype != torch.float32 or step.numel() != 1:
            raise _lib.GcpnetHipError("FusedAdamW: state 'step' must be one fp32 value on the parameter's device")

    @staticmethod
    def _new_state(p, bits):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("FusedAdamW: run at least one eager step before capturing (state is created there)")
        st = {"step": torch.zeros((), dtype=torch.float32, device=p.device)}
        dtype = torch.float32 if bits == 32 else torch.float8_e4m3fn
        for key in ("exp_avg", "exp_avg_sq"):
            # (zeros of one-byte codes through their bytes)
            st[key] = torch.empty_like(p, dtype=dtype, memory_format=torch.preserve_format)
            (st[key] if bits == 32 else st[key].view(torch.uint8)).zero_()
            if bits == 8:
                st[key + "_scale"] = torch.ones(-(-p.numel() // 256), dtype=torch.float32, device=p.device)
        if p.dtype == torch.bfloat16:
            st["master"] = p.detach().to(torch.float32, memory_format=torch.preserve_format)
        return st

    @staticmethod
    def _dense(t) -> bool:
        """Every element of the tensor's span once: elements in memory order are the tensor's."""
        if t.is_contiguous():
            return True
        want = 1
        for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
            if stride != want:
                return False
            want *= size
        return True

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        lib = _lib.load()
        if list(map(id, self.state.values())) != self._state_ids:  # (a state was put in, taken out or exchanged)
            self._parts = {}
        devices, touched, ordinal, built = {}, [], 0, False  # device index -> [(group, _Part)]
        for gi, group in enumerate(self.param_groups):
            self._check_options(group)
            parts = self._parts.get(gi)
            if parts is None or parts[0] != (ordinal, group["state_bits"]) or not self._refresh(parts[1], group["params"]):
                parts = self._parts[gi] = ((ordinal, group["state_bits"]), self._build(group, ordinal))
                built = True
            ordinal += len(group["params"])
            for part in parts[1]:
                devices.setdefault(part.device, []).append((group, part))
                touched.extend(part.params)
        if built:
            self._state_ids = list(map(id, self.state.values()))
        if len(devices) > 1 and self.max_grad_norm is not None:
            raise _lib.GcpnetHipError("FusedAdamW: max_grad_norm with parameters on several devices is not supported")
        if not devices and self.max_grad_norm is not None:  # (no gradient: not the norm of the step before)
            self.grad_norm = next((torch.zeros((), device=p.device) for g in self.param_groups for p in g["params"]), None)
        for dev, parts in devices.items():
            with torch.cuda.device(dev):
                self._step_device(lib, dev, parts)
        if touched:
            torch.autograd.graph.increment_version(touched)  # (written through raw pointers: autograd's and the packs' caches must notice)
            ops.invalidate_packs()
        if built:
            for _, parts in self._parts.values():
                for part in parts:
                    part.copies.clear()
        return loss

    def _build(self, group, ordinal):
        """The launch tables of one group: every tensor looked at in full.  They hold what the optimizer owns (state addresses, sizes)
        from step to step; parameters and gradients are looked up anew in each (`_refresh`)."""
        parts = {}
        bits = group["state_bits"]
        for k, p in enumerate(group["params"]):
            g = p.grad
            if g is None:
                continue
            if not p.is_cuda:
                raise _lib.GcpnetHipError("FusedAdamW: parameters on the GPU only (gcpnet_amd has no CPU path)")
            if g.is_sparse or g.dtype != p.dtype or g.device != p.device or g.shape != p.shape:
                raise _lib.GcpnetHipError("FusedAdamW: a gradient must be dense and have its parameter's type, shape and device")
            if p.dtype not in (torch.float32, torch.bfloat16):
                raise TypeError(f"FusedAdamW: fp32 and bf16 parameters only, got {p.dtype}")
            if not self._dense(p):
                raise _lib.GcpnetHipError("FusedAdamW: a parameter must fill its memory (a permuted tensor does, a slice of one does not)")
            st = self.state[p]
            with torch.cuda.device(p.device):
                if "exp_avg" not in st:
                    st.update(self._new_state(p, bits))
                else:
                    self._check_state(p, st, bits)
                parts.setdefault((p.device.index, p.dtype), []).append((p, g, st, ordinal + k))
        for items in parts.values():  # (the updates of a launch run at once)
            end = 0
            for start, size in sorted((p.data_ptr(), p.numel() * p.element_size()) for p, _, _, _ in items if p.numel()):
                if start < end:
                    raise _lib.GcpnetHipError("FusedAdamW: parameters of one group must not share memory")
                end = start + size
        return [_Part(dev, dtype, items, bits) for (dev, dtype), items in parts.items()]

    def _refresh(self, parts, params) -> bool:
        """Whether the same parameters take part with the same state as when `parts` were built; puts this step's gradients in."""
        try:
            if len(parts) == 1 and list(map(id, params)) == parts[0].live:
                return self._same(parts[0], list(map(_grad, params)))
            if [id(p) for p in params if p.grad is not None] != self._live(parts):
                return False
            return all([self._same(part, list(map(_grad, part.params))) for part in parts])
        except TypeError:  # (something is not a tensor: a gradient that is None, a value put into a state)
            return False

    @staticmethod
    def _same(part, grads) -> bool:
        if (part.where is None or list(map(_address, part.params)) != part.addresses or list(map(_numel, part.params)) != part.sizes
                or not all(map(_contiguous, part.params))  # (turned where it lies)
                or list(map(_numel, grads)) != part.sizes or set(map(_dtype, grads)) != {part.dtype} or not all(map(_contiguous, grads))
                or list(map(_address, itertools.chain.from_iterable(map(dict.values, part.states)))) != part.where):
            return False
        pointers = list(map(_address, grads))
        if pointers != part.grads:
            for t, g in zip(part.arr, pointers):
                t.grad = g
            part.grads = pointers
        return True

    @staticmethod
    def _live(parts):
        if len(parts) == 1:
            return parts[0].live
        return [i for _, i in sorted((k, i) for part in parts for k, i in zip(part.order, part.live))]

    def _step_device(self, lib, dev, parts):
        stream, where = ops._stream(), torch.device("cuda", dev)
        corr = torch.empty(4 * sum(len(part.arr) for _, part in parts), dtype=torch.float32, device=where)
        clip = partials = None
        count = 0
        if self.max_grad_norm is not None:
            counts = [int(lib.gcpnet_grad_norm_partials(len(part.arr), part.arr)) for _, part in parts]
            count = sum(counts)
            partials = torch.empty(max(count, 1), dtype=torch.float32, device=where)
            clip = torch.empty(2, dtype=torch.float32, device=where)
            at = 0
            for (_, part), c in zip(parts, counts):
                check(lib.gcpnet_grad_norm(len(part.arr), part.arr, part.type, partials.data_ptr() + 4 * at, stream), "grad_norm")
                at += c
            self.grad_norm = clip[0]
        at = 0
        for k, (group, part) in enumerate(parts):
            arr = part.arr
            (b1, b2), lr, here = group["betas"], float(group["lr"]), corr.data_ptr() + 16 * at
            at += len(arr)
            first = clip is not None and k == 0
            check(lib.gcpnet_adamw_begin(len(arr), arr, lr, float(b1), float(b2), here, partials.data_ptr() if first else None, count,
                                         float(self.max_grad_norm or 0.0), clip.data_ptr() if first else None, stream), "adamw_begin")
            check(lib.gcpnet_adamw_step(len(arr), arr, part.type, int(group["state_bits"]), lr, float(b1), float(b2), float(group["eps"]),
                                        float(group["weight_decay"]), here, None if clip is None else clip.data_ptr(),
                                        int(group["seed"]) & 0xFFFFFFFF, stream), "adamw_step")
