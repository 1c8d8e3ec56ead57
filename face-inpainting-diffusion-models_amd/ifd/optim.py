"""AdamW over many tensors in one pass, with 8-bit or 32-bit states (csrc/adamw.hip).

    opt = AdamW(params, lr=5e-5, weight_decay=0.01, max_norm=1.0, state_bits=8)
    opt.step(grads)                     # or opt.step() with the parameters' .grad

params: a list of tensors, or of groups {"params": [...], "lr": ..., "weight_decay": ...} ("params" may be one tensor); fp32,
bf16 or fp16, contiguous, on one GPU; gradients likewise, of any of these types. The arithmetic is torch.optim.AdamW's
(decoupled decay, bias correction), with clip_grad_norm_(max_norm) over all tensors folded in (the gradients themselves are
not changed).

State memory: 8 bytes a value with state_bits=32, 2 with state_bits=8 (a byte per moment and one scale per 256 values; the
format and its rounding are described in include/ifd_ops.h). The step uses the moments before they are rounded.

With max_norm a step whose gradient norm is not finite leaves parameters and states as they were; it counts as a step all the
same (step_count, and with it the bias corrections: the host does not learn of the norm). Without max_norm such a gradient
spoils what ifd_op_adamw in include/ifd_ops.h says. opt.norm_coef (fp64, on the GPU) holds the norm and the clip coefficient.
Nothing synchronises; a step can be captured into a graph only with its step number fixed, so the optimizer refuses capture.
"""
from __future__ import annotations

import ctypes

import torch

from ._ops import DTYPES, AdamwArgs, call, lib, refuse, same_device, workspace

BLOCK = 256  # values per scale


def need(cond, msg):
    if not cond:
        refuse(msg)


class AdamW:
    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, state_bits=32, max_norm=None,
                 seed=0):
        need(state_bits in (8, 32), f"state_bits must be 8 or 32, got {state_bits!r}")
        need(0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0, f"betas must be in [0, 1), got {betas}")
        need(eps > 0.0 and lr >= 0.0 and weight_decay >= 0.0, "eps must be positive, lr and weight_decay not negative")
        need(max_norm is None or max_norm > 0.0, f"max_norm must be positive or None, got {max_norm}")
        need(not isinstance(params, (torch.Tensor, dict)), "params: a list of tensors or of groups")
        params = list(params)
        if params and not isinstance(params[0], dict):
            params = [{"params": params}]
        need(all(isinstance(g, dict) for g in params), "params: a list of tensors or of groups")
        for g in params:
            need("params" in g, "a group without params")
            other = sorted(set(g) - {"params", "lr", "weight_decay"})
            need(not other, f"a group sets its lr and weight_decay alone, not {', '.join(map(str, other))}")
            need(g.get("lr", lr) >= 0.0 and g.get("weight_decay", weight_decay) >= 0.0, "a group's lr and weight_decay: not negative")
        one = lambda p: [p] if isinstance(p, torch.Tensor) else list(p)  # noqa: E731
        self.groups = [{"lr": lr, "weight_decay": weight_decay, **g, "params": one(g["params"])} for g in params]
        self.params = [p for g in self.groups for p in g["params"]]
        need(self.params, "no parameters")
        self.betas, self.eps, self.max_norm, self.state_bits = tuple(betas), float(eps), max_norm, state_bits
        self.seed, self.step_count = int(seed) & 0xFFFFFFFF, 0
        for p in self.params:
            need(p.dtype in DTYPES and p.is_contiguous(), "parameters must be contiguous fp32, bf16 or fp16 tensors")
        need(len({id(p) for p in self.params}) == len(self.params), "a parameter is listed twice")
        self.device = same_device(*self.params)
        at = sorted((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size()) for p in self.params if p.numel())
        need(all(a[1] <= b[0] for a, b in zip(at, at[1:])), "two parameters share memory")
        at = 0
        for g in self.groups:
            g["block0"] = at
            g["shapes"] = [p.shape for p in g["params"]]
            g["sizes"] = (ctypes.c_int64 * len(g["params"]))(*[p.numel() for p in g["params"]])
            at += sum(-(-p.numel() // BLOCK) for p in g["params"])
        self.nblocks = at
        z = lambda n, dt: torch.zeros(n, dtype=dt, device=self.device)  # noqa: E731
        dt = torch.uint8 if state_bits == 8 else torch.float32
        self.m, self.v = z(at * BLOCK, dt), z(at * BLOCK, dt)
        self.m_scale, self.v_scale = (z(at, torch.float32), z(at, torch.float32)) if state_bits == 8 else (None, None)
        self.norm_coef = torch.ones(2, dtype=torch.float64, device=self.device)

    def _arrays(self, grp, grads):
        """Host arrays of one group: addresses, counts, types (read afresh at every step: tensors may have moved)."""
        n, dev, types = len(grads), self.device.index, DTYPES
        pp, gp, pt, gt = [], [], [], []
        for x, d, shape in zip(grp["params"], grads, grp["shapes"]):
            if x.shape != shape or not x.is_contiguous() or x.get_device() != dev or x.dtype not in types:
                refuse(f"parameter {len(pp)} is no longer the contiguous {tuple(shape)} tensor on {self.device} it was")
            pp.append(x.data_ptr())
            pt.append(types[x.dtype])
            if d is None:
                gp.append(0)
                gt.append(0)
                continue
            if d.shape != shape or not d.is_contiguous() or d.get_device() != dev or d.dtype not in types:
                refuse(f"gradient {len(gp)}: contiguous fp32, bf16 or fp16 of shape {tuple(shape)} on {self.device} expected, "
                       f"got {d.dtype} {tuple(d.shape)} on {d.device}")
            gp.append(d.data_ptr())
            gt.append(types[d.dtype])
        ptrs = ctypes.c_void_p * n
        return ptrs(*pp), ptrs(*gp), grp["sizes"], bytes(pt), bytes(gt)

    def step(self, grads=None):
        """One step; grads in the order of the parameters (None entries: that tensor is left alone)."""
        grads = [p.grad for p in self.params] if grads is None else list(grads)
        need(len(grads) == len(self.params), f"{len(grads)} gradients for {len(self.params)} parameters")
        need(not torch.cuda.is_current_stream_capturing(), "an optimizer step cannot be captured: its step number would stay")
        L, dev = lib(), self.device
        at, arrays = 0, []
        for grp in self.groups:
            k = len(grp["params"])
            arrays.append(self._arrays(grp, grads[at:at + k]))
            at += k
        if self.max_norm is not None:
            self._norm(L, arrays)
        k = self.step_count + 1
        for grp, (p, g, cnt, pt, gt) in zip(self.groups, arrays):
            a = AdamwArgs(len(cnt), self.state_bits, k, self.seed)
            keep = ctypes.create_string_buffer(pt, len(pt)), ctypes.create_string_buffer(gt, len(gt))
            a.p, a.g, a.n, a.ptype, a.gtype = (ctypes.addressof(x) for x in (p, g, cnt, *keep))
            a.m, a.v = self.m.data_ptr(), self.v.data_ptr()
            if self.state_bits == 8:
                a.m_scale, a.v_scale = self.m_scale.data_ptr(), self.v_scale.data_ptr()
            a.block0, a.lr, a.b1, a.b2 = grp["block0"], grp["lr"], self.betas[0], self.betas[1]
            a.eps, a.wd = self.eps, grp["weight_decay"]
            a.norm_coef = None if self.max_norm is None else self.norm_coef.data_ptr()
            call(L.ifd_op_adamw, dev, ctypes.byref(a))
        self.step_count = k
        if any([p.requires_grad for p in self.params]):  # (autograd learns that saved parameters have changed)
            torch.autograd.graph.increment_version(self.params)

    def _norm(self, L, arrays):
        if len(arrays) == 1:
            _, g, cnt, _, gt = arrays[0]
        else:
            n = len(self.params)
            g = (ctypes.c_void_p * n)(*[x for a in arrays for x in a[1]])
            cnt = (ctypes.c_int64 * n)(*[x for a in arrays for x in a[2]])
            gt = b"".join(a[4] for a in arrays)
        nb = L.ifd_op_grad_norm_ws_bytes(len(cnt), cnt)
        ws = workspace(nb, self.m)
        call(L.ifd_op_grad_norm, self.device, len(cnt), g, cnt, gt, float(self.max_norm), self.norm_coef.data_ptr(),
             None if ws is None else ws.data_ptr(), nb)

    def moments(self):
        """(m, v): both moments as fp32 [blocks * 256], each tensor from a multiple of 256 on (the states themselves with
        state_bits=32, what the bytes stand for with 8)."""
        if self.state_bits == 32:
            return self.m, self.v
        m = torch.empty(self.nblocks * BLOCK, dtype=torch.float32, device=self.device)
        v = torch.empty_like(m)
        call(lib().ifd_op_state_values, self.device, self.m.data_ptr(), self.m_scale.data_ptr(), self.v.data_ptr(),
             self.v_scale.data_ptr(), self.nblocks, m.data_ptr(), v.data_ptr())
        return m, v

    def load_moments(self, m, v, m_scale=None, v_scale=None):
        """Copies states in, in the layout of m, v (and m_scale, v_scale) of this optimizer."""
        given = {"m": m, "v": v, "m_scale": m_scale, "v_scale": v_scale}
        for n, t in given.items():
            own = getattr(self, n)
            need((own is None) == (t is None), f"{n}: {'not used with' if own is None else 'needed with'} {self.state_bits}-bit states")
            if own is not None:
                need(t.dtype == own.dtype and t.shape == own.shape, f"{n} must be {own.dtype} {tuple(own.shape)}")
        for n, t in given.items():
            if t is not None:
                getattr(self, n).copy_(t)

    def state_dict(self):
        """Everything a resumed run needs, bit for bit (copies)."""
        d = {"step": self.step_count, "seed": self.seed, "state_bits": self.state_bits}
        d.update({n: getattr(self, n).clone() for n in ("m", "v", "m_scale", "v_scale") if getattr(self, n) is not None})
        return d

    def load_state_dict(self, d):
        need(d["state_bits"] == self.state_bits, f"states of {d['state_bits']} bits for an optimizer of {self.state_bits}")
        step, seed = int(d["step"]), int(d["seed"]) & 0xFFFFFFFF
        need(step >= 0, f"a step number of {step}")
        self.load_moments(d["m"], d["v"], d.get("m_scale"), d.get("v_scale"))
        self.step_count, self.seed = step, seed
