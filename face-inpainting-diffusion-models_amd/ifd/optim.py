"""AdamW over many tensors in one pass, with 8-bit or 32-bit states (csrc/adamw.hip).

    opt = AdamW(params, lr=5e-5, weight_decay=0.01, max_norm=1.0, state_bits=8)
    opt.step(grads)                     # or opt.step() with the parameters' .grad

params: a list of tensors, or of groups {"params": [...], "lr": ..., "weight_decay": ...}; fp32, bf16 or fp16, contiguous, on
one GPU; gradients likewise, of any of these types. The arithmetic is torch.optim.AdamW's (decoupled decay, bias correction),
with clip_grad_norm_(max_norm) over all tensors folded in (the gradients themselves are not changed).

State memory: 8 bytes a value with state_bits=32, 2 with state_bits=8 (a byte per moment and one scale per 256 values; the
format and its rounding are described in include/ifd_ops.h). The step uses the moments before they are rounded.

With max_norm a step whose gradient norm is not finite leaves parameters and states as they were. opt.norm_coef (fp64, on the
GPU) holds the norm and the clip coefficient. Nothing synchronises; a step can be captured into a graph only with its step
number fixed, so the optimizer refuses capture.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._ops import DTYPES, AdamwArgs, lib, need, same_device, workspace

BLOCK = 256  # values per scale


class AdamW:
    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, state_bits=32, max_norm=None,
                 seed=0):
        need(state_bits in (8, 32), f"state_bits must be 8 or 32, got {state_bits!r}")
        need(0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0, f"betas must be in [0, 1), got {betas}")
        need(eps > 0.0 and lr >= 0.0 and weight_decay >= 0.0, "eps must be positive, lr and weight_decay not negative")
        need(max_norm is None or max_norm > 0.0, f"max_norm must be positive or None, got {max_norm}")
        params = list(params)
        if params and not isinstance(params[0], dict):
            params = [{"params": params}]
        need(all(isinstance(g, dict) for g in params), "params: a list of tensors or of groups")
        self.groups = [{"lr": lr, "weight_decay": weight_decay, **g, "params": list(g["params"])} for g in params]
        self.params = [p for g in self.groups for p in g["params"]]
        need(self.params, "no parameters")
        self.betas, self.eps, self.max_norm, self.state_bits = tuple(betas), float(eps), max_norm, state_bits
        self.seed, self.step_count = int(seed) & 0xFFFFFFFF, 0
        for p in self.params:
            need(p.dtype in DTYPES and p.is_contiguous(), "parameters must be contiguous fp32, bf16 or fp16 tensors")
        need(len({id(p) for p in self.params}) == len(self.params), "a parameter is listed twice")
        self.device = same_device(*self.params)
        at = 0
        for g in self.groups:
            g["block0"] = at
            at += sum(-(-p.numel() // BLOCK) for p in g["params"])
        self.nblocks = at
        z = lambda n, dt: torch.zeros(n, dtype=dt, device=self.device)  # noqa: E731
        dt = torch.uint8 if state_bits == 8 else torch.float32
        self.m, self.v = z(at * BLOCK, dt), z(at * BLOCK, dt)
        self.m_scale, self.v_scale = (z(at, torch.float32), z(at, torch.float32)) if state_bits == 8 else (None, None)
        self.norm_coef = torch.ones(2, dtype=torch.float64, device=self.device)

    def _arrays(self, params, grads):
        """Host arrays of one group: addresses, counts, types (read afresh at every step: tensors may have moved)."""
        n = len(params)
        p, g, cnt = (ctypes.c_void_p * n)(), (ctypes.c_void_p * n)(), (ctypes.c_int64 * n)()
        pt, gt = (ctypes.c_uint8 * n)(), (ctypes.c_uint8 * n)()
        dev = self.device
        for i, (x, d) in enumerate(zip(params, grads)):
            p[i], cnt[i], pt[i] = x.data_ptr(), x.numel(), DTYPES[x.dtype]
            if d is None:
                continue
            if not (d.dtype in DTYPES and d.shape == x.shape and d.device == dev and d.is_contiguous() and x.is_contiguous()
                    and x.device == dev):
                raise ValueError(f"ifd: gradient {i}: contiguous fp32, bf16 or fp16 of shape {tuple(x.shape)} on {dev} "
                                 f"expected, got {d.dtype} {tuple(d.shape)} on {d.device}")
            g[i], gt[i] = d.data_ptr(), DTYPES[d.dtype]
        return p, g, cnt, pt, gt

    def step(self, grads=None):
        """One step; grads in the order of the parameters (None entries: that tensor is left alone)."""
        if grads is None:
            grads = [p.grad for p in self.params]
        grads = list(grads)
        need(len(grads) == len(self.params), f"{len(grads)} gradients for {len(self.params)} parameters")
        need(not torch.cuda.is_current_stream_capturing(), "an optimizer step cannot be captured: its step number would stay")
        L = lib()
        at, arrays = 0, []
        for grp in self.groups:
            k = len(grp["params"])
            arrays.append(self._arrays(grp["params"], grads[at:at + k]))
            at += k
        with torch.cuda.device(self.device):
            s = _lib.stream_ptr(self.device)
            if self.max_norm is not None:
                self._norm(L, arrays, s)
            self.step_count += 1
            for grp, (p, g, cnt, pt, gt) in zip(self.groups, arrays):
                vp = ctypes.c_void_p
                a = AdamwArgs(nt=len(cnt), bits=self.state_bits, step=self.step_count, seed=self.seed, block0=grp["block0"],
                              lr=grp["lr"], b1=self.betas[0], b2=self.betas[1], eps=self.eps, wd=grp["weight_decay"])
                a.p, a.g, a.n, a.ptype, a.gtype = (ctypes.cast(x, vp) for x in (p, g, cnt, pt, gt))
                a.m, a.v = self.m.data_ptr(), self.v.data_ptr()
                if self.state_bits == 8:
                    a.m_scale, a.v_scale = self.m_scale.data_ptr(), self.v_scale.data_ptr()
                a.norm_coef = self.norm_coef.data_ptr() if self.max_norm is not None else None
                _lib.check(L.ifd_op_adamw(ctypes.byref(a), s))

    def _norm(self, L, arrays, s):
        n = sum(len(a[2]) for a in arrays)
        if len(arrays) == 1:
            _, g, cnt, _, gt = arrays[0]
        else:
            g, cnt, gt = (ctypes.c_void_p * n)(), (ctypes.c_int64 * n)(), (ctypes.c_uint8 * n)()
            i = 0
            for _, ga, ca, _, ta in arrays:
                for j in range(len(ca)):
                    g[i], cnt[i], gt[i] = ga[j], ca[j], ta[j]
                    i += 1
        nb = L.ifd_op_grad_norm_ws_bytes(n, cnt)
        ws = workspace(nb, self.device)
        _lib.check(L.ifd_op_grad_norm(n, g, cnt, gt, float(self.max_norm), _lib.ptr(self.norm_coef), _lib.ptr(ws), nb, s))

    def moments(self):
        """(m, v): both moments as fp32 [blocks * 256], each tensor from a multiple of 256 on (the states themselves with
        state_bits=32, what the bytes stand for with 8)."""
        if self.state_bits == 32:
            return self.m, self.v
        m = torch.empty(self.nblocks * BLOCK, dtype=torch.float32, device=self.device)
        v = torch.empty_like(m)
        with torch.cuda.device(self.device):
            _lib.check(lib().ifd_op_state_values(_lib.ptr(self.m), _lib.ptr(self.m_scale), _lib.ptr(self.v),
                                                 _lib.ptr(self.v_scale), self.nblocks, _lib.ptr(m), _lib.ptr(v),
                                                 _lib.stream_ptr(self.device)))
        return m, v

    def load_moments(self, m, v, m_scale=None, v_scale=None):
        """Copies states in, in the layout of m, v (and m_scale, v_scale) of this optimizer."""
        for n, t in (("m", m), ("v", v), ("m_scale", m_scale), ("v_scale", v_scale)):
            own = getattr(self, n)
            need((own is None) == (t is None), f"{n}: {'not used with' if own is None else 'needed with'} {self.state_bits}-bit states")
            if own is not None:
                need(t.dtype == own.dtype and t.shape == own.shape, f"{n} must be {own.dtype} {tuple(own.shape)}")
                own.copy_(t)

    def state_dict(self):
        """Everything a resumed run needs, bit for bit (copies)."""
        d = {"step": self.step_count, "seed": self.seed, "state_bits": self.state_bits}
        d.update({n: getattr(self, n).clone() for n in ("m", "v", "m_scale", "v_scale") if getattr(self, n) is not None})
        return d

    def load_state_dict(self, d):
        need(d["state_bits"] == self.state_bits, f"states of {d['state_bits']} bits for an optimizer of {self.state_bits}")
        self.load_moments(d["m"], d["v"], d.get("m_scale"), d.get("v_scale"))
        self.step_count, self.seed = int(d["step"]), int(d["seed"])
