"""Per-head RMS norm of queries and keys with the position rotation in the same pass (csrc/qk_rope.hip).

    rope = Rotary(64, device="cuda:0")                        # rotated channels; interleaved=..., scaling=...
    q2, k2 = qk_norm_rope(q, k, wq, wk, pos, rope)            # then ifd.attention.attention(q2, k2, v)
    dq, dk, dwq, dwk = qk_norm_rope_bwd(dq2, dk2, q, k, wq, wk, pos, rope)

q: [B, T, Hq, D], k: [B, T, Hk, D], one type (fp32, bf16, fp16), D <= 128 and even, any strides with adjacent channels (the
slices of a packed projection). n = x / sqrt(mean x^2 + eps) * w over each head's channels; the first `rope.rot` channels
are then turned in pairs by the angle pos * inv_freq (fp64, so that far positions keep their angle) and scaled by
rope.mscale. norm=False leaves out the norm, rope=None the rotation, wq / wk=None the weights; k=None takes queries alone.
pos: int64 [B, T] or [T]. Statistics and products are fp32, each output is rounded once. Deterministic.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from ._ops import DTYPES, QkArgs, Strides, lib, need, same_device, workspace


class Rotary:
    """Frequencies of the position rotation (fp64, on the device) and its amplitude.

    rot: rotated channels (even); base: inv_freq[i] = base^(-2 i / rot); interleaved: pairs (2i, 2i + 1) instead of
    (i, i + rot / 2). scaling, for contexts longer than the training's:
      ("linear", s)            positions divided by s
      ("base", s)              the base widened by s^(rot / (rot - 2)): the lowest frequency is divided by s, the highest kept
      ("bands", s, length)     frequencies that turn 32 times and more over `length` positions are kept, those that turn
                               once or less are divided by s, linear in the turns between; amplitude 0.1 ln(s) + 1
    """

    def __init__(self, rot, base=10000.0, interleaved=False, scaling=None, device="cuda"):
        need(isinstance(rot, int) and rot > 0 and rot % 2 == 0, f"rotated channels must be even and positive, got {rot}")
        need(base > 1.0, f"base must be larger than 1, got {base}")
        kind = scaling[0] if scaling else None
        need(kind in (None, "linear", "base", "bands"), f"unknown scaling {scaling!r}")
        need(kind is None or (len(scaling) == (3 if kind == "bands" else 2) and scaling[1] >= 1.0),
             f"scaling {scaling!r}: a factor of at least 1" + (" and a length" if kind == "bands" else ""))
        self.rot, self.base, self.interleaved, self.scaling, self.mscale = rot, float(base), bool(interleaved), scaling, 1.0
        if kind == "base":
            base = base * scaling[1] ** (rot / max(rot - 2, 1))
        f = base ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64) / rot)
        if kind == "linear":
            f = f / scaling[1]
        elif kind == "bands":
            need(scaling[2] > 0, f"scaling {scaling!r}: the length must be positive")
            keep = ((scaling[2] * f / (2 * math.pi) - 1.0) / 31.0).clamp(0, 1)
            f = f * keep + f / scaling[1] * (1 - keep)
            self.mscale = 0.1 * math.log(scaling[1]) + 1.0
        self.inv_freq = f
        self.turns = (f / (2 * math.pi)).to(device)


def _st(t):
    return Strides(*t.stride()[:3])


def _rows(t):
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _weight(w, D, name, dev):
    if w is None:
        return None
    need(w.shape == (D,) and w.is_floating_point() and w.device == dev, f"{name} must be a float [{D}] on {dev}")
    return w.detach().float().contiguous()


def _args(q, k, wq, wk, pos, rope, eps, norm):
    need(q.dim() == 4 and (k is None or k.dim() == 4), "q, k must be [batch, tokens, heads, channels]")
    B, T, Hq, D = q.shape
    need(q.dtype in DTYPES and (k is None or k.dtype == q.dtype), "q, k must have one type: fp32, bf16 or fp16")
    need(k is None or (k.shape[0], k.shape[1], k.shape[3]) == (B, T, D), f"k must be [{B}, {T}, heads, {D}]")
    need(0 < D <= 128 and D % 2 == 0, f"head width {D}: at most 128 and even")
    need(eps >= 0.0, f"eps must not be negative, got {eps}")
    need(rope is None or rope.rot <= D, f"{rope and rope.rot} rotated channels of {D}")
    need(rope is None or pos is not None, "a rotation needs positions")
    need(norm or (wq is None and wk is None), "weights without the norm")
    dev = same_device(q, k)
    a = QkArgs(dtype=DTYPES[q.dtype], B=B, T=T, Hq=Hq, Hk=0 if k is None else k.shape[2], D=D, norm=int(bool(norm)), eps=eps,
               mscale=1.0)
    keep = [_rows(q), None if k is None else _rows(k), _weight(wq, D, "wq", dev), _weight(wk, D, "wk", dev)]
    for n, t in zip(("q", "k"), keep):
        if t is not None:
            setattr(a, n, t.data_ptr())
            setattr(a, n + "_s", _st(t))
    a.wq, a.wk = (None if t is None else t.data_ptr() for t in keep[2:4])
    if rope is not None:
        need(pos.dtype == torch.int64 and pos.shape in ((B, T), (T,)), f"pos must be int64 [{B}, {T}] or [{T}]")
        need(pos.device == dev and rope.turns.device == dev, f"pos and the rotation's frequencies must be on {dev}")
        a.rot, a.interleaved, a.mscale = rope.rot, int(rope.interleaved), rope.mscale
        a.pos, a.turns = pos.data_ptr(), rope.turns.data_ptr()
        a.pos_s = (ctypes.c_int64 * 2)(*((0,) + pos.stride() if pos.dim() == 1 else pos.stride()))
        keep += [pos, rope.turns]
    return a, keep, dev


def _into(t, like, name):
    if like is None:
        return None
    if t is None:
        return torch.empty(like.shape, dtype=like.dtype, device=like.device)
    need(t.shape == like.shape and t.dtype == like.dtype and t.device == like.device and (t.stride(-1) == 1 or
         t.shape[-1] == 1), f"{name} must be like its input, with adjacent channels")
    return t


def qk_norm_rope(q, k, wq=None, wk=None, pos=None, rope=None, eps=1e-6, norm=True, q_out=None, k_out=None):
    """(q_out, k_out); q_out=q and k_out=k work in place. k=None: (q_out, None)."""
    a, keep, dev = _args(q, k, wq, wk, pos, rope, eps, norm)
    q_out, k_out = _into(q_out, q, "q_out"), _into(k_out, k, "k_out")
    for n, t in (("q_out", q_out), ("k_out", k_out)):
        if t is not None:
            setattr(a, n, t.data_ptr())
            setattr(a, n + "_s", _st(t))
    with torch.cuda.device(dev):
        _lib.check(lib().ifd_op_qk_norm_rope(ctypes.byref(a), _lib.stream_ptr(dev)))
    return q_out, k_out


def qk_norm_rope_bwd(gq, gk, q, k, wq=None, wk=None, pos=None, rope=None, eps=1e-6, norm=True, dq=None, dk=None):
    """(dq, dk, dwq, dwk) from the gradients of the outputs; q, k are the forward's inputs. dwq, dwk are fp32 sums over
    tokens and heads (None without weights); dq=gq and dk=gk work in place."""
    a, keep, dev = _args(q, k, wq, wk, pos, rope, eps, norm)
    need((gk is None) == (k is None), "gk without k")
    for n, t, like in (("gq", gq, q), ("gk", gk, k)):
        if t is not None:
            need(t.shape == like.shape and t.dtype == like.dtype, f"{n} must be like {n[1]}")
    same_device(q, gq, gk)
    gq, gk = _rows(gq), None if gk is None else _rows(gk)
    dq, dk = _into(dq, q, "dq"), _into(dk, k, "dk")
    dwq = None if wq is None else torch.empty(q.shape[3], dtype=torch.float32, device=dev)
    dwk = None if wk is None else torch.empty(q.shape[3], dtype=torch.float32, device=dev)
    for n, t in (("gq", gq), ("gk", gk), ("dq", dq), ("dk", dk)):
        if t is not None:
            setattr(a, n, t.data_ptr())
            setattr(a, n + "_s", _st(t))
    a.dwq, a.dwk = (None if t is None else t.data_ptr() for t in (dwq, dwk))
    L = lib()
    with torch.cuda.device(dev):
        n = L.ifd_op_qk_norm_rope_bwd_ws_bytes(ctypes.byref(a))
        ws = workspace(n, dev)
        _lib.check(L.ifd_op_qk_norm_rope_bwd(ctypes.byref(a), _lib.ptr(ws), n, _lib.stream_ptr(dev)))
    return dq, dk, dwq, dwk
