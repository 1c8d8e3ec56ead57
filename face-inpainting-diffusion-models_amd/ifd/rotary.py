"""Per-head RMS norm of queries and keys with the position rotation in the same pass (csrc/qk_rope.hip).

    rope = Rotary(64, device="cuda:0")                        # rotated channels; interleaved=..., scaling=...
    q2, k2 = qk_norm_rope(q, k, wq, wk, pos, rope)            # then ifd.attention.attention(q2, k2, v)
    dq, dk, dwq, dwk = qk_norm_rope_bwd(dq2, dk2, q, k, wq, wk, pos, rope)

q: [B, T, Hq, D], k: [B, T, Hk, D], one type (fp32, bf16, fp16), D <= 128 and even, any strides with adjacent channels (the
slices of a packed projection). n = x / sqrt(mean x^2 + eps) * w over each head's channels; the first `rope.rot` channels
are then turned in pairs by the angle pos * inv_freq (fp64, so that far positions keep their angle) and scaled by
rope.mscale. norm=False leaves out the norm, rope=None the rotation, wq / wk=None the weights; k=None takes queries alone.
pos: int64 [B, T] or [T]. Statistics and products are fp32, each output is rounded once. Deterministic. An output may be the
tensor of its own input (of its own gradient, backward) and must else overlap no input, no other output and not itself.
Nothing is recorded for autograd: tensors that require gradients are refused unless under torch.no_grad(), those with a
forward-mode tangent always.
"""
from __future__ import annotations

import math
import struct

import torch

from ._ops import DTYPES, call, lib, may_overlap, no_grad, output, refuse, same_device, workspace

# ifd_qk_args (include/ifd_ops.h; _ops.QkArgs has the same layout)
_HEAD, _MORE = struct.Struct("9i2fi 8P 14q"), struct.Struct("6P 12q")
_NO_BWD = bytes(_MORE.size)
_NO_ST = (0, 0, 0)


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
        if not (isinstance(rot, int) and rot > 0 and rot % 2 == 0):
            refuse(f"rotated channels must be even and positive, got {rot}")
        if not base > 1.0:
            refuse(f"base must be larger than 1, got {base}")
        kind = scaling[0] if scaling else None
        if kind not in (None, "linear", "base", "bands"):
            refuse(f"unknown scaling {scaling!r}")
        if kind and not (len(scaling) == (3 if kind == "bands" else 2) and scaling[1] >= 1.0):
            refuse(f"scaling {scaling!r}: a factor of at least 1" + (" and a length" if kind == "bands" else ""))
        self.rot, self.base, self.interleaved, self.scaling, self.mscale = rot, float(base), bool(interleaved), scaling, 1.0
        if kind == "base":
            base = base * scaling[1] ** (rot / max(rot - 2, 1))
        f = base ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64) / rot)
        if kind == "linear":
            f = f / scaling[1]
        elif kind == "bands":
            if not scaling[2] > 0:
                refuse(f"scaling {scaling!r}: the length must be positive")
            keep = ((scaling[2] * f / (2 * math.pi) - 1.0) / 31.0).clamp(0, 1)
            f = f * keep + f / scaling[1] * (1 - keep)
            self.mscale = 0.1 * math.log(scaling[1]) + 1.0
        self.inv_freq = f
        self.turns = (f / (2 * math.pi)).to(device)


def _rows(t):
    return t if t.stride()[3] == 1 or t.shape[3] == 1 else t.contiguous()


def _weight(w, D, name, dev):
    if w.dtype is torch.float32 and w.shape == (D,) and w.device == dev and w.is_contiguous():
        return w
    if not (w.shape == (D,) and w.is_floating_point() and w.device == dev):
        refuse(f"{name} must be a float [{D}] on {dev}")
    return w.detach().float().contiguous()


def _inputs(q, k, wq, wk, pos, rope, eps, norm):
    if q.dim() != 4 or (k is not None and k.dim() != 4):
        refuse("q, k must be [batch, tokens, heads, channels]")
    B, T, _, D = q.shape
    if q.dtype not in DTYPES or (k is not None and k.dtype != q.dtype):
        refuse("q, k must have one type: fp32, bf16 or fp16")
    if k is not None:
        kB, kT, _, kD = k.shape
        if kB != B or kT != T or kD != D:
            refuse(f"k must be [{B}, {T}, heads, {D}], got {tuple(k.shape)}")
    if not 0 < D <= 128 or D & 1:
        refuse(f"head width {D}: at most 128 and even")
    if not eps >= 0.0:
        refuse(f"eps must not be negative, got {eps}")
    if rope is not None and (rope.rot > D or pos is None):
        refuse("a rotation needs positions" if pos is None else f"{rope.rot} rotated channels of {D}")
    if not norm and not (wq is None and wk is None):
        refuse("weights without the norm")
    dev = same_device(q, k)
    no_grad(q, k, wq, wk)
    if wq is not None:
        wq = _weight(wq, D, "wq", dev)
    if wk is not None:
        wk = _weight(wk, D, "wk", dev)
    if rope is not None:
        if pos.dtype is not torch.int64 or pos.shape not in ((B, T), (T,)):
            refuse(f"pos must be int64 [{B}, {T}] or [{T}]")
        if pos.device != dev or rope.turns.device != dev:
            refuse(f"pos and the rotation's frequencies must be on {dev}")
    return _rows(q), None if k is None else _rows(k), wq, wk, dev


def _pack(q, k, wq, wk, pos, rope, eps, norm, q_out, k_out):
    B, T, Hq, D = q.shape
    kp, ks, Hk = (0, _NO_ST, 0) if k is None else (k.data_ptr(), k.stride()[:3], k.shape[2])
    qo, qos = (0, _NO_ST) if q_out is None else (q_out.data_ptr(), q_out.stride()[:3])
    ko, kos = (0, _NO_ST) if k_out is None else (k_out.data_ptr(), k_out.stride()[:3])
    rot, il, ms, pp, tp, ps = 0, 0, 1.0, 0, 0, (0, 0)
    if rope is not None:
        rot, il, ms, pp, tp = rope.rot, rope.interleaved, rope.mscale, pos.data_ptr(), rope.turns.data_ptr()
        ps = pos.stride() if pos.dim() == 2 else (0, pos.stride(0))
    return _HEAD.pack(DTYPES[q.dtype], B, T, Hq, Hk, D, rot, il, 1 if norm else 0, eps, ms, 0,
                      q.data_ptr(), kp, qo, ko, 0 if wq is None else wq.data_ptr(), 0 if wk is None else wk.data_ptr(), pp, tp,
                      *q.stride()[:3], *ks, *qos, *kos, *ps)


def _into(t, like, name, place, *others):
    """A caller's output (checked) or a new one. It may be `place` itself (each head is read, then written, by the same
    lanes), else it must be apart from it, and from `others` in any case."""
    if like is None:
        return None
    if t is None:
        return torch.empty_like(like, memory_format=torch.contiguous_format)
    if t.dim() != 4 or (t.stride(3) != 1 and t.shape[3] != 1):
        refuse(f"{name} must be like its input, with adjacent channels")
    if t is not place and t.data_ptr() == place.data_ptr() and t.stride() == place.stride():
        place = t
    if (t is not place and may_overlap(t, place)) or any(x is not None and may_overlap(t, x) for x in others):
        refuse(f"{name} overlaps an input or another output")
    return output(t, like, name)


def qk_norm_rope(q, k, wq=None, wk=None, pos=None, rope=None, eps=1e-6, norm=True, q_out=None, k_out=None):
    """(q_out, k_out); q_out=q and k_out=k work in place. k=None: (q_out, None)."""
    q, k, wq, wk, dev = _inputs(q, k, wq, wk, pos, rope, eps, norm)
    q_out = _into(q_out, q, "q_out", q, k)
    k_out = _into(k_out, k, "k_out", k, q, q_out)
    call(lib().ifd_op_qk_norm_rope, dev, _pack(q, k, wq, wk, pos, rope, eps, norm, q_out, k_out) + _NO_BWD)
    return q_out, k_out


def qk_norm_rope_bwd(gq, gk, q, k, wq=None, wk=None, pos=None, rope=None, eps=1e-6, norm=True, dq=None, dk=None):
    """(dq, dk, dwq, dwk) from the gradients of the outputs; q, k are the forward's inputs. dwq, dwk are fp32 sums over
    tokens and heads (None without weights); dq=gq and dk=gk work in place."""
    q, k, wq, wk, dev = _inputs(q, k, wq, wk, pos, rope, eps, norm)
    if (gk is None) != (k is None):
        refuse("gk without k")
    if gq.shape != q.shape or gq.dtype != q.dtype or (k is not None and (gk.shape != k.shape or gk.dtype != k.dtype)):
        refuse("gq, gk must be like q, k")
    same_device(q, gq, gk)
    no_grad(gq, gk)
    gq, gk = _rows(gq), None if gk is None else _rows(gk)
    dq = _into(dq, q, "dq", gq, q, k, gk)
    dk = _into(dk, k, "dk", gk, q, k, gq, dq)
    dwq = None if wq is None else q.new_empty(q.shape[3], dtype=torch.float32)
    dwk = None if wk is None else q.new_empty(q.shape[3], dtype=torch.float32)
    gkp, gks, dkp, dks = (0, _NO_ST, 0, _NO_ST) if k is None else (gk.data_ptr(), gk.stride()[:3], dk.data_ptr(), dk.stride()[:3])
    a = _pack(q, k, wq, wk, pos, rope, eps, norm, None, None) + _MORE.pack(
        gq.data_ptr(), gkp, dq.data_ptr(), dkp, 0 if dwq is None else dwq.data_ptr(), 0 if dwk is None else dwk.data_ptr(),
        *gq.stride()[:3], *gks, *dq.stride()[:3], *dks)
    L = lib()
    n = L.ifd_op_qk_norm_rope_bwd_ws_bytes(a)
    ws = workspace(n, q)
    call(L.ifd_op_qk_norm_rope_bwd, dev, a, None if ws is None else ws.data_ptr(), n)
    return dq, dk, dwq, dwk
