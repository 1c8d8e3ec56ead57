"""ctypes binding of the attention-layer operators (the C ABI declared in include/ifd_ops.h)."""
from __future__ import annotations

import ctypes

import torch
from torch.autograd import forward_ad

from . import _lib

_c = ctypes
vp, i32, i64, f32 = _c.c_void_p, _c.c_int, _c.c_int64, _c.c_float
DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
Strides = i64 * 3


class AttentionArgs(ctypes.Structure):
    """ifd_attention_args"""
    _fields_ = ([(n, i32) for n in ("dtype", "B", "Tq", "Tk", "Hq", "Hk", "D", "causal")]
                + [("scale", f32), ("pad", i32)]
                + [(n, vp) for n in ("q", "k", "v", "out", "lse", "kv_len", "q_start")]
                + [(n, Strides) for n in ("q_s", "k_s", "v_s", "out_s")]
                + [(n, vp) for n in ("dout", "dq", "dk", "dv")]
                + [(n, Strides) for n in ("dout_s", "dq_s", "dk_s", "dv_s")])


class QkArgs(ctypes.Structure):
    """ifd_qk_args"""
    _fields_ = ([(n, i32) for n in ("dtype", "B", "T", "Hq", "Hk", "D", "rot", "interleaved", "norm")]
                + [("eps", f32), ("mscale", f32), ("pad", i32)]
                + [(n, vp) for n in ("q", "k", "q_out", "k_out", "wq", "wk", "pos", "turns")]
                + [(n, Strides) for n in ("q_s", "k_s", "q_out_s", "k_out_s")] + [("pos_s", i64 * 2)]
                + [(n, vp) for n in ("gq", "gk", "dq", "dk", "dwq", "dwk")]
                + [(n, Strides) for n in ("gq_s", "gk_s", "dq_s", "dk_s")])


class AdamwArgs(ctypes.Structure):
    """ifd_adamw_args"""
    _fields_ = ([(n, i32) for n in ("nt", "bits", "step")] + [("seed", _c.c_uint32)]
                + [(n, vp) for n in ("p", "g", "n", "ptype", "gtype", "m", "v", "m_scale", "v_scale")]
                + [("block0", i64)] + [(n, _c.c_double) for n in ("lr", "b1", "b2", "eps", "wd")] + [("norm_coef", vp)])


OPS_EXPORTS = {
    "ifd_op_attention_ws_bytes": (i64, [vp]),
    "ifd_op_attention": (i32, [vp, vp, i64, vp]),
    "ifd_op_attention_bwd_ws_bytes": (i64, [vp]),
    "ifd_op_attention_bwd": (i32, [vp, vp, i64, vp]),
    "ifd_op_qk_norm_rope": (i32, [vp, vp]),
    "ifd_op_qk_norm_rope_bwd_ws_bytes": (i64, [vp]),
    "ifd_op_qk_norm_rope_bwd": (i32, [vp, vp, i64, vp]),
    "ifd_op_grad_norm_ws_bytes": (i64, [i32, vp]),
    "ifd_op_grad_norm": (i32, [i32, vp, vp, vp, _c.c_double, vp, vp, i64, vp]),
    "ifd_op_adamw": (i32, [vp, vp]),
    "ifd_op_state_values": (i32, [vp, vp, vp, vp, i64, vp, vp, vp]),
}

_bound = None


def lib():
    global _bound
    L = _lib.lib()
    if _bound is not L:
        for name, (res, args) in OPS_EXPORTS.items():
            f = getattr(L, name)
            f.restype = res
            f.argtypes = args
        _bound = L
    return L


def _raw_stream(i):
    return torch.cuda.current_stream(i).cuda_stream


# the same without building a Stream object, where torch has it (2 us of the smallest calls' 16)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _raw_stream)


def refuse(msg):
    raise ValueError("ifd: " + msg)


def same_device(*tensors):
    """The device all the tensors live on (they must be on one GPU)."""
    dev = None
    for t in tensors:
        if t is None:
            continue
        d = t.device
        if d != dev:
            if d.type != "cuda":
                refuse(f"expected a GPU tensor, got one on {d}")
            if dev is not None:
                refuse(f"tensors on {dev} and on {d}")
            dev = d
    return dev


def no_grad(*tensors):
    """These operators record nothing for autograd: a call that autograd would have to follow, in either direction, is refused,
    not cut off."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                refuse("the operator records no gradients: call it under torch.no_grad() (or with detached tensors) and its "
                       "backward function yourself")
    # (the level spares the usual call 6 us a tensor; a torch that does not tell it is asked tensor by tensor)
    if getattr(forward_ad, "_current_level", 0) >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                refuse("the operator has no forward-mode derivative: a tensor carries a tangent")


def _apart(t):
    """Whether t's strides nest: every dimension steps over all that the dimensions of smaller strides reach, so that no two
    elements are one place. (Slices and permutations of a buffer nest; strides that interleave without meeting do not.)"""
    if not t.numel():
        return True
    reach = 0
    for s, n in sorted(zip(t.stride(), t.shape)):
        if n > 1:
            if s <= reach:
                return False
            reach += (n - 1) * s
    return True


def output(t, like, name):
    """Checks a caller's output tensor: like its input, every element a place of its own; marks it as written."""
    if not (t.shape == like.shape and t.dtype == like.dtype and t.device == like.device):
        refuse(f"{name} must be like its input")
    if not _apart(t):
        refuse(f"{name} has elements that share their place, or strides {t.stride()} that do not nest")
    no_grad(t)
    torch.autograd.graph.increment_version(t)
    return t


def may_overlap(a, b):
    """Whether two [batch, tokens, heads, channels] tensors could share elements. Told apart: other storages, ranges one
    behind the other, and different channel ranges of the same token rows (slices of one packed buffer)."""
    if a.untyped_storage().data_ptr() != b.untyped_storage().data_ptr() or not a.numel() or not b.numel():
        return False
    end = lambda t: t.storage_offset() + sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1  # noqa: E731
    if min(a.stride() + b.stride()) < 0 or a.storage_offset() >= end(b) or b.storage_offset() >= end(a):
        return min(a.stride() + b.stride()) < 0
    row = a.stride(1)
    if a.stride()[:2] != b.stride()[:2] or row <= 0 or a.stride(0) % row:
        return True
    lo = [t.storage_offset() % row for t in (a, b)]
    hi = [o + (t.shape[2] - 1) * t.stride(2) + t.shape[3] for o, t in zip(lo, (a, b))]
    return max(hi) > row or not (hi[0] <= lo[1] or hi[1] <= lo[0])


def workspace(nbytes, t):
    """Scratch of one call on t's device, from torch's stream-ordered allocator (None when the call needs none)."""
    return t.new_empty(nbytes, dtype=torch.uint8) if nbytes else None


def call(fn, dev, *args):
    """fn(*args, stream) on the current stream of `dev`, with that device current; raises on a non-zero status."""
    i = dev.index
    if torch.cuda.current_device() == i:
        rc = fn(*args, _raw_stream(i))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _raw_stream(i))
    if rc:
        _lib.check(rc)
