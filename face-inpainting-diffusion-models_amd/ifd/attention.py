"""Attention with its log-sum-exp, and its backward pass (csrc/attn_fwd.hip, csrc/attn_bwd.hip).

    out, lse = attention(q, k, v, causal=True)
    dq, dk, dv = attention_bwd(dout, q, k, v, out, lse, causal=True)

q, out: [B, Tq, Hq, D]; k, v: [B, Tk, Hk, D]; one type (fp32, bf16, fp16); Hq a multiple of Hk, query head h reads
key-value head h // (Hq // Hk). D <= 128 and a multiple of 8 (4 in fp32). Any strides with the channels adjacent, e.g. the
three slices of a packed projection or a slice of a longer key-value cache; tensors whose strides are not multiples of
16 bytes (or which are not 16-byte aligned) are copied first.

Row i of sequence b sees key j when j < kv_len[b] (default Tk) and, with causal=True, j <= q_start[b] + i (default
Tk - Tq: the rows are the last ones). kv_len, q_start: int32 [B] on the GPU, read by the kernels (no synchronisation).
Keys at and past kv_len are never read, whatever they hold. A row that sees no key gets out = 0, lse = -inf and zero
gradients. Keys that only the causal mask hides are read: they must be finite in v.

The backward pass keeps no score matrix: it recomputes the probabilities from lse. Both directions are deterministic.
Calls run on the current stream of the tensors' device and can be captured into a graph.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from ._ops import DTYPES, AttentionArgs, Strides, lib, need, same_device, workspace


def _lay(t):
    """t itself when the kernels can read it, else a contiguous copy."""
    e = t.element_size()
    ok = t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all((s * e) % 16 == 0 for s in t.stride()[:3])
    if ok and 0 <= t.stride(1) * e < 1 << 24:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _st(t):
    return Strides(*t.stride()[:3])


def _int_arg(t, B, name, dev):
    if t is None:
        return None
    need(isinstance(t, torch.Tensor) and t.dtype == torch.int32 and t.dim() == 1 and t.shape[0] == B,
         f"{name} must be an int32 tensor of shape [{B}]")
    need(t.device == dev, f"{name} must be on {dev}")
    return t.contiguous()


def _args(q, k, v, scale, causal, kv_len, q_start):
    for n, t in (("q", q), ("k", k), ("v", v)):
        need(t.dim() == 4, f"{n} must be [batch, tokens, heads, channels]")
    B, Tq, Hq, D = q.shape
    Tk, Hk = k.shape[1], k.shape[2]
    need(q.dtype in DTYPES and k.dtype == q.dtype and v.dtype == q.dtype, "q, k, v must have one type: fp32, bf16 or fp16")
    need(k.shape == (B, Tk, Hk, D) and v.shape == k.shape, f"k, v must be [{B}, tokens, heads, {D}] and alike")
    need(Hk > 0 and Hq > 0 and Hq % Hk == 0, f"{Hq} query heads are not a multiple of {Hk} key-value heads")
    ce = 16 // q.element_size()
    need(0 < D <= 128 and D % ce == 0, f"head width {D}: at most 128 and a multiple of {ce}")
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    need(0.0 < scale < 3e38, f"scale must be positive and finite, got {scale}")
    dev = same_device(q, k, v)
    kv_len, q_start = _int_arg(kv_len, B, "kv_len", dev), _int_arg(q_start, B, "q_start", dev)
    q, k, v = _lay(q), _lay(k), _lay(v)
    a = AttentionArgs(dtype=DTYPES[q.dtype], B=B, Tq=Tq, Tk=Tk, Hq=Hq, Hk=Hk, D=D, causal=int(bool(causal)), scale=scale)
    a.q, a.k, a.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
    a.q_s, a.k_s, a.v_s = _st(q), _st(k), _st(v)
    a.kv_len = None if kv_len is None else kv_len.data_ptr()
    a.q_start = None if q_start is None else q_start.data_ptr()
    return a, (q, k, v, kv_len, q_start), dev


def _into(t, like, name):
    """A caller's output tensor (checked) or a new contiguous one."""
    if t is None:
        return torch.empty(like.shape, dtype=like.dtype, device=like.device)
    need(t.shape == like.shape and t.dtype == like.dtype and t.device == like.device, f"{name} must be like its input")
    need(_lay(t) is t, f"{name}: adjacent channels, 16-byte aligned, strides in multiples of 16 bytes")
    return t


def attention(q, k, v, scale=None, causal=False, kv_len=None, q_start=None, out=None):
    """(out, lse): attention of every query row, and its log-sum-exp fp32 [B, Hq, Tq]."""
    a, keep, dev = _args(q, k, v, scale, causal, kv_len, q_start)
    out = _into(out, q, "out")
    lse = torch.empty(a.B, a.Hq, a.Tq, dtype=torch.float32, device=dev)
    a.out, a.out_s, a.lse = out.data_ptr(), _st(out), lse.data_ptr()
    L = lib()
    with torch.cuda.device(dev):
        n = L.ifd_op_attention_ws_bytes(ctypes.byref(a))
        ws = workspace(n, dev)
        _lib.check(L.ifd_op_attention(ctypes.byref(a), _lib.ptr(ws), n, _lib.stream_ptr(dev)))
    return out, lse


def attention_bwd(dout, q, k, v, out, lse, scale=None, causal=False, kv_len=None, q_start=None, dq=None, dk=None, dv=None):
    """(dq, dk, dv) from the gradient of `out`; out, lse and the other arguments as the forward call had them.
    Keys at and past kv_len get zero gradients."""
    a, keep, dev = _args(q, k, v, scale, causal, kv_len, q_start)
    for n, t in (("dout", dout), ("out", out)):
        need(t.shape == q.shape and t.dtype == q.dtype, f"{n} must be like q")
    need(lse.shape == (a.B, a.Hq, a.Tq) and lse.dtype == torch.float32, f"lse must be fp32 [{a.B}, {a.Hq}, {a.Tq}]")
    same_device(q, dout, out, lse)
    dout, out, lse = _lay(dout), _lay(out), lse.contiguous()
    dq, dk, dv = _into(dq, q, "dq"), _into(dk, k, "dk"), _into(dv, v, "dv")
    for n in ("dout", "out", "dq", "dk", "dv"):
        t = locals()[n]
        setattr(a, n, t.data_ptr())
        setattr(a, n + "_s", _st(t))
    a.lse = lse.data_ptr()
    L = lib()
    with torch.cuda.device(dev):
        n = L.ifd_op_attention_bwd_ws_bytes(ctypes.byref(a))
        ws = workspace(n, dev)
        _lib.check(L.ifd_op_attention_bwd(ctypes.byref(a), _lib.ptr(ws), n, _lib.stream_ptr(dev)))
    return dq, dk, dv
