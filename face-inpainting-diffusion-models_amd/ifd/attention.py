"""Attention with its log-sum-exp, and its backward pass (csrc/attn_fwd.hip, csrc/attn_bwd.hip).

    out, lse = attention(q, k, v, causal=True)
    dq, dk, dv = attention_bwd(dout, q, k, v, out, lse, causal=True)

q, out: [B, Tq, Hq, D]; k, v: [B, Tk, Hk, D]; one type (fp32, bf16, fp16); Hq a multiple of Hk, query head h reads
key-value head h // (Hq // Hk). D <= 128 and a multiple of 8 (4 in fp32). Any strides with the channels adjacent, e.g. the
three slices of a packed projection or a slice of a longer key-value cache; tensors whose strides are not multiples of
16 bytes (or which are not 16-byte aligned) are copied first.

Row i of sequence b sees key j when j < kv_len[b] (default Tk) and, with causal=True, j <= q_start[b] + i (default
Tk - Tq: the rows are the last ones). kv_len, q_start: int32 [B] on the GPU, read by the kernels (no synchronisation).
Keys that no row of their sequence sees (at and past kv_len, or behind the last row's) change nothing, whatever they hold.
A key that some rows see and others not must be finite in v (for the backward pass in k too), or it may spoil those others;
so may, in the backward pass, a row that sees some keys and is not finite in q, out or dout the gradients of the others.
A row that sees no key gets out = 0, lse = -inf and zero gradients, whatever q and dout hold there. Output tensors of the
caller (out, dq, dk, dv) must not overlap the inputs, each other or themselves (strides must nest).

The backward pass keeps no score matrix: it recomputes the probabilities from lse. Both directions are deterministic. Scores
(scale q.k) may reach 1e8 in magnitude; from 4e8 on results are not finite. In fp16 small gradients need a loss scale.
Calls run on the current stream of the tensors' device and can be captured into a graph. They record nothing for autograd:
tensors that require gradients are refused unless under torch.no_grad(), tensors with a forward-mode tangent always.
"""
from __future__ import annotations

import math
import struct

import torch

from ._ops import DTYPES, call, lib, may_overlap as _may_overlap, no_grad, output, refuse, same_device, workspace

# ifd_attention_args (include/ifd_ops.h): packed here because filling a ctypes structure field by field costs more than
# the smallest kernels run (_ops.AttentionArgs has the same layout)
_FWD, _BWD = struct.Struct("8if i 7P 12q"), struct.Struct("4P 12q")
_NO_BWD = bytes(_BWD.size)


def _lay(t, e):
    """t itself when the kernels can read it (elements of e bytes), else a contiguous copy."""
    s0, s1, s2, s3 = t.stride()
    if s3 == 1 and 0 <= s1 * e < 1 << 24 and not ((s0 | s1 | s2) * e | t.data_ptr()) & 15:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _int_arg(t, B, name, dev):
    if not (isinstance(t, torch.Tensor) and t.dtype == torch.int32 and t.shape == (B,)):
        refuse(f"{name} must be an int32 tensor of shape [{B}]")
    if t.device != dev:
        refuse(f"{name} must be on {dev}")
    return t.contiguous()


def _inputs(q, k, v, scale, kv_len, q_start):
    """Checked inputs: (q, k, v as the kernels read them, scale, kv_len, q_start, device)."""
    dt = q.dtype
    if not q.dim() == k.dim() == v.dim() == 4:
        refuse("q, k, v must be [batch, tokens, heads, channels]")
    B, _, Hq, D = q.shape
    kB, Tk, Hk, kD = k.shape
    if not (dt in DTYPES and k.dtype is dt and v.dtype is dt):
        refuse(f"q, k, v must have one type, fp32, bf16 or fp16, got {q.dtype}, {k.dtype}, {v.dtype}")
    if kB != B or kD != D or v.shape != k.shape:
        refuse(f"k, v must be [{B}, tokens, heads, {D}] and alike, got {tuple(k.shape)} and {tuple(v.shape)}")
    if not (Hk > 0 and Hq > 0 and Hq % Hk == 0):
        refuse(f"{Hq} query heads are not a multiple of {Hk} key-value heads")
    e = 4 if dt is torch.float32 else 2
    if not 0 < D <= 128 or D * e & 15:
        refuse(f"head width {D}: at most 128 and a multiple of {16 // e}")
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not 0.0 < scale < 3e38:
        refuse(f"scale must be positive and finite, got {scale}")
    dev = same_device(q, k, v)
    no_grad(q, k, v)
    if kv_len is not None:
        kv_len = _int_arg(kv_len, B, "kv_len", dev)
    if q_start is not None:
        q_start = _int_arg(q_start, B, "q_start", dev)
    return _lay(q, e), _lay(k, e), _lay(v, e), scale, kv_len, q_start, dev


def _pack(q, k, v, scale, causal, kv_len, q_start, out, lse):
    B, Tq, Hq, D = q.shape
    return _FWD.pack(DTYPES[q.dtype], B, Tq, k.shape[1], Hq, k.shape[2], D, 1 if causal else 0, scale, 0, q.data_ptr(),
                     k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(), 0 if kv_len is None else kv_len.data_ptr(),
                     0 if q_start is None else q_start.data_ptr(), *q.stride()[:3], *k.stride()[:3], *v.stride()[:3],
                     *out.stride()[:3])


def _into(t, like, name, *inputs):
    """A caller's output tensor (checked) or a new contiguous one."""
    if t is None:
        return torch.empty_like(like, memory_format=torch.contiguous_format)
    if not (t.dim() == 4 and _lay(t, t.element_size()) is t):
        refuse(f"{name}: adjacent channels, 16-byte aligned, strides in multiples of 16 bytes")
    if any(_may_overlap(t, x) for x in inputs):
        refuse(f"{name} overlaps an input or another output")
    return output(t, like, name)


def attention(q, k, v, scale=None, causal=False, kv_len=None, q_start=None, out=None):
    """(out, lse): attention of every query row, and its log-sum-exp fp32 [B, Hq, Tq]."""
    q, k, v, scale, kv_len, q_start, dev = _inputs(q, k, v, scale, kv_len, q_start)
    out = _into(out, q, "out", q, k, v)
    lse = q.new_empty((q.shape[0], q.shape[2], q.shape[1]), dtype=torch.float32)
    a = _pack(q, k, v, scale, causal, kv_len, q_start, out, lse) + _NO_BWD
    L = lib()
    n = L.ifd_op_attention_ws_bytes(a)
    ws = workspace(n, q)
    call(L.ifd_op_attention, dev, a, None if ws is None else ws.data_ptr(), n)
    return out, lse


def attention_bwd(dout, q, k, v, out, lse, scale=None, causal=False, kv_len=None, q_start=None, dq=None, dk=None, dv=None):
    """(dq, dk, dv) from the gradient of `out`; out, lse and the other arguments as the forward call had them.
    Keys at and past kv_len get zero gradients."""
    q, k, v, scale, kv_len, q_start, dev = _inputs(q, k, v, scale, kv_len, q_start)
    shape, dt = q.shape, q.dtype
    for n, t in (("dout", dout), ("out", out)):
        if not (t.shape == shape and t.dtype is dt):
            refuse(f"{n} must be like q")
    if lse.shape != (shape[0], shape[2], shape[1]) or lse.dtype is not torch.float32:
        refuse("lse must be the forward's, fp32 [B, Hq, Tq]")
    same_device(q, dout, out, lse)
    no_grad(dout, out, lse)
    e = 4 if dt is torch.float32 else 2
    dout, out, lse = _lay(dout, e), _lay(out, e), lse.contiguous()
    ins = (q, k, v, dout, out)
    dq = _into(dq, q, "dq", *ins)
    dk = _into(dk, k, "dk", *ins, dq)
    dv = _into(dv, v, "dv", *ins, dq, dk)
    a = _pack(q, k, v, scale, causal, kv_len, q_start, out, lse) + _BWD.pack(
        dout.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), *dout.stride()[:3], *dq.stride()[:3],
        *dk.stride()[:3], *dv.stride()[:3])
    L = lib()
    n = L.ifd_op_attention_bwd_ws_bytes(a)
    ws = workspace(n, q)
    call(L.ifd_op_attention_bwd, dev, a, None if ws is None else ws.data_ptr(), n)
    return dq, dk, dv
