"""The operators of include/ifd_ops.h without a GPU: exported symbols, argument checks of the C ABI and of the Python
layer (every refusal happens on the host, before anything is launched)."""
import ctypes
import os
import re

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_library_exports_ops_header_symbols():
    src = open(os.path.join(ROOT, "include", "ifd_ops.h")).read()
    syms = sorted(set(re.findall(r"\b(ifd_op_[a-z_0-9]+)\s*\(", src)))
    from ifd import _ops
    L = _ops.lib()
    for s in syms:
        assert hasattr(L, s), s
    assert set(syms) == set(_ops.OPS_EXPORTS)


def _attention_args(**kw):
    """Valid arguments with made-up addresses: only the checks run."""
    from ifd._ops import AttentionArgs, Strides
    d = dict(dtype=1, B=2, Tq=8, Tk=16, Hq=4, Hk=2, D=64, causal=0, scale=0.125)
    ptrs = {n: 0x10000 for n in ("q", "k", "v", "out", "lse", "dout", "dq", "dk", "dv")}
    for k, v in kw.items():
        (ptrs if k in ptrs else d)[k] = v
    strides = {n: d.pop(n) for n in list(d) if n.endswith("_s")}
    a = AttentionArgs(**d)
    for n, p in ptrs.items():
        setattr(a, n, p)
    for n in ("q", "k", "v", "out", "dout", "dq", "dk", "dv"):
        T, H = (a.Tk, a.Hk) if n in ("k", "v", "dk", "dv") else (a.Tq, a.Hq)
        setattr(a, n + "_s", Strides(*strides.get(n + "_s", (T * H * a.D, H * a.D, a.D))))
    return a


BAD = [
    (dict(dtype=7), "dtype"), (dict(B=-1), "sizes"), (dict(Hk=0), "sizes"), (dict(Hk=3), "multiple"),
    (dict(D=136), "head width"), (dict(D=20), "head width"), (dict(D=6, dtype=0), "head width"),
    (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(q=None), "null tensor"), (dict(k=0x10008), "aligned"),
    (dict(v_s=(1024, 132, 64)), "strides"), (dict(out_s=(1 << 30, 1 << 23, 64)), "token stride"),
    (dict(q_s=(1024, -256, 64)), "token stride"), (dict(lse=None), "lse"), (dict(Tk=1 << 30), "2^30"),
]


@pytest.mark.parametrize("kw,msg", BAD, ids=lambda x: str(x)[:40])
def test_attention_refusals(kw, msg):
    from ifd import _lib, _ops
    L = _ops.lib()
    for name in ("ifd_op_attention", "ifd_op_attention_bwd"):
        rc = getattr(L, name)(ctypes.byref(_attention_args(**kw)), None, 1 << 40, None)
        with pytest.raises(RuntimeError, match=name + ": .*" + re.escape(msg)):
            _lib.check(rc)


def test_attention_workspace_and_empty_calls():
    from ifd import _lib, _ops
    L = _ops.lib()
    a = _attention_args(B=2, Tq=1, Tk=8192, Hq=8, Hk=2, D=128)
    n = L.ifd_op_attention_ws_bytes(ctypes.byref(a))
    assert n > 0
    with pytest.raises(RuntimeError, match="workspace"):
        _lib.check(L.ifd_op_attention(ctypes.byref(a), 0x10000, n - 1, None))
    with pytest.raises(RuntimeError, match="workspace"):
        _lib.check(L.ifd_op_attention(ctypes.byref(a), None, n, None))
    b = L.ifd_op_attention_bwd_ws_bytes(ctypes.byref(a))
    with pytest.raises(RuntimeError, match="workspace"):
        _lib.check(L.ifd_op_attention_bwd(ctypes.byref(a), 0x10000, b - 1, None))
    # scratch is linear in the tensors: no score matrix
    a = _attention_args(B=1, Tq=16384, Tk=16384, Hq=8, Hk=8, D=64)
    assert L.ifd_op_attention_bwd_ws_bytes(ctypes.byref(a)) < 64 * 8 * 16384 * 64 * 4
    for kw in (dict(B=0), dict(Tq=0)):  # nothing to do: no launch
        assert L.ifd_op_attention(ctypes.byref(_attention_args(**kw)), None, 0, None) == 0
    assert L.ifd_op_attention_bwd(ctypes.byref(_attention_args(B=0)), None, 0, None) == 0
    assert L.ifd_op_attention(None, None, 0, None) != 0


def test_attention_python_refusals():
    from ifd.attention import attention, attention_bwd
    q, k = torch.zeros(2, 8, 4, 64), torch.zeros(2, 16, 2, 64)
    bad = [
        (q[0], k, k, {}, "batch, tokens"), (q, k.half(), k, {}, "one type"), (q.double(), k.double(), k.double(), {}, "one type"),
        (q, k, k[:, :8], {}, "alike"), (q, k[..., :32], k[..., :32], {}, "k, v must be"),
        (q[:, :, :3], k, k, {}, "multiple of 2"), (q[..., :3], k[..., :3], k[..., :3], {}, "head width"),
        (q, k, k, dict(scale=0.0), "scale"), (q, k, k, {}, "GPU tensor"),
    ]
    for a, b, c, kw, msg in bad:
        with pytest.raises(ValueError, match=msg):
            attention(a, b, c, **kw)
        with pytest.raises(ValueError, match=msg):
            attention_bwd(a, a, b, c, a, None, **kw)
