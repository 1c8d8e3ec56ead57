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


def test_packed_arguments_have_the_structures_layout():
    from ifd import _ops, attention, rotary
    assert ctypes.sizeof(_ops.AttentionArgs) == attention._FWD.size + attention._BWD.size
    assert _ops.AttentionArgs.dout.offset == attention._FWD.size
    assert ctypes.sizeof(_ops.QkArgs) == rotary._HEAD.size + rotary._MORE.size
    assert _ops.QkArgs.gq.offset == rotary._HEAD.size


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


def test_qk_refusals():
    from ifd import _lib, _ops
    from ifd.rotary import Rotary, qk_norm_rope, qk_norm_rope_bwd
    L = _ops.lib()
    S = _ops.Strides
    good = dict(dtype=1, B=1, T=2, Hq=2, Hk=1, D=64, rot=64, norm=1, eps=1e-6, mscale=1.0)
    for kw, msg in ((dict(dtype=3), "dtype"), (dict(D=130), "head width"), (dict(D=63), "head width"), (dict(rot=66), "rotated"),
                    (dict(rot=3), "rotated"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(B=-1), "sizes"),
                    ({}, "null tensor")):
        a = _ops.QkArgs(**{**good, **kw})
        for name, args in (("ifd_op_qk_norm_rope", ()), ("ifd_op_qk_norm_rope_bwd", (None, 1 << 30))):
            with pytest.raises(RuntimeError, match=name + ": .*" + msg):
                _lib.check(getattr(L, name)(ctypes.byref(a), *args, None))
    a = _ops.QkArgs(**good)
    for n in ("q", "k", "q_out", "k_out", "gq", "gk", "dq", "dk"):
        setattr(a, n, 0x10000)
    with pytest.raises(RuntimeError, match="positions"):
        _lib.check(L.ifd_op_qk_norm_rope(ctypes.byref(a), None))
    a.pos = a.turns = 0x10000
    need = L.ifd_op_qk_norm_rope_bwd_ws_bytes(ctypes.byref(a))
    with pytest.raises(RuntimeError, match="workspace"):
        _lib.check(L.ifd_op_qk_norm_rope_bwd(ctypes.byref(a), 0x10000, need - 1, None))
    assert L.ifd_op_qk_norm_rope(ctypes.byref(_ops.QkArgs(**{**good, "T": 0})), None) == 0
    for args, kw in (((0,), {}), ((7,), {}), ((64,), dict(base=1.0)), ((64,), dict(scaling=("cubic", 2.0))),
                     ((64,), dict(scaling=("linear", 0.5))), ((64,), dict(scaling=("bands", 2.0))),
                     ((64,), dict(scaling=("bands", 2.0, 0)))):
        with pytest.raises(ValueError):
            Rotary(*args, device="cpu", **kw)
    rope, q, k = Rotary(64, device="cpu"), torch.zeros(1, 2, 2, 64), torch.zeros(1, 2, 1, 64)
    pos = torch.arange(2)
    for a, kw, msg in (((q[0], k), {}, "tokens, heads"), ((q, k.half()), {}, "one type"), ((q, k[:, :1]), {}, "k must be"),
                       ((q[..., :32], k[..., :32], None, None, pos, rope), {}, "rotated channels"),
                       ((q, k, None, None, None, rope), {}, "positions"), ((q, k, torch.ones(64)), dict(norm=False), "weights"),
                       ((q, k), dict(eps=-1.0), "eps"), ((q, k), {}, "GPU tensor")):
        with pytest.raises(ValueError, match=msg):
            qk_norm_rope(*a, **kw)
        with pytest.raises(ValueError, match=msg):
            qk_norm_rope_bwd(a[0], a[1], *a, **kw)
    del S


def test_rotary_frequencies():
    """The scalings' defining properties, in fp64."""
    import math
    from ifd.rotary import Rotary
    plain = Rotary(64, device="cpu").inv_freq
    assert plain[0] == 1.0 and abs(plain[16].item() - 10000.0 ** -0.5) < 1e-15
    assert torch.allclose(Rotary(64, scaling=("linear", 4.0), device="cpu").inv_freq, plain / 4, rtol=1e-15)
    wide = Rotary(64, scaling=("base", 4.0), device="cpu").inv_freq
    assert wide[0] == 1.0 and abs(wide[-1] / plain[-1] - 0.25) < 1e-12
    r = Rotary(64, scaling=("bands", 4.0, 4096), device="cpu")
    turns = 4096 * plain / (2 * math.pi)
    assert torch.equal(r.inv_freq[turns >= 32], plain[turns >= 32])
    assert torch.allclose(r.inv_freq[turns <= 1], plain[turns <= 1] / 4, rtol=1e-15)
    assert ((r.inv_freq <= plain) & (r.inv_freq >= plain / 4 * (1 - 1e-12))).all() and abs(r.mscale - 1.1386294) < 1e-6


def _adamw_args(keep, **kw):
    from ifd._ops import AdamwArgs
    c = ctypes
    n = kw.pop("n", [300, 5])
    p, g = kw.pop("p", [0x10000] * len(n)), kw.pop("g", [0x20000] * len(n))
    d = dict(nt=len(n), bits=8, step=1, block0=0, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, wd=0.0)
    arr = dict(p=(c.c_void_p * len(n))(*p), g=(c.c_void_p * len(n))(*g), n=(c.c_int64 * len(n))(*n),
               ptype=(c.c_uint8 * len(n))(*kw.pop("ptype", [0] * len(n))),
               gtype=(c.c_uint8 * len(n))(*kw.pop("gtype", [0] * len(n))))
    st = {s: kw.pop(s, 0x30000) for s in ("m", "v", "m_scale", "v_scale")}
    a = AdamwArgs(**{**d, **kw})
    keep.append(arr)
    for k, v in arr.items():
        setattr(a, k, c.cast(v, c.c_void_p))
    for k, v in st.items():
        setattr(a, k, v)
    return a


def test_adamw_refusals():
    from ifd import _lib, _ops
    L, keep = _ops.lib(), []
    for kw, msg in ((dict(bits=16), "8 or 32"), (dict(step=0), "step"), (dict(b1=1.0), "b1"), (dict(b2=-0.1), "b2"),
                    (dict(eps=0.0), "eps"), (dict(nt=-1), "tensor list"), (dict(n=[-1, 2]), "size"),
                    (dict(gtype=[9, 0]), "gradient type"), (dict(ptype=[3, 0]), "parameter type"),
                    (dict(p=[None, 0x10000]), "without its parameter"), (dict(p=[0x10002, 0x10000]), "element"),
                    (dict(g=[0x20001, 0x20000]), "element"), (dict(m=None), "null"), (dict(v_scale=None), "null"),
                    (dict(m=0x30008), "aligned"), (dict(n=[1 << 39, 1]), "size"), (dict(n=[1 << 37] * 5, p=[0x10000] * 5), "blocks"),
                    (dict(block0=-1), "block0")):
        if "n" in kw and len(kw["n"]) == 5:
            kw["g"] = [0x20000] * 5
        with pytest.raises(RuntimeError, match="ifd_op_adamw: .*" + msg):
            _lib.check(L.ifd_op_adamw(ctypes.byref(_adamw_args(keep, **kw)), None))
    assert L.ifd_op_adamw(ctypes.byref(_adamw_args(keep, g=[None, None])), None) == 0  # no gradients: nothing to do
    n, g, t = (ctypes.c_int64 * 1)(5000), (ctypes.c_void_p * 1)(0x20000), (ctypes.c_uint8 * 1)(0)
    need = L.ifd_op_grad_norm_ws_bytes(1, n)
    assert need > 0
    for args, msg in (((1, g, n, t, 1.0, None, 0x30000, need), "norm_coef"), ((1, g, n, t, -1.0, 0x30000, 0x30000, need), "max_norm"),
                      ((1, g, n, t, 1.0, 0x30000, 0x30000, need - 1), "workspace"), ((1, None, n, t, 1.0, 0x30000, 0x30000, need), "list")):
        with pytest.raises(RuntimeError, match="ifd_op_grad_norm: .*" + msg):
            _lib.check(L.ifd_op_grad_norm(*args, None))
    for args, msg in (((None, None, None, None, 4, None, None), "null"), ((0x1, 0x4, 0x4, 0x4, 4, 0x10, 0x10), "aligned"),
                      ((None, None, None, None, -1, None, None), "nblocks")):
        with pytest.raises(RuntimeError, match="ifd_op_state_values: .*" + msg):
            _lib.check(L.ifd_op_state_values(*args, None))
    assert L.ifd_op_state_values(None, None, None, None, 0, None, None, None) == 0


def test_adamw_python_refusals():
    from ifd.optim import AdamW
    p = torch.zeros(8)
    for args, kw, msg in ((([p],), dict(state_bits=16), "state_bits"), (([p],), dict(betas=(1.0, 0.9)), "betas"),
                          (([p],), dict(eps=0.0), "eps"), (([p],), dict(max_norm=0.0), "max_norm"), (([],), {}, "no parameters"),
                          (([p.double()],), {}, "contiguous fp32"), (([torch.zeros(4, 4).t()[:, :2]],), {}, "contiguous"),
                          (([p, p],), {}, "twice"), (([p],), {}, "GPU tensor"), (([{"params": [p]}, p],), {}, "groups")):
        with pytest.raises(ValueError, match=msg):
            AdamW(*args, **kw)


def test_overlap_of_outputs_and_inputs():
    from ifd.attention import _may_overlap
    x = torch.zeros(2, 6, 8, 16)
    q, k, v = x[:, :, :4], x[:, :, 4:6], x[:, :, 6:]
    assert not _may_overlap(q, k) and not _may_overlap(k, q) and not _may_overlap(v, k) and not _may_overlap(q, torch.zeros_like(q))
    assert _may_overlap(q, q) and _may_overlap(q, x[:, :, 3:5]) and _may_overlap(x[:, 1:, :4], x[:, :5, :4])
    assert not _may_overlap(x[:1], x[1:]) and not _may_overlap(x[:, :0], x)
    assert _may_overlap(x, x.transpose(1, 2))
    y = torch.zeros(2, 4, 6, 16)  # [B, H, T, D] in memory: other rows, so nothing is told apart
    assert _may_overlap(y.transpose(1, 2)[:, :, :2], y.transpose(1, 2)[:, :, 1:])


def test_overlap_of_parameters_and_of_two_outputs(monkeypatch):
    from ifd import _ops, attention, optim, rotary
    for m in (_ops, attention, optim, rotary):
        if hasattr(m, "same_device"):
            monkeypatch.setattr(m, "same_device", lambda *t: t[0].device)
    x = torch.zeros(100)
    with pytest.raises(ValueError, match="share memory"):
        optim.AdamW([x[:60], x[50:]])
    optim.AdamW([x[:50], x[50:], x[:0]])
    q, k = torch.zeros(1, 3, 2, 16), torch.zeros(1, 3, 2, 16)
    o = torch.zeros(1, 3, 4, 16)
    with pytest.raises(ValueError, match="k_out overlaps"):
        rotary.qk_norm_rope(q, k, q_out=o[:, :, :2], k_out=o[:, :, 1:3])
    with pytest.raises(ValueError, match="q_out overlaps"):
        rotary.qk_norm_rope(q, k, q_out=k)
    with pytest.raises(ValueError, match="q_out overlaps"):
        rotary.qk_norm_rope(o[:, :, :2], None, q_out=o[:, :, 1:3])
    with pytest.raises(ValueError, match="dq overlaps"):
        rotary.qk_norm_rope_bwd(q.clone(), k.clone(), q, k, dq=q)
    lse = torch.zeros(1, 2, 3)
    with pytest.raises(ValueError, match="dv overlaps"):
        attention.attention_bwd(q.clone(), q, k, k.clone(), q.clone(), lse, dk=o[:, :, :2], dv=o[:, :, :2])


@pytest.mark.parametrize("kw", [dict(B=1, Tq=129, Tk=2100, Hq=1, Hk=1, D=128), dict(B=3, Tq=33, Tk=1000, Hq=1, Hk=1, D=64, dtype=0),
                                dict(B=1, Tq=1, Tk=700, Hq=1, Hk=1, D=96), dict(B=1, Tq=777, Tk=777, Hq=3, Hk=3, D=80, causal=1)])
def test_backward_workspace_parts_are_aligned(kw):
    """The partial sums behind lse2 and delta (2 B Hq Tq floats, here an odd number of pairs) are written in 16-byte pieces:
    their start has to be a multiple of 16 bytes, as all that follows it is."""
    from ifd import _ops
    assert kw["B"] * kw["Hq"] * kw["Tq"] % 2
    n = _ops.lib().ifd_op_attention_bwd_ws_bytes(ctypes.byref(_attention_args(**kw)))
    assert n > 8 * kw["B"] * kw["Hq"] * kw["Tq"] and n % 16 == 0


def test_addresses_off_their_elements_are_refused():
    """Every array that a kernel reads or writes element by element starts on a multiple of its element."""
    from ifd import _lib, _ops
    L, keep = _ops.lib(), []
    for n in ("lse", "kv_len", "q_start"):
        a = _attention_args()
        setattr(a, n, 0x10002)
        for name in ("ifd_op_attention", "ifd_op_attention_bwd"):
            with pytest.raises(RuntimeError, match=name + ": .*address"):
                _lib.check(getattr(L, name)(ctypes.byref(a), 0x10000, 1 << 40, None))
    good = dict(dtype=1, B=1, T=2, Hq=2, Hk=1, D=64, rot=64, norm=1, eps=1e-6, mscale=1.0)
    ptrs = ("q", "k", "q_out", "k_out", "gq", "gk", "dq", "dk", "wq", "wk", "pos", "turns", "dwq", "dwk")
    for n in ptrs:
        a = _ops.QkArgs(**good)
        for m in ptrs:
            setattr(a, m, 0x10000)
        setattr(a, n, 0x10001 if n[0] in "qkgd" and n[:2] != "dw" else 0x10002 if n[0] in "wd" else 0x10004)
        if n not in ("gq", "gk", "dq", "dk", "dwq", "dwk"):
            with pytest.raises(RuntimeError, match="ifd_op_qk_norm_rope: .*address"):
                _lib.check(L.ifd_op_qk_norm_rope(ctypes.byref(a), None))
        if n not in ("q_out", "k_out"):
            with pytest.raises(RuntimeError, match="ifd_op_qk_norm_rope_bwd: .*address"):
                _lib.check(L.ifd_op_qk_norm_rope_bwd(ctypes.byref(a), 0x10000, 1 << 30, None))
    with pytest.raises(RuntimeError, match="ifd_op_qk_norm_rope_bwd: .*address"):
        for m in ptrs:
            setattr(a, m, 0x10000)
        _lib.check(L.ifd_op_qk_norm_rope_bwd(ctypes.byref(a), 0x10002, 1 << 30, None))
    n, g, t = (ctypes.c_int64 * 1)(5000), (ctypes.c_void_p * 1)(0x20000), (ctypes.c_uint8 * 1)(0)
    for coef, ws in ((0x30004, 0x30000), (0x30000, 0x30004)):
        with pytest.raises(RuntimeError, match="ifd_op_grad_norm: .*address"):
            _lib.check(L.ifd_op_grad_norm(1, g, n, t, 1.0, coef, ws, 1 << 20, None))
    for kw in (dict(m_scale=0x30002), dict(v_scale=0x30001), dict(norm_coef=0x30004)):
        with pytest.raises(RuntimeError, match="ifd_op_adamw: .*address"):
            _lib.check(L.ifd_op_adamw(ctypes.byref(_adamw_args(keep, **kw)), None))
    for args in ((0x10, 0x2, 0x10, 0x10), (0x10, 0x10, 0x10, 0x2)):
        with pytest.raises(RuntimeError, match="ifd_op_state_values: .*address"):
            _lib.check(L.ifd_op_state_values(*args, 4, 0x10, 0x10, None))


def test_shares_of_wide_fp32_heads_count_the_kernels_tiles():
    """Shares of the keys in the many-row forward kernel: four tiles at least in fp32, and a tile of heads of 65 to 128
    channels is 32 keys (64 of narrower ones). 700 keys of 80 channels are 22 tiles, five shares, and not half as many. Heads
    of 65 to 96 channels take eight tiles where four would make more than 256 workgroups."""
    from ifd import _ops
    for D, dp, keys in ((64, 64, 64), (80, 96, 32), (96, 96, 32), (128, 128, 32)):
        for Tq, Tk in ((700, 700), (200, 3000), (129, 257), (2000, 2000), (500, 1100)):
            kw = dict(dtype=0, B=1, Tq=Tq, Tk=Tk, Hq=4, Hk=4, D=D)
            n = _ops.lib().ifd_op_attention_ws_bytes(ctypes.byref(_attention_args(**kw)))
            wgs, tiles = -(-Tq // 128) * 4, -(-Tk // keys)
            shares = max(tiles // 8, min(tiles // 4, 256 // wgs)) if dp == 96 else tiles // 4
            want = min(512 // wgs, shares, 64)
            assert n == (4 * Tq * want * (dp + 4) * 4 if want > 1 else 0), (D, Tq, Tk)
