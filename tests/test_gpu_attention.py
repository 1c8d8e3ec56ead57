"""Attention and its backward pass (ifd.attention, csrc/attn_fwd.hip, csrc/attn_bwd.hip) against the formulas in fp64.

Tolerances, per element, from the roundings that the kernels make (eps = finfo(type).eps):
  out: P is rounded once to the type (16-bit), the result once. |err| <= eps/2 * (sum_j p_j |v_j| + |out|), times 1.25 for
       the fp32 sums and exponentials beneath it; fp32: products and sums of n <= 512 terms, exponent arguments up to
       |s| 2^-24 each: 40 eps (sum_j p_j |v_j|).
  lse: fp32 sums and logarithm of values up to |lse|: 1e-5 (1 + |lse|).
  dv:  P rounded once, the result once; the same form over the rows: eps/2 * (sum_i p_ij |dout_i| + |dv|) * 1.25.
  dk, dq: dS rounded once (after P, dP, delta in fp32; delta uses the type-rounded out, as the definition does):
       eps/2 * (scale sum |ds| |q| + |dq|) * 1.25, and the fp32 error of dP - delta (a sum of D products with
       cancellation): 2^-24 * 64 * scale * sum p (|dout| |v| + |delta|) |q|.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def _visible(B, Tq, Tk, causal, kv_len, q_start):
    j = torch.arange(Tk)
    n = torch.full((B,), Tk) if kv_len is None else torch.as_tensor(kv_len)
    keep = (j[None, None] < n[:, None, None]).expand(B, Tq, Tk).clone()
    if causal:
        s = torch.full((B,), Tk - Tq) if q_start is None else torch.as_tensor(q_start)
        keep &= j[None, None] <= (s[:, None] + torch.arange(Tq))[:, :, None]
    return keep


def _ref(q, k, v, keep, scale, dout=None, out_given=None):
    """fp64 on the CPU: outputs and, per output, the sums that its tolerance counts."""
    q, k, v = (t.detach().cpu().double().transpose(1, 2) for t in (q, k, v))
    G = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    keep = keep[:, None]
    v = torch.where(keep.any(2)[..., None], v, torch.zeros((), dtype=v.dtype))  # keys nobody sees may hold anything
    k = torch.where(keep.any(2)[..., None], k, torch.zeros((), dtype=v.dtype))
    s = (q @ k.transpose(-1, -2)) * scale
    s = s.masked_fill(~keep, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.where(keep, torch.exp(s - torch.where(torch.isinf(lse), 0.0, lse)[..., None]), 0.0)
    out = p @ v
    r = dict(out=out.transpose(1, 2), lse=lse, out_b=(p @ v.abs()).transpose(1, 2))
    if dout is None:
        return r
    do = dout.detach().cpu().double().transpose(1, 2)
    o = out_given.detach().cpu().double().transpose(1, 2)
    delta = (do * o).sum(-1, keepdim=True)
    ds = p * (do @ v.transpose(-1, -2) - delta)
    rough = p * (do.abs() @ v.abs().transpose(-1, -2) + (do * o).abs().sum(-1, keepdim=True))

    def fold(x):
        B, H, T, D = x.shape
        return x.view(B, H // G, G, T, D).sum(2).transpose(1, 2)

    r.update(dq=(ds @ k).transpose(1, 2) * scale, dq_b=(ds.abs() @ k.abs()).transpose(1, 2) * scale,
             dq_f=(rough @ k.abs()).transpose(1, 2) * scale,
             dk=fold(ds.transpose(-1, -2) @ q) * scale, dk_b=fold(ds.abs().transpose(-1, -2) @ q.abs()) * scale,
             dk_f=fold(rough.transpose(-1, -2) @ q.abs()) * scale,
             dv=fold(p.transpose(-1, -2) @ do), dv_b=fold(p.transpose(-1, -2) @ do.abs()))
    return r


def _within(got, ref, tol, name):
    got = got.detach().cpu().double()
    assert torch.isfinite(got).all(), f"{name}: not finite"
    bad = (got - ref).abs() - tol
    assert (bad <= 0).all(), f"{name}: off by {(got - ref).abs().max():.3e}, past its tolerance by {bad.max():.3e}"


def _check_fwd(out, lse, r, dt):
    eps = torch.finfo(dt).eps
    t = 40 * eps * r["out_b"] if dt == F32 else 0.5 * eps * (r["out_b"] + r["out"].abs()) * 1.25
    _within(out, r["out"], t + 1e-30 if dt != HF else t + 6e-8, "out")
    got, fin = lse.cpu().double(), torch.isfinite(r["lse"])
    assert torch.equal(torch.isneginf(got), torch.isneginf(r["lse"])), "rows without keys"
    assert ((got - r["lse"]).abs()[fin] <= 1e-5 * (1 + r["lse"].abs()[fin])).all(), "lse"
    assert (out.cpu().double()[~fin.transpose(1, 2)] == 0).all(), "rows without keys must be 0"


def _check_bwd(dq, dk, dv, r, dt):
    eps = torch.finfo(dt).eps
    sub = 6e-8 if dt == HF else 1e-30
    for n, g in (("dq", dq), ("dk", dk), ("dv", dv)):
        b, f = r[n + "_b"], r.get(n + "_f", 0)
        if dt == F32:
            t = 40 * eps * b + 64 * 2.0 ** -24 * f
        else:
            t = 0.5 * eps * (b + r[n].abs()) * 1.25 + 64 * 2.0 ** -24 * f
        if dt == HF:  # P and dS below fp16's normal range round to multiples of 2^-24
            t = t + 2.0 ** -25 * 4 * r[n].shape[1] * 4
        _within(g, r[n], t + sub, n)


def _inputs(B, Tq, Tk, Hq, Hk, D, dt, seed, big=1.0):
    g = torch.Generator().manual_seed(seed)
    mk = lambda *s: torch.randn(*s, generator=g).mul(big).to(dt).to(DEV)  # noqa: E731
    return mk(B, Tq, Hq, D), mk(B, Tk, Hk, D), mk(B, Tk, Hk, D), mk(B, Tq, Hq, D)


def _ints(x):
    return None if x is None else torch.tensor(x, dtype=torch.int32, device=DEV)


# B, Tq, Tk, Hq, Hk, D, type, causal, kv_len, q_start
CASES = [
    (1, 1, 1, 1, 1, 64, BF, False, None, None),
    (2, 32, 32, 2, 2, 64, BF, False, None, None),
    (1, 64, 64, 1, 1, 64, F32, False, None, None),
    (2, 256, 256, 4, 4, 64, F32, False, None, None),
    (1, 128, 128, 2, 2, 128, HF, False, None, None),
    (1, 130, 67, 2, 1, 128, BF, False, None, None),
    (2, 300, 300, 4, 2, 64, BF, True, None, None),
    (2, 257, 257, 4, 2, 128, HF, True, None, None),
    (3, 129, 129, 3, 3, 40, BF, True, [129, 0, 77], [0, 0, 0]),
    (2, 200, 200, 2, 1, 128, F32, True, None, None),
    (2, 200, 200, 2, 1, 32, F32, False, [1, 199], None),
    (2, 160, 33, 4, 1, 80, HF, True, None, None),          # more rows than keys: the first see nothing
    (2, 33, 160, 4, 4, 64, BF, True, [160, 40], [127, 20]),
    (3, 1, 515, 8, 2, 128, BF, True, [515, 0, 64], [514, -1, 63]),
    (2, 3, 700, 4, 1, 64, HF, True, [700, 350], [697, 347]),
    (1, 5, 1030, 2, 2, 128, F32, True, None, None),
    (1, 40, 2048, 2, 1, 64, BF, False, None, None),        # more than one tile of rows against split keys
    (5, 1, 300, 1, 1, 64, F32, False, [0, 1, 63, 64, 65], None),
    (1, 512, 512, 1, 1, 8, BF, True, None, None),
    (1, 70, 70, 2, 2, 4, F32, True, None, [5]),            # q_start past the keys' own offset
    (2, 96, 96, 2, 2, 64, BF, True, None, [-50, -200]),    # some rows, then every row, before the first key
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c[:8]))
def test_forward_and_backward(case):
    from ifd.attention import attention, attention_bwd
    B, Tq, Tk, Hq, Hk, D, dt, causal, kv_len, q_start = case
    q, k, v, dout = _inputs(B, Tq, Tk, Hq, Hk, D, dt, seed=Tq * 7 + Tk + D)
    keep = _visible(B, Tq, Tk, causal, kv_len, q_start)
    kw = dict(causal=causal, kv_len=_ints(kv_len), q_start=_ints(q_start))
    scale = 1 / math.sqrt(D)
    print(case, flush=True)
    out, lse = attention(q, k, v, **kw)
    torch.cuda.synchronize()
    _check_fwd(out, lse, _ref(q, k, v, keep, scale), dt)
    print("backward", flush=True)
    dq, dk, dv = attention_bwd(dout, q, k, v, out, lse, **kw)
    torch.cuda.synchronize()
    _check_bwd(dq, dk, dv, _ref(q, k, v, keep, scale, dout, out), dt)


def _same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def _both(q, k, v, dout, **kw):
    from ifd.attention import attention, attention_bwd
    out, lse = attention(q, k, v, **kw)
    return (out, lse) + attention_bwd(dout, q, k, v, out, lse, **kw)


@pytest.mark.parametrize("D,dt", [(64, BF), (80, HF), (128, F32)])
def test_strided_tensors_give_the_same_bits(D, dt):
    """Slices of a packed projection, a longer cache, a [B, H, T, D] layout, a broadcast batch, and tensors that the kernels
    cannot read in place (odd alignment, channels apart: copied) against contiguous copies."""
    from ifd.attention import attention, attention_bwd
    B, T, Hq, Hk = 3, 70, 4, 2
    g = torch.Generator().manual_seed(D)
    mk = lambda *s: torch.randn(*s, generator=g).to(dt).to(DEV)  # noqa: E731
    qkv = mk(B, T, Hq + 2 * Hk, D)
    q, k, v = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hk], qkv[:, :, Hq + Hk:]
    dout = mk(B, Hq, T, D).transpose(1, 2)
    want = _both(q.contiguous(), k.contiguous(), v.contiguous(), dout.contiguous(), causal=True)
    assert _same(_both(q, k, v, dout, causal=True), want)
    cache = mk(B, 2 * T, Hk, D)
    cache[:, 5:5 + T] = k
    assert _same(_both(q, cache[:, 5:5 + T], v, dout, causal=True), want)
    odd = torch.zeros(B, T, Hq, D + 3, dtype=dt, device=DEV)
    odd[..., 1:D + 1] = q
    apart = torch.zeros(B, T, Hk, 2 * D, dtype=dt, device=DEV)
    apart[..., ::2] = v
    assert _same(_both(odd[..., 1:D + 1], k, apart[..., ::2], dout, causal=True), want)
    # outputs into slices of the caller's buffers; what lies between them stays as it was
    d3 = torch.full((B, T, Hq + 2 * Hk + 1, D), 7.0, dtype=dt, device=DEV)
    dq, dk, dv = d3[:, :, :Hq], d3[:, :, Hq:Hq + Hk], d3[:, :, Hq + Hk:Hq + 2 * Hk]
    r = attention_bwd(dout, q, k, v, want[0], want[1], causal=True, dq=dq, dk=dk, dv=dv)
    assert r[0] is dq and _same((dq, dk, dv), want[2:]) and (d3[:, :, -1] == 7.0).all()
    o3 = torch.full((B, T, Hq + 1, D), 7.0, dtype=dt, device=DEV)
    attention(q, k, v, causal=True, out=o3[:, :, 1:])
    assert torch.equal(o3[:, :, 1:], want[0]) and (o3[:, :, 0] == 7.0).all()
    one = q[:1].expand(B, -1, -1, -1)
    assert _same(_both(one, k, v, dout, causal=True), _both(one.contiguous(), k, v, dout, causal=True))


@pytest.mark.parametrize("Tq,dt", [(1, BF), (150, HF), (150, F32), (300, BF)])
def test_anything_behind_the_last_key(Tq, dt):
    """NaN, infinities and the type's extremes past kv_len (a cache's unused end) change nothing, in the gradients either."""
    B, Tk, Hq, Hk, D = 2, 300, 4, 2, 64
    q, k, v, dout = _inputs(B, Tq, Tk, Hq, Hk, D, dt, seed=Tq)
    n = [131, 64]
    kw = dict(causal=Tq > 1, kv_len=_ints(n), q_start=_ints([x - Tq for x in n]))
    want = _both(q, k, v, dout, **kw)
    big = torch.finfo(dt).max
    for junk in (float("nan"), float("inf"), -float("inf"), big, -big):
        k2, v2 = k.clone(), v.clone()
        for b in range(B):
            k2[b, n[b]:], v2[b, n[b]:] = junk, junk
        got = _both(q, k2, v2, dout, **kw)
        assert _same(got, want), junk
        assert all((g[b, n[b]:] == 0).all() for g in got[3:] for b in range(B))


def test_large_scores_and_a_reference_point_that_moves():
    """Scores that rise along the keys by far more than the running softmax lets its reference point lag behind, and ones so
    low that no probability may underflow before the row's own maximum is found."""
    B, T, H, D = 1, 512, 2, 64
    for dt in (BF, HF, F32):
        q, k, v, dout = _inputs(B, T, T, H, H, D, dt, seed=3)
        q = q.abs() + 0.5
        ramp = torch.linspace(-6, 6, T, device=DEV).view(1, T, 1, 1)
        for k2 in ((k * 0.1 + ramp).to(dt), (k * 0.1 - 2 * ramp).to(dt), (k * 0.1 - 12).to(dt)):
            for causal in (False, True):
                got = _both(q, k2, v, dout, causal=causal)
                torch.cuda.synchronize()
                r = _ref(q, k2, v, _visible(B, T, T, causal, None, None), D ** -0.5, dout, got[0])
                # scores reach +-300: their own fp32 rounding moves p by |s| 2^-23, which the small-score bounds leave out
                s = 1 + 320 * 2.0 ** -23 * 2 / (40 * torch.finfo(F32).eps) if dt == F32 else 1.02
                for n in ("out_b", "dq_b", "dk_b", "dv_b", "dq_f", "dk_f"):
                    r[n] = r[n] * s
                _check_fwd(got[0], got[1], r, dt)
                _check_bwd(*got[2:], r, dt)


def test_not_finite_values_in_seen_places():
    """An infinity or NaN that a row sees reaches that row's result, and only rows that see it."""
    from ifd.attention import attention
    q, k, v, _ = _inputs(1, 200, 200, 1, 1, 64, BF, seed=1)
    k2 = k.clone()
    k2[0, 100, 0, 5] = float("nan")
    out, lse = attention(q, k2, v, causal=True)
    o0, l0 = attention(q, k, v, causal=True)
    assert torch.equal(out[:, :100], o0[:, :100]) and torch.equal(lse[..., :100], l0[..., :100])
    assert torch.isnan(out[:, 100:]).all() and torch.isnan(lse[..., 100:]).all()


def test_repeats_streams_and_concurrent_calls():
    q, k, v, dout = _inputs(2, 400, 400, 4, 2, 128, BF, seed=9)
    t = _inputs(4, 2, 3000, 8, 2, 64, HF, seed=10)
    kw = dict(causal=True)
    want, want2 = _both(q, k, v, dout, **kw), _both(*t, **kw)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(s1):
            a = _both(q, k, v, dout, **kw)
        with torch.cuda.stream(s2):
            b = _both(*t, **kw)
        torch.cuda.synchronize()
        assert _same(a, want) and _same(b, want2)


def test_captured_and_replayed():
    """Forward (split over the keys) and backward in one graph; replays follow the inputs, lengths among them."""
    from ifd.attention import attention, attention_bwd
    q, k, v, dout = _inputs(2, 2, 2048, 4, 2, 64, BF, seed=2)
    n, s = _ints([2048, 700]), _ints([2046, 698])
    kw = dict(causal=True, kv_len=n, q_start=s)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(2):
            _both(q, k, v, dout, **kw)
    torch.cuda.synchronize()
    gr, gr2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out, lse = attention(q, k, v, **kw)
    with torch.cuda.graph(gr2):
        grads = attention_bwd(dout, q, k, v, out, lse, **kw)
    g = torch.Generator().manual_seed(8)
    for it in range(4):
        for x in (q, k, v, dout):
            x.copy_(torch.randn(x.shape, generator=g).to(x.dtype))
        n.copy_(torch.tensor([2048 - 500 * it, 33 + it], dtype=torch.int32))
        s.copy_(n - 2)
        gr.replay()
        gr2.replay()
        torch.cuda.synchronize()
        assert _same((out, lse) + grads, _both(q, k, v, dout, **kw)), it


@pytest.mark.parametrize("Tq", [1, 160])
def test_offsets_past_32_bits(Tq):
    """A cache whose tokens lie 4 MiB apart and whose sequences lie 5 GiB apart."""
    from ifd.attention import attention, attention_bwd
    B, Tk, H, D, dt = 2, 1200, 2, 64, BF
    step, far = 1 << 21, 5 << 29  # in elements
    buf = torch.empty(far + Tk * step, dtype=dt, device=DEV)
    big = buf.as_strided((B, Tk, H, D), (far, step, D, 1))
    q, k, v, dout = _inputs(B, Tq, Tk, H, H, D, dt, seed=4)
    big.copy_(k)
    out, lse = attention(q, big, big, causal=True)
    assert _same((out, lse), attention(q, k, k, causal=True))
    dk = buf.as_strided((B, Tk, H, D), (far, step, D, 1), storage_offset=D * H)
    r = attention_bwd(dout, q, big, big, out, lse, causal=True, dk=dk)
    assert _same(r, attention_bwd(dout, q, k, k, out, lse, causal=True))


def test_empty_tensors_and_lengths():
    from ifd.attention import attention, attention_bwd
    q, k, v, dout = _inputs(2, 5, 7, 2, 1, 64, BF, seed=0)
    out, lse = attention(q[:0], k[:0], v[:0])
    assert out.shape[0] == 0 and lse.shape[0] == 0
    out, lse = attention(q[:, :0], k, v)
    dq, dk, dv = attention_bwd(dout[:, :0], q[:, :0], k, v, out, lse)
    torch.cuda.synchronize()
    assert out.shape[1] == 0 and (dk == 0).all() and (dv == 0).all()
    out, lse = attention(q, k[:, :0], v[:, :0], causal=True)
    dq, dk, dv = attention_bwd(dout, q, k[:, :0], v[:, :0], out, lse, causal=True)
    torch.cuda.synchronize()
    assert (out == 0).all() and torch.isneginf(lse).all() and (dq == 0).all() and dk.shape[1] == 0
    for n in ([-3, 0], [99, 1 << 30]):  # lengths out of range are clamped
        want = [min(max(x, 0), 7) for x in n]
        assert _same(_both(q, k, v, dout, kv_len=_ints(n)), _both(q, k, v, dout, kv_len=_ints(want)))


def test_gradients_against_differences():
    """The backward's values are the derivative of the forward, in fp32: directional differences of sum(out * dout)."""
    from ifd.attention import attention, attention_bwd
    B, Tq, Tk, Hq, Hk, D = 2, 37, 53, 4, 2, 32
    q, k, v, dout = _inputs(B, Tq, Tk, Hq, Hk, D, F32, seed=6)
    kw = dict(causal=True, kv_len=_ints([53, 20]), q_start=_ints([16, -4]))
    out, lse = attention(q, k, v, **kw)
    grads = attention_bwd(dout, q, k, v, out, lse, **kw)
    g = torch.Generator().manual_seed(7)
    for i, gr in enumerate(grads):
        e = torch.randn(gr.shape, generator=g).to(DEV)
        e = e / e.norm() * gr.norm() ** 0  # unit direction
        h = 0.05

        def f(s):
            t = [q, k, v]
            t[i] = t[i] + s * e
            return float((attention(*t, **kw)[0].double() * dout.double()).sum())
        diff = (8 * (f(h) - f(-h)) - (f(2 * h) - f(-2 * h))) / (12 * h)
        want = float((gr.double() * e.double()).sum())
        # fourth-order difference; fp32 outputs of norm |out| carry 2^-24 each, over h: 2^-24 * |dout| |out| / h * 2
        tol = 2e-4 * float(gr.norm()) + 2 * 2.0 ** -24 * float(dout.norm() * out.norm()) / h
        assert abs(diff - want) <= tol, (i, diff, want)


def test_norm_rotation_attention_and_optimizer_together():
    """A layer's step as it is used: packed projection -> norm and rotation -> attention -> its backward -> norm and rotation
    backward -> AdamW on the norm weights and the projection's values, against fp64 autograd. fp32: every stage is within
    40 eps of its magnitudes, together below 2e-5 of each gradient's norm."""
    from ifd.attention import attention, attention_bwd
    from ifd.optim import AdamW
    from ifd.rotary import Rotary, qk_norm_rope, qk_norm_rope_bwd
    B, T, Hq, Hk, D = 2, 200, 4, 2, 64
    g = torch.Generator().manual_seed(12)
    qkv = torch.randn(B, T, Hq + 2 * Hk, D, generator=g)
    w = [1 + 0.2 * torch.randn(D, generator=g) for _ in range(2)]
    dout = torch.randn(B, T, Hq, D, generator=g)
    pos, lens = torch.arange(T), [200, 150]
    rope = Rotary(D, scaling=("bands", 2.0, 128), device=DEV)
    params = [t.to(DEV) for t in (qkv, *w)]
    x, wq, wk = params
    q, k, v = x[:, :, :Hq], x[:, :, Hq:Hq + Hk], x[:, :, Hq + Hk:]
    q2, k2 = qk_norm_rope(q, k, wq, wk, pos.to(DEV), rope)
    kw = dict(causal=True, kv_len=_ints(lens), q_start=_ints([0, 0]))
    out, lse = attention(q2, k2, v, **kw)
    dx = torch.empty_like(x)
    dq2, dk2, _ = attention_bwd(dout.to(DEV), q2, k2, v, out, lse, dv=dx[:, :, Hq + Hk:], **kw)
    _, _, dwq, dwk = qk_norm_rope_bwd(dq2, dk2, q, k, wq, wk, pos.to(DEV), rope, dq=dx[:, :, :Hq], dk=dx[:, :, Hq:Hq + Hk])
    # fp64
    p64 = [t.double().requires_grad_() for t in (qkv, *w)]
    ang = pos.double()[:, None] * rope.inv_freq
    c, s = ang.cos()[:, None] * rope.mscale, ang.sin()[:, None] * rope.mscale

    def nr(t, wt):
        n = t / torch.sqrt(t.pow(2).mean(-1, keepdim=True) + 1e-6) * wt
        a, b = n[..., :D // 2], n[..., D // 2:]
        return torch.cat([a * c - b * s, b * c + a * s], -1)
    Q, K = nr(p64[0][:, :, :Hq], p64[1]), nr(p64[0][:, :, Hq:Hq + Hk], p64[2])
    rep = lambda t: t.repeat_interleave(Hq // Hk, 2).transpose(1, 2)  # noqa: E731
    sc = (Q.transpose(1, 2) @ rep(K).transpose(-1, -2)) / math.sqrt(D)
    sc = sc.masked_fill(~_visible(B, T, T, True, lens, [0, 0])[:, None], -math.inf)
    o64 = (torch.softmax(sc, -1) @ rep(p64[0][:, :, Hq + Hk:])).transpose(1, 2)
    refs = torch.autograd.grad(o64, p64, dout.double())
    rel = lambda a, b: float((a.cpu().double() - b).norm() / b.norm())  # noqa: E731
    assert rel(out, o64.detach()) <= 2e-5
    for a, b in zip((dx, dwq, dwk), refs):
        assert rel(a, b) <= 2e-5
    opt = AdamW(params, lr=1e-3, weight_decay=0.0, max_norm=1.0)
    before = [t.clone() for t in params]
    opt.step([dx, dwq, dwk])
    torch.cuda.synchronize()
    n = math.sqrt(sum(float((r ** 2).sum()) for r in refs))
    assert abs(float(opt.norm_coef[0]) - n) <= 2e-5 * n
    for p, b, r in zip(params, before, refs):  # the first step moves by lr g / (|g| + eps'): its sign where g is not small
        move, gn = (p - b).cpu().double(), r / n
        ok = gn.abs() > 1e-4
        assert ((move + 1e-3 * torch.sign(r))[ok].abs() <= 1e-3 * (1e-8 / 1e-4 + 1e-3) + 2.0 ** -23 * b.cpu().abs()[ok]).all()


def test_refusals_that_need_tensors_on_the_gpu():
    from ifd.attention import attention, attention_bwd
    from ifd.rotary import qk_norm_rope
    q, k, v, dout = _inputs(2, 8, 8, 2, 1, 64, BF, seed=0)
    for kw, msg in ((dict(kv_len=_ints([8])), "kv_len"), (dict(kv_len=_ints([8, 8]).long()), "kv_len"),
                    (dict(q_start=torch.zeros(2, dtype=torch.int32)), "q_start"), (dict(out=q), "overlaps"),
                    (dict(out=torch.empty(2, 8, 2, 64, device=DEV)), "like"),
                    (dict(out=torch.empty(2, 8, 2, 65, dtype=BF, device=DEV)[..., 1:]), "16-byte"),
                    (dict(out=torch.empty(1, 8, 2, 64, dtype=BF, device=DEV).expand(2, -1, -1, -1)), "share their place")):
        with pytest.raises(ValueError, match=msg):
            attention(q, k, v, **kw)
    with pytest.raises(ValueError, match="GPU tensor"):
        attention(q, k, v.cpu())
    out, lse = attention(q, k, v)
    for kw, msg in ((dict(dq=dout), "overlaps"), (dict(dk=k), "overlaps"), (dict(dv=torch.empty_like(q)), "like")):
        with pytest.raises(ValueError, match=msg):
            attention_bwd(dout, q, k, v, out, lse, **kw)
    with pytest.raises(ValueError, match="lse"):
        attention_bwd(dout, q, k, v, out, lse[:, :1])
    p = q.clone().requires_grad_()
    for call in (lambda: attention(p, k, v), lambda: attention_bwd(dout, p, k, v, out, lse), lambda: qk_norm_rope(p, k)):
        with pytest.raises(ValueError, match="records no gradients"):
            call()
        with torch.no_grad():
            call()
    # in-place outputs count as writes: autograd notices a saved tensor that has changed
    y = (q.clone().requires_grad_() * k[:, :, :1]).sum()
    kk = k.clone()
    w = torch.ones(64, device=DEV, dtype=BF, requires_grad=True)
    y = (w * kk).sum()
    with torch.no_grad():
        qk_norm_rope(q, kk, k_out=kk)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_norm_and_rotation_captured_and_replayed():
    from ifd.rotary import Rotary, qk_norm_rope, qk_norm_rope_bwd
    rope = Rotary(64, device=DEV)
    q, k, _, g = _inputs(4, 1, 1, 8, 2, 64, BF, seed=1)
    gk = torch.randn_like(k)
    w = torch.ones(64, device=DEV)
    pos = torch.zeros(4, 1, dtype=torch.int64, device=DEV)
    args = (w, w, pos, rope)
    with torch.cuda.stream(torch.cuda.Stream()):
        qk_norm_rope(q, k, *args), qk_norm_rope_bwd(g, gk, q, k, *args)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        a = qk_norm_rope(q, k, *args)
        b = qk_norm_rope_bwd(g, gk, q, k, *args)
    for it in range(3):
        for t in (q, k, g, gk, w):
            t.copy_(torch.randn(t.shape, device=DEV))
        pos.fill_(100 * it)
        gr.replay()
        torch.cuda.synchronize()
        assert _same(a, qk_norm_rope(q, k, *args)) and _same(b, qk_norm_rope_bwd(g, gk, q, k, *args))


@pytest.mark.parametrize("Tq,dt,D", [(1, BF, 64), (40, HF, 128), (200, F32, 64), (200, BF, 128), (333, BF, 96)])
def test_anything_behind_the_last_row_and_in_rows_without_keys(Tq, dt, D):
    """A cache's unused end without kv_len (causal, q_start tells where the rows are), and rows before the first key: what
    the keys that no row sees, and q and dout of the rows that see no key, hold changes nothing."""
    B, Tk, Hq, Hk = 3, 500, 4, 2
    q, k, v, dout = _inputs(B, Tq, Tk, Hq, Hk, D, dt, seed=Tq + 1)
    start = [100, 0, -Tq // 3 if Tq > 1 else -1]
    kw = dict(causal=True, q_start=_ints(start))
    want = _both(q, k, v, dout, **kw)
    r = _ref(q, k, v, _visible(B, Tq, Tk, True, None, start), D ** -0.5, dout, want[0])
    _check_fwd(want[0], want[1], r, dt)
    _check_bwd(*want[2:], r, dt)
    for junk in (float("nan"), float("inf"), -float("inf")):
        q2, k2, v2, d2 = q.clone(), k.clone(), v.clone(), dout.clone()
        for b, s in enumerate(start):
            k2[b, max(s + Tq, 0):], v2[b, max(s + Tq, 0):] = junk, junk
            q2[b, :max(-s, 0)], d2[b, :max(-s, 0)] = junk, junk
        assert _same(_both(q2, k2, v2, d2, **kw), want), junk


@pytest.mark.parametrize("case", [(1, 2500, 130, 4, 1, 64, BF, True, None, None), (1, 2500, 130, 4, 1, 128, HF, False, [97], None),
                                  (1, 2500, 66, 4, 1, 80, F32, True, None, [-7]), (40, 64, 64, 16, 16, 40, HF, True, None, None),
                                  (24, 200, 130, 8, 8, 128, BF, False, None, None), (1, 1, 4000, 4, 4, 64, F32, False, None, None),
                                  (1, 4000, 1, 2, 1, 96, BF, False, None, None), (2, 130, 130, 4, 1, 64, F32, False, None, None)],
                         ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c[:8]))
def test_backward_as_two_launches_and_as_one(case):
    """Long shares and many workgroups (row pass and key pass one after the other), and short calls around them (both in one
    launch)."""
    test_forward_and_backward(case)


@pytest.mark.parametrize("case", [(1, 150, 1100, 2, 1, 64, BF, False, None, None), (1, 150, 700, 2, 2, 128, F32, True, None, None),
                                  (2, 140, 1500, 4, 2, 80, HF, True, [1499, 600], [1300, 500]),
                                  (3, 200, 1100, 2, 1, 96, F32, True, [0, 1100, 70], [-150, 900, 0]),
                                  (1, 129, 2100, 1, 1, 128, BF, True, None, [-100]), (1, 40, 1700, 3, 1, 72, HF, False, None, None),
                                  (2, 16, 1000, 8, 1, 128, BF, True, [999, 3], [980, 0]), (1, 33, 300, 4, 1, 64, F32, True, None, None)],
                         ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c[:8]))
def test_rows_whose_keys_are_shared_out(case):
    """Enough rows for the many-row kernel and enough keys to split them, with ragged lengths and rows without keys."""
    test_forward_and_backward(case)


@pytest.mark.parametrize("case", [(2, 70, 90, 2, 1, 8, BF, True, None, None), (1, 200, 70, 2, 2, 4, F32, False, None, None),
                                  (1, 150, 1100, 1, 1, 8, HF, False, None, None), (2, 5, 700, 4, 2, 4, F32, True, [700, 9], None),
                                  (1, 90, 100, 2, 1, 104, BF, True, None, None), (1, 90, 100, 2, 1, 120, HF, False, None, None),
                                  (1, 90, 100, 2, 1, 100, F32, True, None, None), (1, 3, 600, 2, 2, 88, BF, False, [599], None)],
                         ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c[:8]))
def test_narrow_and_odd_heads(case):
    test_forward_and_backward(case)


@pytest.mark.parametrize("case", [(1, 300, 1000, 2, 1, 64, F32, True, [900], [600]), (2, 129, 700, 3, 1, 80, HF, False, [700, 0], None),
                                  (1, 77, 3000, 2, 2, 128, BF, True, None, [-20]), (1, 1, 900, 1, 1, 96, F32, False, None, None),
                                  (1, 2500, 640, 4, 1, 64, BF, False, [635], None), (3, 33, 513, 1, 1, 128, F32, True, [513, 40, 512], None)],
                         ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c[:8]))
def test_backward_whose_rows_keys_are_shared_out(case):
    """Few rows and many keys: the row pass in shares, joined beside the key pass'; in one launch and in two."""
    test_forward_and_backward(case)
