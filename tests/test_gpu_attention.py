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
