"""Calls of the attention-layer operators that their documentation allows, beside the usual ones: inference mode, heads off
their alignment, expanded gradients, positions at the ends of int32, tens of thousands of short sequences, very large scores.

Tolerances. Attention: as in test_gpu_attention.py, P and the result rounded once to the type, finfo.eps / 2 each of
sum_j p_j |v_j| and of |out|, times 1.25 for the fp32 beneath; fp32 40 eps of the sum. Norm and rotation: as in
test_gpu_qk_rope.py, half a step of the type and 32 * 2^-24 of the magnitudes that meet in an output; dw 128 * 2^-24 of the
terms' sum.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24


def _rand(gen, *shape, dt=F32):
    return torch.randn(*shape, generator=gen).to(dt).to(DEV)


def _ref(q, k, v, keep=None, scale=None):
    """(out, lse, sum_j p_j |v_j|) in fp64 on the CPU"""
    q, k, v = (t.detach().cpu().double().transpose(1, 2) for t in (q, k, v))
    G = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    s = (q @ k.transpose(-1, -2)) * (q.shape[-1] ** -0.5 if scale is None else scale)
    if keep is not None:
        s = s.masked_fill(~keep[:, None], -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - torch.where(torch.isinf(lse), 0.0, lse)[..., None])
    return (p @ v).transpose(1, 2), lse, (p @ v.abs()).transpose(1, 2)


def _near(out, lse, ref, dt):
    r, l, b = ref
    eps = torch.finfo(dt).eps
    tol = 40 * eps * b if dt == F32 else 0.625 * eps * (b + r.abs()) + (6e-8 if dt == HF else 0)
    assert ((out.cpu().double() - r).abs() <= tol + 1e-30).all()
    fin = torch.isfinite(l)
    assert torch.equal(torch.isneginf(lse.cpu()), ~fin)
    assert ((lse.cpu().double() - l).abs()[fin] <= 1e-5 * (1 + l.abs()[fin])).all()


@pytest.mark.parametrize("mode", [torch.inference_mode, torch.no_grad])
def test_tokens_written_into_a_cache(mode):
    """Step after step as serving does it, the key's rotation written into the cache, all of it made in inference mode."""
    from ifd.attention import attention
    from ifd.rotary import Rotary, qk_norm_rope
    gen = torch.Generator().manual_seed(1)
    with mode():
        B, L, Hq, Hk, D = 3, 70, 4, 2, 64
        rope = Rotary(D, device=DEV)
        kc, vc = (torch.full((B, L, Hk, D), float("nan"), dtype=BF, device=DEV) for _ in range(2))
        w = (1 + 0.2 * torch.randn(D, generator=gen)).to(DEV)
        for t in range(40):
            qkv = _rand(gen, B, 1, Hq + 2 * Hk, D, dt=BF)
            q, k, v = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hk], qkv[:, :, Hq + Hk:]
            pos = torch.full((B, 1), t, device=DEV)
            q2, k2 = qk_norm_rope(q, k, w, w, pos, rope, k_out=kc[:, t:t + 1])
            assert k2.data_ptr() == kc[:, t].data_ptr()
            vc[:, t:t + 1] = v
            out, lse = attention(q2, kc, vc, causal=True, q_start=torch.full((B,), t, dtype=torch.int32, device=DEV))
            if t in (0, 1, 31, 32, 39):
                _near(out, lse, _ref(q2, kc[:, :t + 1], vc[:, :t + 1]), BF)
        assert torch.isnan(kc[:, 40:]).all()


def test_expanded_gradients_and_rows():
    """dout as a sum's backward hands it out (one value, or one row, for all), and a key shared by all positions."""
    from ifd.attention import attention, attention_bwd
    gen = torch.Generator().manual_seed(2)
    q, k, v = _rand(gen, 2, 300, 4, 64), _rand(gen, 2, 300, 2, 64), _rand(gen, 2, 300, 2, 64)
    k1 = k[:, :1].expand(-1, 300, -1, -1)
    out, lse = attention(q, k1, v, causal=True)
    o2, l2 = attention(q, k1.contiguous(), v, causal=True)
    assert torch.equal(out, o2) and torch.equal(lse, l2)
    for d in (torch.ones((), device=DEV).expand_as(q), _rand(gen, 1, 1, 1, 64).expand_as(q)):
        a = attention_bwd(d, q, k1, v, out, lse, causal=True)
        b = attention_bwd(d.contiguous(), q, k1.contiguous(), v, out, lse, causal=True)
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("start", [(2 ** 31 - 1, -2 ** 31), (-1, 0), (-300, -299), (299, 2 ** 31 - 300)])
def test_positions_at_the_ends_of_int32(start):
    from ifd.attention import attention, attention_bwd
    gen = torch.Generator().manual_seed(3)
    T = 300
    q, k, v, d = (_rand(gen, 2, T, h, 64) for h in (4, 2, 2, 4))
    keep = torch.arange(T)[None, None] <= (torch.tensor(start)[:, None] + torch.arange(T))[:, :, None]
    st = torch.tensor(start, dtype=torch.int32, device=DEV)
    out, lse = attention(q, k, v, causal=True, q_start=st)
    _near(out, lse, _ref(q, k, v, keep), F32)
    dq, dk, dv = attention_bwd(d, q, k, v, out, lse, causal=True, q_start=st)
    torch.cuda.synchronize()
    none = ~keep.any(2)
    unseen = ~keep.any(1)
    assert (dq.cpu()[none] == 0).all() and (dk.cpu()[unseen] == 0).all() and (dv.cpu()[unseen] == 0).all()
    assert all(torch.isfinite(t).all() for t in (dq, dk, dv))


@pytest.mark.parametrize("B,Tq,Tk,Hq,Hk,D", [(70000, 1, 3, 1, 1, 32), (66000, 33, 2, 1, 1, 8), (5000, 3, 40, 4, 2, 64)])
def test_many_short_sequences(B, Tq, Tk, Hq, Hk, D):
    """More sequences than 16 bits count."""
    from ifd.attention import attention, attention_bwd
    gen = torch.Generator().manual_seed(4)
    q, k, v, d = _rand(gen, B, Tq, Hq, D, dt=HF), _rand(gen, B, Tk, Hk, D, dt=HF), _rand(gen, B, Tk, Hk, D, dt=HF), \
        _rand(gen, B, Tq, Hq, D, dt=HF)
    print(B, Tq, Tk, flush=True)
    out, lse = attention(q, k, v)
    g = attention_bwd(d, q, k, v, out, lse)
    torch.cuda.synchronize()
    at = [0, 1, 7, 4999 if B < 60000 else 65535, B - 1]  # the reference of a few, the others against a call of their own
    _near(out[at], lse[at], _ref(q[at], k[at], v[at]), HF)
    half = B // 2 + 1
    o2, l2 = attention(q[half:], k[half:], v[half:])
    assert torch.equal(o2, out[half:]) and torch.equal(l2, lse[half:])
    g2 = attention_bwd(d[half:], q[half:], k[half:], v[half:], o2, l2)
    for x, y in zip(g, g2):  # (the number of shares may differ, and with it the last bit of fp32 sums before rounding)
        x, y = x[half:].float(), y.float()
        assert ((x - y).abs() <= torch.finfo(HF).eps * x.abs() + 6e-8 * 8).all()


@pytest.mark.parametrize("dt,big", [(BF, 2.0 ** 11), (HF, 2.0 ** 11), (F32, 2.0 ** 11)])
def test_scores_up_to_1e8(dt, big):
    """Products of powers of two and eight bits, so that every score is exact: up to 2^26, rising and falling along the keys.
    The largest leads by more than any exponent reaches, so that the row is its key's value. The exponent's reference point
    in units of log2 is off by up to 2^26 log2(e) 2^-24, so p is not 1 but some power of two near it: rounded once to the
    type, as the result is; lse: the constant, its product, the sum and the product back, 2^-24 each."""
    from ifd.attention import attention
    T, D = 500, 32
    gen = torch.Generator().manual_seed(5)
    v = _rand(gen, 1, T, 1, D, dt=dt)
    q = torch.zeros(1, 160, 1, D)
    q[..., 0] = big
    perm = torch.randperm(T, generator=gen)
    k = torch.zeros(1, T, 1, D)
    k[..., 0] = ((perm - T // 2).float() * 2.0 ** 7).view(1, T, 1)  # steps of 2^7: 8 bits of (perm - 250)
    q, k = q.to(dt).to(DEV), k.to(dt).to(DEV)
    s = float(k.float().abs().max()) * big
    assert 2.0 ** 25 < s < 2.0 ** 27
    for Tq in (160, 1):
        out, lse = attention(q[:, :Tq], k, v, scale=1.0)
        top = int(k[0, :, 0, 0].float().argmax())
        want, eps = v[:, top:top + 1].cpu().double(), torch.finfo(dt).eps
        tol = (40 * eps if dt == F32 else 1.25 * eps) * want.abs()
        assert ((out.cpu().double() - want).abs() <= tol).all()
        best = float(k[0, top, 0, 0]) * big
        assert ((lse.double() - best).abs() <= 4 * U * best).all()


@pytest.mark.parametrize("dt,D,off", [(BF, 128, 1), (HF, 64, 3), (F32, 128, 1), (BF, 40, 2)])
def test_heads_off_their_alignment_forward_and_backward(dt, D, off):
    """Queries, keys and their gradients whose heads start `off` elements into their rows, against fp64 and against aligned
    copies: the narrow loads sum the norm in another order, so that both results lie within the tolerance, not one on the
    other."""
    from ifd.rotary import Rotary, qk_norm_rope, qk_norm_rope_bwd
    gen = torch.Generator().manual_seed(D + off)
    B, T, Hq, Hk, eps = 2, 7, 4, 2, 1e-6
    rope = Rotary(D, device=DEV)

    def odd(H):
        return _rand(gen, B, T, H, D + 8, dt=dt)[..., off:off + D]
    q, k, gq, gk = odd(Hq), odd(Hk), odd(Hq), odd(Hk)
    wq, wk = ((1 + 0.3 * torch.randn(D, generator=gen)).to(DEV) for _ in range(2))
    pos = (torch.arange(T) + 1000).to(DEV)
    ang = pos.cpu().double()[:, None] * rope.inv_freq
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    h = D // 2
    turn = lambda x, sg: torch.cat([x[..., :h] * c - sg * x[..., h:] * s, x[..., h:] * c + sg * x[..., :h] * s], -1)  # noqa: E731
    mag = lambda x: (x[..., :h].abs() + x[..., h:].abs()).repeat(1, 1, 1, 2)  # noqa: E731
    same = lambda a, r, m: ((a.cpu().double() - r).abs()  # noqa: E731
                            <= torch.finfo(dt).eps / 2 * r.abs() + 32 * U * m + (3e-8 if dt == HF else 0)).all()
    got = [qk_norm_rope(q, k, wq, wk, pos, rope, eps=eps) + qk_norm_rope_bwd(gq, gk, q, k, wq, wk, pos, rope, eps=eps),
           qk_norm_rope(q.contiguous(), k.contiguous(), wq, wk, pos, rope, eps=eps)
           + qk_norm_rope_bwd(gq.contiguous(), gk.contiguous(), q.contiguous(), k.contiguous(), wq, wk, pos, rope, eps=eps)]
    torch.cuda.synchronize()
    for i, (x, w, g) in enumerate(((q, wq, gq), (k, wk, gk))):
        x, w, g = x.cpu().double(), w.cpu().double(), g.cpu().double()
        r = 1 / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps)
        dn, u = turn(g, -1), turn(g, -1) * w
        um, xh = mag(g) * w.abs(), x * r
        dx = r * (u - xh * (u * xh).mean(-1, keepdim=True))
        dm = r * (um + xh.abs() * (um * xh.abs()).mean(-1, keepdim=True))
        for y in got:
            assert same(y[i], turn(xh * w, 1), mag(xh * w))
            assert same(y[2 + i], dx, dm)
            rw, mw = (dn * xh).sum((0, 1, 2)), (mag(g) * xh.abs()).sum((0, 1, 2))
            assert ((y[4 + i].cpu().double() - rw).abs() <= 128 * U * mw + U * rw.abs()).all()


def test_infinite_gradient_without_the_clip_spoils_its_block_alone():
    from ifd.optim import AdamW
    gen = torch.Generator().manual_seed(6)
    for bad in (math.inf, -math.inf):
        p = _rand(gen, 600)
        opt = AdamW([p], lr=1e-3, state_bits=8)
        for i in range(3):
            g = _rand(gen, 600)
            if i == 1:
                g[300] = bad
            opt.step([g])
            m, v = (~torch.isfinite(t) for t in opt.moments())
            want = torch.zeros(768, dtype=torch.bool, device=DEV)
            want[256:512] = i > 0
            assert torch.equal(m, want) and torch.equal(v, want)
            bad_p = ~torch.isfinite(p)
            assert bad_p.sum() == (0, 1, 256)[i] and not bad_p[:256].any() and not bad_p[512:].any()
