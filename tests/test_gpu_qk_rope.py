"""The per-head norm with the position rotation and its backward (ifd.rotary, csrc/qk_rope.hip) against fp64.

Tolerances: each output is rounded once to its type (half a step, finfo.eps / 2 relative) after fp32 arithmetic: the norm's
sum (D <= 128 terms), rsqrt, two products and the rotation, whose reduced angle carries 2^-25 of a turn: together below
32 * 2^-24 of the magnitudes that meet in an output. dw: fp32 partial sums of at most 128 terms in a chain: 128 * 2^-24 of
sum |dn xhat|.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24


def _turn(x, pos, rope, sign):
    if rope is None:
        return x, x.abs()
    r, h = rope.rot, rope.rot // 2
    ang = sign * pos.double().cpu()[..., None] * rope.inv_freq
    c, s = ang.cos()[:, :, None] * rope.mscale, ang.sin()[:, :, None] * rope.mscale
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if rope.interleaved else (x[..., :h], x[..., h:r])
    ya, yb, m = a * c - b * s, b * c + a * s, (a.abs() + b.abs()) * rope.mscale
    j = (lambda u, v: torch.stack([u, v], -1).flatten(-2)) if rope.interleaved else (lambda u, v: torch.cat([u, v], -1))
    return torch.cat([j(ya, yb), x[..., r:]], -1), torch.cat([j(m, m), x[..., r:].abs()], -1)


def _ref(x, w, pos, rope, eps, norm, g=None):
    x = x.detach().cpu().double()
    w = torch.ones(x.shape[-1], dtype=torch.float64) if w is None else w.detach().cpu().double()
    rstd = 1 / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps) if norm else torch.ones(())
    n = x * rstd * w if norm else x
    y, ym = _turn(n, pos, rope, 1)
    if g is None:
        return y, ym
    dn, dm = _turn(g.detach().cpu().double(), pos, rope, -1)
    if not norm:
        return dn, dm, None, None
    xh = x * rstd
    u, um = dn * w, dm * w.abs()
    dx = rstd * (u - xh * (u * xh).mean(-1, keepdim=True))
    dxm = rstd * (um + xh.abs() * (um * xh.abs()).mean(-1, keepdim=True))
    return dx, dxm, (dn * xh).sum((0, 1, 2)), (dm * xh.abs()).sum((0, 1, 2))


def _near(got, ref, mag, dt, name):
    tol = torch.finfo(dt).eps / 2 * ref.abs() + 32 * U * mag + (3e-8 if dt == HF else 0)
    bad = (got.detach().cpu().double() - ref).abs() - tol
    assert (bad <= 0).all(), f"{name}: past its tolerance by {bad.max():.3e}"


# B, T, Hq, Hk, D, rot, type, interleaved, scaling, first position
CASES = [
    (1, 1, 1, 1, 64, 64, BF, False, None, 0),
    (2, 5, 4, 2, 128, 128, BF, False, ("linear", 4.0), 999_000),
    (2, 17, 3, 1, 128, 64, HF, True, ("bands", 4.0, 4096), 0),
    (1, 33, 8, 8, 64, 32, F32, True, None, 123_456_789),
    (3, 7, 5, 1, 40, 40, BF, False, ("base", 8.0), 77),
    (2, 9, 2, 2, 80, 40, HF, False, None, 0),
    (1, 3, 2, 1, 6, 2, F32, True, None, 5),
    (1, 4, 1, 1, 2, 2, BF, False, None, 5),
    (4, 130, 16, 4, 128, 128, BF, True, None, 0),
    (1, 2, 70, 3, 96, 96, F32, False, ("linear", 1.0), 0),
    (2, 3, 1, 1, 10, 4, HF, True, None, -7),      # positions before the origin
]


def _data(case, seed=0, bits=None):
    B, T, Hq, Hk, D, rot, dt, il, sc, first = case
    g = torch.Generator().manual_seed(seed + D * 3 + T)
    mk = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    from ifd.rotary import Rotary
    rope = Rotary(rot, interleaved=il, scaling=sc, device=DEV)
    qkv = mk(B, T, Hq + 2 * Hk, D).to(dt).to(DEV)
    q, k = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hk]
    wq, wk = (1 + 0.3 * mk(D)).to(DEV), (1 + 0.3 * mk(D)).to(DEV)
    pos = (first + torch.arange(T) + torch.randint(0, 50, (B, 1), generator=g)).to(DEV)
    gq, gk = mk(B, T, Hq, D).to(dt).to(DEV), mk(B, T, Hk, D).to(dt).to(DEV)
    return q, k, wq, wk, pos, rope, gq, gk, dt


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c[:8]))
@pytest.mark.parametrize("norm", [True, False])
def test_forward_and_backward(case, norm):
    from ifd.rotary import qk_norm_rope, qk_norm_rope_bwd
    q, k, wq, wk, pos, rope, gq, gk, dt = _data(case)
    eps = 1e-5
    if not norm:
        wq = wk = None
    print(case, flush=True)
    yq, yk = qk_norm_rope(q, k, wq, wk, pos, rope, eps=eps, norm=norm)
    dq, dk, dwq, dwk = qk_norm_rope_bwd(gq, gk, q, k, wq, wk, pos, rope, eps=eps, norm=norm)
    torch.cuda.synchronize()
    for x, w, y, g, dx, dw in ((q, wq, yq, gq, dq, dwq), (k, wk, yk, gk, dk, dwk)):
        _near(y, *_ref(x, w, pos, rope, eps, norm), dt, "y")
        rx, mx, rw, mw = _ref(x, w, pos, rope, eps, norm, g)
        _near(dx, rx, mx, dt, "dx")
        if norm:
            assert ((dw.cpu().double() - rw).abs() <= 128 * U * mw + U * rw.abs()).all(), "dw"
        else:
            assert dw is None


def test_norm_only_rotation_only_queries_only_and_in_place():
    from ifd.rotary import qk_norm_rope, qk_norm_rope_bwd
    q, k, wq, wk, pos, rope, gq, gk, dt = _data(CASES[8])
    y, none = qk_norm_rope(q, None, wq, None, eps=1e-6)
    assert none is None
    _near(y, *_ref(q, wq, pos, None, 1e-6, True), dt, "norm only")
    y, yk = qk_norm_rope(q, k, None, None, pos[0], rope, norm=True, eps=0.0)  # shared positions, no weights
    p0 = pos[:1].expand(q.shape[0], -1)
    _near(y, *_ref(q, None, p0, rope, 0.0, True), dt, "shared positions")
    dq, dk, dwq, dwk = qk_norm_rope_bwd(gq, gk, q, k, wq, wk, pos, rope)
    g1, g2 = gq.clone(), gk.clone()
    e = qk_norm_rope_bwd(g1, g2, q, k, wq, wk, pos, rope, dq=g1, dk=g2)
    assert e[0] is g1 and torch.equal(g1, dq) and torch.equal(g2, dk) and torch.equal(e[2], dwq) and torch.equal(e[3], dwk)
    yq, yk = qk_norm_rope(q, k, wq, wk, pos, rope)
    buf = torch.cat([q, k, k], 2)
    a, b = buf[:, :, :q.shape[2]], buf[:, :, q.shape[2]:q.shape[2] + k.shape[2]]
    tail = buf[:, :, q.shape[2] + k.shape[2]:].clone()
    qk_norm_rope(a, b, wq, wk, pos, rope, q_out=a, k_out=b)
    assert torch.equal(a, yq) and torch.equal(b, yk) and torch.equal(buf[:, :, -k.shape[2]:], tail)


def test_unaligned_rows_and_zero_rows():
    """Heads that start at odd elements take the narrow path with the same bits; a zero row stays zero, also with eps 0 in
    its gradient's place only when eps > 0."""
    from ifd.rotary import qk_norm_rope, qk_norm_rope_bwd
    q, k, wq, wk, pos, rope, gq, gk, dt = _data(CASES[1])
    odd = torch.zeros(q.shape[0], q.shape[1], q.shape[2], q.shape[3] + 3, dtype=dt, device=DEV)
    odd[..., 1:-2] = q
    y, _ = qk_norm_rope(q, None, wq, None, pos, rope)
    z, _ = qk_norm_rope(odd[..., 1:-2], None, wq, None, pos, rope)
    _near(z, *_ref(q, wq, pos, rope, 1e-6, True), dt, "odd start")
    q0 = q.clone()
    q0[0, 0, 0] = 0
    y, _ = qk_norm_rope(q0, None, wq, None, pos, rope)
    assert (y[0, 0, 0] == 0).all() and torch.isfinite(y).all()
    dq, _, dwq, _ = qk_norm_rope_bwd(gq, None, q0, None, wq, None, pos, rope)
    assert torch.isfinite(dq.float()).all() and torch.isfinite(dwq).all()


def test_empty_and_repeatable():
    from ifd.rotary import qk_norm_rope, qk_norm_rope_bwd
    q, k, wq, wk, pos, rope, gq, gk, dt = _data(CASES[8])
    y, _ = qk_norm_rope(q[:0], k[:0], wq, wk, pos[:0], rope)
    assert y.shape[0] == 0
    r = qk_norm_rope_bwd(gq[:, :0], gk[:, :0], q[:, :0], k[:, :0], wq, wk, pos[:, :0], rope)
    torch.cuda.synchronize()
    assert (r[2] == 0).all() and (r[3] == 0).all()
    a = qk_norm_rope_bwd(gq, gk, q, k, wq, wk, pos, rope)
    b = qk_norm_rope_bwd(gq, gk, q, k, wq, wk, pos, rope)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_gradient_against_differences():
    """The fp64 formula above is itself the derivative of the forward formula."""
    case = (1, 2, 2, 1, 16, 8, F32, True, ("bands", 2.0, 64), 3)
    q, k, wq, wk, pos, rope, gq, gk, dt = _data(case)
    dx, _, dw, _ = _ref(q, wq, pos, rope, 1e-3, True, gq)
    g = gq.cpu().double()
    for t, d in ((q, dx), (wq, dw)):
        e = torch.randn(t.shape, generator=torch.Generator().manual_seed(1), dtype=torch.float64)
        f = lambda s: float((_ref(q.cpu().double() + (s * e if t is q else 0), wq.cpu().double() + (s * e if t is wq else 0),  # noqa: E731
                                  pos, rope, 1e-3, True)[0] * g).sum())
        diff = (f(1e-5) - f(-1e-5)) / 2e-5
        assert abs(diff - float((d * e).sum())) <= 1e-6 * float((d * e).abs().sum())
