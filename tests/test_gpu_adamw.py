"""AdamW over many tensors (ifd.optim, csrc/adamw.hip) against the formulas in fp64.

Tolerances. 32-bit states: m and v are three fp32 operations: 3 * 2^-24 of the terms' magnitudes. Parameters: one rounding to
their type (half a step) after fp32 arithmetic: decay and subtraction (2 * 2^-24 |p|) and the step's own relative error (m, v,
square root, two divisions, a sum: 12 * 2^-24 of its size; where the gradient's and the moment's terms cancel in m, of the
terms'). 8-bit states: the bytes and scales are decided in fp64 and must be equal.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24
LR, B1, B2, EPS, WD = 1e-3, 0.9, 0.999, 1e-8, 0.02


def _mix(x):
    x = x.astype(np.uint32)
    with np.errstate(over="ignore"):
        for mul, sh in ((0x9E3779B9, 15), (0x6A09E667, 13), (0xBB67AE85, 16)):
            x = x * np.uint32(mul)
            x = x ^ (x >> np.uint32(sh))
    return x


def _values(ebits):
    n, bias = 1 << (ebits + 3), (1 << ebits) - 1
    v = np.array([0.0] + [2.0 ** (c // 8 - bias) * (1 + c % 8 / 8) for c in range(1, n)])
    return np.concatenate([v, -v]) if ebits == 4 else v


def _round(x, r16, ebits):
    """Blocks [n, 256] -> (bytes, scales): up where the share of the gap plus the random number passes one."""
    tab = _values(ebits)[:1 << (ebits + 3)]
    s = (np.abs(x).max(1) / 1.875).astype(np.float32)
    s64 = s.astype(np.float64)[:, None]
    y = np.where(s64 > 0, np.abs(x) / np.where(s64 > 0, s64, 1), 0)
    lo = np.clip(np.searchsorted(tab, y, side="right") - 1, 0, len(tab) - 2)
    up = (y - tab[lo]) / (tab[lo + 1] - tab[lo]) * 65536 + r16 >= 65536
    if ebits == 5:
        up |= (lo == 0) & (y > 0)
    c = lo + up
    return (c + np.where((x < 0) & (c > 0), 128, 0) if ebits == 4 else c).astype(np.uint8), s


class Ref:
    """fp64 AdamW on host copies, states laid out in blocks of 256."""

    def __init__(self, params, bits, seed, groups=None):
        self.p = [p.detach().cpu().double().numpy().reshape(-1) for p in params]
        self.bits, self.seed, self.k = bits, seed, 0
        self.nb = [-(-len(p) // 256) for p in self.p]
        n = sum(self.nb)
        self.m, self.v = np.zeros((n, 256)), np.zeros((n, 256))
        self.hyper = groups or [(LR, WD)] * len(params)

    def step(self, grads, max_norm=None):
        self.k += 1
        gs = [None if g is None else g.detach().cpu().double().numpy().reshape(-1) for g in grads]
        coef = 1.0
        if max_norm is not None:
            coef = min(1.0, max_norm / (math.sqrt(sum(float((g * g).sum()) for g in gs if g is not None)) + 1e-6))
        at = 0
        key = _mix(_mix(np.array([self.seed])) + np.uint32(self.k))
        out = []
        for p, g, nb, (lr, wd) in zip(self.p, gs, self.nb, self.hyper):
            if g is not None and nb:
                gb = np.zeros((nb, 256))
                gb.reshape(-1)[:len(g)] = g * coef
                m = B1 * self.m[at:at + nb] + (1 - B1) * gb
                v = B2 * self.v[at:at + nb] + (1 - B2) * gb * gb
                self.m_mag = np.abs(B1 * self.m[at:at + nb]) + np.abs((1 - B1) * gb)
                c1, c2 = 1 - B1 ** self.k, 1 - B2 ** self.k
                den = np.sqrt(v.reshape(-1)[:len(p)] / c2) + EPS
                st = lr / c1 * m.reshape(-1)[:len(p)] / den
                mag = lr / c1 * self.m_mag.reshape(-1)[:len(p)] / den
                new = p * (1 - lr * wd) - st
                out.append((new, 2 * U * np.abs(p) + 12 * U * mag))
                if self.bits == 8:
                    idx = (np.arange(at * 256, (at + nb) * 256, dtype=np.uint64) + key.astype(np.uint64)).astype(np.uint32)
                    r = _mix(idx).reshape(nb, 256)
                    cm, sm = _round(m, (r & 0xFFFF).astype(np.float64), 4)
                    cv, sv = _round(v, (r >> 16).astype(np.float64), 5)
                    m = _values(4)[cm] * sm.astype(np.float64)[:, None]
                    v = _values(5)[cv] * sv.astype(np.float64)[:, None]
                self.m[at:at + nb], self.v[at:at + nb] = m, v
                p[:] = new
            else:
                out.append((p.copy(), np.zeros(len(p))))
            at += nb
        return out


def _check(opt, ref, params, out):
    for p, (new, tol) in zip(params, out):
        got = p.detach().cpu().double().numpy().reshape(-1)
        t = tol + torch.finfo(p.dtype).eps / 2 * np.abs(new) + (3e-8 if p.dtype == HF else 0)
        assert (np.abs(got - new) <= t).all(), float((np.abs(got - new) - t).max())
    m, v = (t.cpu().double().numpy().reshape(-1, 256) for t in opt.moments())
    if ref.bits == 8:
        assert np.array_equal(m.astype(np.float32), ref.m.astype(np.float32))
        assert np.array_equal(v.astype(np.float32), ref.v.astype(np.float32))
    else:
        s = np.abs(ref.m).max() + 1e-30
        assert (np.abs(m - ref.m) <= 16 * U * (np.abs(ref.m) + s * 0.2)).all()
        assert (np.abs(v - ref.v) <= 16 * U * np.abs(ref.v) + 1e-38).all()


def _sync(ref, params):
    """The next step starts from what the kernel stored (a rounded parameter)."""
    for i, p in enumerate(params):
        ref.p[i][:] = p.detach().cpu().double().numpy().reshape(-1)


SHAPES = [(1,), (255,), (256,), (257,), (33, 65), (1, 4099), (0,), (128, 9, 3, 3), (3, 5, 7)]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("pdt,gdt", [(F32, F32), (F32, BF), (BF, BF), (HF, F32), (BF, HF)],
                         ids=lambda x: str(x).replace("torch.", ""))
@pytest.mark.parametrize("max_norm", [None, 0.5])
def test_steps(bits, pdt, gdt, max_norm):
    from ifd.optim import AdamW
    g = torch.Generator().manual_seed(5)
    params = [(0.1 * torch.randn(*s, generator=g)).to(pdt).to(DEV) for s in SHAPES]
    opt = AdamW(params, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, state_bits=bits, max_norm=max_norm, seed=11)
    ref = Ref(params, bits, 11)
    for k in range(4):
        grads = [(torch.randn(*s, generator=g) * 10.0 ** (-2 + 0.5 * i)).to(gdt).to(DEV) for i, s in enumerate(SHAPES)]
        grads[2] = None if k == 1 else grads[2]  # one tensor without a gradient now and then
        if k == 2:
            grads[4].zero_()
        print(bits, pdt, gdt, max_norm, k, flush=True)
        opt.step(grads)
        torch.cuda.synchronize()
        out = ref.step(grads, max_norm)
        if max_norm is not None:
            n = math.sqrt(sum(float((x.double() ** 2).sum()) for x in grads if x is not None))
            assert abs(float(opt.norm_coef[0]) - n) <= 1e-12 * n
        _check(opt, ref, params, out)
        _sync(ref, params)
        if bits == 32:
            m, v = opt.moments()
            ref.m, ref.v = (t.cpu().double().numpy().reshape(-1, 256).copy() for t in (m, v))


def test_views_of_one_buffer_groups_and_many_tensors():
    """More tensors than one launch takes, at odd addresses, in two groups with rates of their own."""
    from ifd.optim import AdamW
    g = torch.Generator().manual_seed(3)
    n = [1 + 37 * i % 613 for i in range(230)]
    buf, gbuf = torch.randn(sum(n) + 64, generator=g).to(DEV), torch.randn(sum(n) + 64, generator=g).to(DEV)
    params, grads, at = [], [], 1
    for x in n:
        params.append(buf[at:at + x])
        grads.append(gbuf[at:at + x])
        at += x
    edge = buf[:1].clone(), buf[at:].clone()
    for bits in (32, 8):
        opt = AdamW([{"params": params[:150], "lr": 2e-3, "weight_decay": 0.0}, {"params": params[150:]}], lr=LR, eps=EPS,
                    weight_decay=WD, state_bits=bits, max_norm=1.0, seed=2)
        ref = Ref(params, bits, 2, [(2e-3, 0.0)] * 150 + [(LR, WD)] * 80)
        opt.step(grads)
        torch.cuda.synchronize()
        _check(opt, ref, params, ref.step(grads, 1.0))
        assert torch.equal(buf[:1], edge[0]) and torch.equal(buf[at:], edge[1])


def test_not_finite_gradients():
    from ifd.optim import AdamW
    for bits in (32, 8):
        for bad in (float("nan"), float("inf"), -float("inf")):
            p = [torch.randn(300, device=DEV), torch.randn(500, device=DEV)]
            opt = AdamW(p, lr=LR, state_bits=bits, max_norm=1.0)
            g = [torch.randn(300, device=DEV), torch.randn(500, device=DEV)]
            opt.step(g)
            before = [t.clone() for t in p] + [t.clone() for t in opt.moments()]
            g[1][77] = bad
            opt.step(g)
            assert all(torch.equal(a, b) for a, b in zip(before, p + list(opt.moments())))
            # without the clip only the values that share a scale with it are spoilt
            opt2 = AdamW(p, lr=LR, state_bits=bits)
            opt2.step(g)
            opt2.step([torch.ones_like(t) for t in p])
            assert torch.isfinite(p[0]).all() and torch.isfinite(p[1][256:]).all()


def test_no_gradient_no_change_and_p_grad():
    from ifd.optim import AdamW
    p = [torch.nn.Parameter(torch.randn(300, device=DEV)), torch.nn.Parameter(torch.randn(40, device=DEV))]
    opt = AdamW(p, lr=LR, state_bits=8)
    was = p[1].detach().clone()
    p[0].grad = torch.randn(300, device=DEV)
    opt.step()
    assert torch.equal(p[1].detach(), was) and (opt.moments()[0][512:] == 0).all() and opt.step_count == 1


def test_second_moment_falls_on_average():
    """With zero gradients v must decay by b2 per step although a step moves it by less than half of its byte's spacing:
    rounding is right on average. Each rounding adds a variance of at most (v / 16)^2; the mean over N values after n steps
    is within 6 sqrt(n) / 16 / sqrt(N) of b2^n, and the v that shares its block with a constant larger one does not stick."""
    from ifd.optim import AdamW
    N, n = 256 * 512, 300
    p = torch.zeros(N, device=DEV)
    opt = AdamW([p], lr=0.0, betas=(B1, B2), weight_decay=0.0, state_bits=8, seed=9)
    opt.v.fill_(20 * 8 + 3)
    opt.v_scale.fill_(1.0)
    opt.v[::256] = 255
    g = torch.zeros(N, device=DEV)
    g[::256] = math.sqrt(1.875)  # keeps its v, and with it the block's scale, where it is
    v0 = opt.moments()[1].clone()
    for _ in range(n):
        opt.step([g])
    ratio = (opt.moments()[1] / v0).view(-1, 256)[:, 1:].double().mean().item()
    assert abs(ratio / B2 ** n - 1) <= 6 * math.sqrt(n) / 16 / math.sqrt(N), ratio
    assert (opt.moments()[1] > 0).all()


def test_resume_is_bit_exact_and_steps_repeat():
    from ifd.optim import AdamW
    g = torch.Generator().manual_seed(1)
    p0 = torch.randn(1000, generator=g).to(DEV)
    gs = [torch.randn(1000, generator=g).to(DEV) for _ in range(6)]
    for bits in (32, 8):
        runs = []
        for cut in (None, 3, None):
            p = p0.clone()
            opt = AdamW([p], lr=LR, state_bits=bits, max_norm=1.0, seed=4)
            for i, x in enumerate(gs):
                if i == cut:
                    sd = opt.state_dict()
                    opt = AdamW([p], lr=LR, state_bits=bits, max_norm=1.0)
                    opt.load_state_dict(sd)
                opt.step([x])
            runs.append((p, *opt.moments()))
        for r in runs[1:]:
            assert all(torch.equal(a, b) for a, b in zip(runs[0], r))


def test_agrees_with_the_flat_optimizer():
    """32-bit states do what the UNet trainer's ifd_tr_clip_adamw does on one flat buffer."""
    from ifd import _lib
    from ifd.optim import AdamW
    from ifd.train import P, chk, lib
    g = torch.Generator().manual_seed(8)
    n = 256 * 40
    p = (0.1 * torch.randn(n, generator=g)).to(DEV)
    q, m, v, nc = p.clone(), torch.zeros(n, device=DEV), torch.zeros(n, device=DEV), torch.zeros(2, device=DEV)
    opt = AdamW([q], lr=5e-5, weight_decay=0.01, max_norm=1.0)
    work = torch.empty(1024, dtype=torch.float64, device=DEV)
    for k in range(3):
        d = torch.randn(n, generator=g).to(DEV)
        opt.step([d])
        chk(lib().ifd_tr_clip_adamw(P(p), P(d.clone()), P(m), P(v), n, 1.0, 5e-5, 0.9, 0.999, 1e-8, 0.01, k + 1, P(work),
                                    P(nc), _lib.stream_ptr(torch.device(DEV))))
    torch.cuda.synchronize()
    # both round the same fp32 formulas; the clip coefficient here is formed in fp64: 2 ulp of the parameters
    assert ((p - q).abs() <= 4 * U * p.abs() + 12 * U * 3 * 5e-5).all()


def test_wrong_gradients_and_changed_parameters_are_refused():
    from ifd.optim import AdamW
    p = [torch.randn(8, 6, device=DEV), torch.randn(5, device=DEV)]
    opt = AdamW(p, lr=LR)
    good = [torch.randn(8, 6, device=DEV), torch.randn(5, device=DEV)]
    for bad, msg in (([good[0]], "1 gradients for 2"), ([good[0].t(), good[1]], "gradient 0"),
                     ([good[0].double(), good[1]], "gradient 0"), ([good[0], good[1].cpu()], "gradient 1"),
                     ([good[0], torch.randn(10, device=DEV)[::2]], "gradient 1")):
        with pytest.raises(ValueError, match=msg):
            opt.step(bad)
    assert opt.step_count == 0
    p[1].data = torch.randn(300, device=DEV)
    with pytest.raises(ValueError, match="parameter 1"):
        opt.step(good)
    graph = torch.cuda.CUDAGraph()
    opt2 = AdamW([good[0]], lr=LR)
    with torch.cuda.graph(graph):
        good[1].mul_(1.0)
        with pytest.raises(ValueError, match="captured"):
            opt2.step([good[0]])
