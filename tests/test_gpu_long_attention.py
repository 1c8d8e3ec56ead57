"""Attention above the 16x16 map on the framework's own paths (32x32 = 1024 tokens): the sampler's UNet forward, one
AttentionBlock's forward and backward in the trainer, and the trainer's step with 8-bit optimizer states.

References: the oracle's modules in fp64 on the CPU (autograd for the gradients). Tolerances as for the same modules at
16x16: the block within 1e-5 (outputs, dx) and 1e-4 (parameter gradients) of each tensor's largest value, the UNet
evaluation in fp32 within 2e-4 of its largest value.
"""
import dataclasses

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def _rel(a, b):
    return float((a.detach().double().cpu() - b).abs().max() / b.abs().max())


@pytest.mark.parametrize("r,C", [(32, 128), (64, 64)])  # 1024 and 4096 tokens (the block's convs take these maps)
def test_attention_block_forward_backward(r, C):
    from ifd.train import BlockTrainer
    from oracle import ref_unet
    g = torch.Generator().manual_seed(r)
    bt = BlockTrainer("attn", C, C, device=DEV)
    sd = {}
    for k, s in bt.spec:
        sd[k] = 0.1 * torch.randn(s, generator=g) + (1.0 if k == "norm.weight" else 0.0)
        if len(s) > 1:
            sd[k] = torch.randn(s, generator=g) * (1.5 if k == "qkv.weight" else 1.0) / s[1] ** 0.5
    bt.load_state_dict(sd)
    x, dy = torch.randn(2, C, r, r, generator=g), torch.randn(2, C, r, r, generator=g)
    y = bt.forward_block(x.to(DEV))
    dx, _ = bt.backward_block(dy.to(DEV))
    torch.cuda.synchronize()
    p64 = {k: v.double().requires_grad_() for k, v in sd.items()}
    x64 = x.double().requires_grad_()
    ref = ref_unet.attention(p64, "", x64, 64)
    grads = torch.autograd.grad(ref, [x64, *p64.values()], dy.double())
    assert _rel(y, ref.detach()) <= 1e-5 and _rel(dx, grads[0]) <= 1e-5
    for (k, _), gr in zip(p64.items(), grads[1:]):
        assert _rel(bt.g(k), gr) <= 1e-4, k


def test_unet_forward_with_32x32_attention():
    from ifd.manifest import make_state_dict
    from ifd.model import DiffusionInpaintingModel
    from ifd.topology import REDUCED
    from oracle import ref_unet
    cfg = dataclasses.replace(REDUCED, attention_resolutions=(2, 16))
    ocfg = dataclasses.replace(ref_unet.REDUCED, attention_resolutions=(2, 16))
    sd = make_state_dict(cfg, seed=3)
    m = DiffusionInpaintingModel(cfg, device=DEV, precision="fp32")
    m.load_state_dict(sd)
    g = torch.Generator().manual_seed(2)
    x, mi = torch.randn(2, 3, 64, 64, generator=g), torch.randn(2, 3, 64, 64, generator=g)
    mk = (torch.rand(2, 1, 64, 64, generator=g) > 0.5).float()
    t = torch.tensor([3, 700])
    with torch.no_grad():
        y = m(x.to(DEV), t.to(DEV), mi.to(DEV), mk.to(DEV))
        sd64 = {k: v.double() for k, v in ref_unet.strip_prefix(sd).items()}
        ref = ref_unet.inpaint_forward(sd64, x.double(), t, mi.double(), mk.double(), ocfg)
    assert _rel(y, ref) <= 2e-4


def _trainer(bits, **kw):
    from ifd.manifest import make_state_dict
    from ifd.topology import REDUCED
    from ifd.train import UNetTrainer
    cfg = dataclasses.replace(REDUCED, attention_resolutions=(2, 16))
    tr = UNetTrainer(cfg, device=DEV, state_bits=bits, **kw)
    tr.load_state_dict(make_state_dict(cfg, seed=3))
    return tr


def test_train_step_with_32x32_attention_and_8bit_states():
    """The first step starts from empty states, so that 8-bit states change nothing yet: both optimizers move every
    parameter alike, up to the fp32 forms of the same formula (the clip coefficient is fp64 in one). The 8-bit states then
    are within one byte's spacing (1/8, or the block's smallest value) of the 32-bit ones, and the trainer goes on."""
    from ifd.schedules import create_gaussian_diffusion
    diff = create_gaussian_diffusion(steps=1000, learn_sigma=True, noise_schedule="cosine")
    g = torch.Generator().manual_seed(4)
    img = torch.randn(2, 3, 64, 64, generator=g).to(DEV)
    mask = torch.zeros(2, 1, 64, 64, device=DEV)
    mask[:, :, 16:48, 16:48] = 1
    noise = torch.randn(2, 3, 64, 64, generator=g).to(DEV)
    t = torch.tensor([20, 500], device=DEV)
    trs = []
    for bits in (32, 8):
        tr = _trainer(bits)
        torch.manual_seed(0)
        tr.train_step(diff, img, img * (1 - mask), mask, t, noise=noise)
        trs.append(tr)
    a, b = trs
    torch.cuda.synchronize()
    U = 2.0 ** -24
    assert abs(float(a.norm_coef[0]) - float(b.norm_coef[0])) <= 1e-6 * float(a.norm_coef[0])
    # the step's size is lr m / sqrt(v) <= lr (first step): two roundings of p and 40 of the step
    assert ((a.flat - b.flat).abs() <= 3 * U * a.flat.abs() + 80 * U * a.lr).all()
    m8, v8 = b.opt.moments()
    at = 0
    for k, _ in a.spec:
        o, shape = a.offsets[k]
        n = a.p(k).numel()
        for flat, q, low in ((a.m, m8, 2.0 ** -15), (a.v, v8, 2.0 ** -31)):
            x, y = flat[o:o + n].double(), q[at:at + n].double()
            top = torch.nn.functional.pad(x.abs(), (0, -n % 256)).view(-1, 256).amax(1).repeat_interleave(256)[:n]
            assert ((x - y).abs() <= x.abs() * (1 / 8 + 1e-5) + top * low * 1.2).all(), k
        at += -(-n // 256) * 256
    loss = [float(b.train_step(diff, img, img * (1 - mask), mask, t, noise=noise)) for _ in range(2)]
    assert all(torch.isfinite(torch.tensor(loss))) and b.step_count == 3 and b.opt.step_count == 3


def test_attention_entry_covers_long_maps():
    """ifd_tr_attention at T > 256 (the kernel it had keeps one row of 256 scores)."""
    from ifd import _lib
    from ifd.train import P, chk, lib
    g = torch.Generator().manual_seed(0)
    for T in (257, 300, 1024):
        qkv = torch.randn(2, T, 3 * 128, generator=g)
        out = torch.empty(2, T, 128, device=DEV)
        chk(lib().ifd_tr_attention(P(qkv.to(DEV)), 2, T, 128, 64 ** -0.25, P(out), _lib.stream_ptr(DEV)))
        q, k, v = qkv.double().view(2, T, 3, 2, 64).permute(2, 0, 3, 1, 4)
        ref = (torch.softmax(q @ k.transpose(-1, -2) / 8, -1) @ v).transpose(1, 2).reshape(2, T, 128)
        torch.cuda.synchronize()
        assert _rel(out, ref) <= 2e-5
