"""The optimizer's states where a run is cut or goes wrong: a trainer with 8-bit states saved and resumed, and states after a
gradient that is not finite.

The resumed run does the same launches on the same bytes as the uncut one, so every bit has to be equal. A block of 8-bit
states has one scale, the largest magnitude over 1.875: where one of its values is NaN the scale is NaN, and so are the values
that its 256 bytes stand for (NaN times any byte's value, 0 too).
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def _trainer(**kw):
    from ifd.manifest import make_state_dict
    from ifd.topology import REDUCED
    from ifd.train import UNetTrainer
    tr = UNetTrainer(REDUCED, device=DEV, state_bits=8, **kw)
    tr.load_state_dict(make_state_dict(REDUCED, seed=3))
    return tr


def test_trainer_with_8bit_states_resumes_where_it_stopped():
    """Saved through state_dict() and opt.state_dict(), loaded into a new trainer: the steps that follow are the uncut run's,
    bit for bit (bias corrections and the rounding's random bits go by the step number)."""
    gen = torch.Generator(device=DEV).manual_seed(1)
    runs = []
    a = _trainer(seed=5)
    grads = [torch.randn(a.numel, generator=gen, device=DEV) * 1e-3 for _ in range(6)]
    for cut in (None, 3):
        tr = _trainer(seed=5)
        for i, g in enumerate(grads):
            if i == cut:
                params = {k: v.clone() for k, v in tr.state_dict().items()}
                states = tr.opt.state_dict()
                tr = _trainer()
                tr.load_state_dict(params)
                tr.opt.load_state_dict(states)
                assert tr.step_count == 3
            tr.grad.copy_(g)
            tr.optimizer_step()
            assert tr.step_count == tr.opt.step_count == i + 1
        runs.append((tr.flat.clone(), *tr.opt.moments()))
    assert all(torch.equal(x, y) for x, y in zip(*runs))


def test_a_refused_step_is_not_counted():
    tr = _trainer()
    tr.grad.normal_()
    tr.optimizer_step()
    good, tr.grad = tr.grad, tr.grad.double()
    with pytest.raises(ValueError, match="gradient 0"):
        tr.optimizer_step()
    tr.grad = good
    assert tr.step_count == tr.opt.step_count == 1
    tr.step_count = 41  # a caller may set it, as with 32-bit states
    tr.optimizer_step()
    assert tr.step_count == tr.opt.step_count == 42


@pytest.mark.parametrize("at", [0, 77, 255, 511, 599])
def test_nan_gradient_spoils_its_8bit_block(at):
    """Without the clip. Every lane of the block's maximum, both directions of a first and of a later step."""
    from ifd.optim import AdamW
    g = torch.Generator(device=DEV).manual_seed(at)
    p = torch.randn(600, device=DEV, generator=g)
    opt = AdamW([p], lr=1e-3, state_bits=8)
    for k in range(3):
        d = torch.randn(600, device=DEV, generator=g)
        if k == 1:
            d[at] = float("nan")
        opt.step([d])
        m, v = opt.moments()
        b = at // 256
        bad = torch.zeros(m.numel(), dtype=torch.bool, device=DEV)
        if k:
            bad[b * 256:(b + 1) * 256] = True
        assert torch.equal(torch.isnan(m), bad) and torch.equal(torch.isnan(v), bad), k
        spoilt = torch.isnan(p)
        assert (spoilt.sum() == 1 and spoilt[at]) if k == 1 else torch.equal(spoilt, bad[:600] & (k == 2))


def test_a_step_that_the_library_refuses_is_not_counted():
    """Hyperparameters are the caller's to change between steps; the library checks them at the call."""
    from ifd.optim import AdamW
    for bits in (8, 32):
        p = torch.ones(300, device=DEV)
        opt = AdamW([p], lr=1e-3, state_bits=bits)
        opt.betas = (1.5, 0.999)
        with pytest.raises(RuntimeError, match="b1, b2 or eps"):
            opt.step([torch.ones_like(p)])
        assert opt.step_count == 0 and (p == 1).all()
        opt.betas = (0.9, 0.999)
        opt.step([torch.ones_like(p)])
        assert opt.step_count == 1 and (p < 1).all()
