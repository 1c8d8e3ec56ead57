"""The optimizer's states where a run is cut or a step is refused: a trainer with 8-bit states saved and resumed.

The resumed run does the same launches on the same bytes as the uncut one, so every bit has to be equal.
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
