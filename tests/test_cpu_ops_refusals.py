"""Calls of the attention-layer operators that must be refused before anything is written, on the host (no GPU): the device
check is replaced, so that every other check runs on CPU tensors."""
import pytest
import torch


@pytest.fixture
def anywhere(monkeypatch):
    """CPU tensors pass the device check; a call that reaches the library fails the test."""
    from ifd import _ops, attention, optim, rotary

    def reached(*a):
        raise AssertionError("the call was not refused")
    for m in (_ops, attention, optim, rotary):
        if hasattr(m, "same_device"):
            monkeypatch.setattr(m, "same_device", lambda *t: t[0].device)
        if hasattr(m, "call"):
            monkeypatch.setattr(m, "call", reached)


def _qkv():
    return torch.zeros(2, 6, 4, 16), torch.zeros(2, 6, 2, 16), torch.zeros(2, 6, 2, 16)


# strides of a [2, 6, 4, 16] tensor some of whose elements are one place
SHARED = [(384, 64, 0, 1), (0, 64, 16, 1), (384, 16, 16, 1), (64, 64, 16, 1), (384, 64, 12, 1), (320, 64, 16, 1), (16, 64, 16, 1)]
# and of one whose elements are all apart: padded, transposed, every other head, batch innermost
APART = [(384, 64, 16, 1), (500, 80, 20, 1), (384, 16, 96, 1), (1024, 128, 32, 1), (64, 128, 16, 1)]


@pytest.mark.parametrize("st", SHARED)
def test_outputs_whose_elements_share_a_place(anywhere, st):
    from ifd.attention import attention, attention_bwd
    from ifd.rotary import qk_norm_rope, qk_norm_rope_bwd
    q, k, v = _qkv()
    o = torch.zeros(4096).as_strided((2, 6, 4, 16), st)
    calls = [lambda: attention(q, k, v, out=o), lambda: qk_norm_rope(q, k, q_out=o),
             lambda: attention_bwd(q, q, k, v, q, torch.zeros(2, 4, 6), dq=o),
             lambda: qk_norm_rope_bwd(q, k, q, k, dq=o), lambda: qk_norm_rope(o, k, q_out=o)]
    for f in calls:
        with pytest.raises(ValueError, match="share their place"):
            f()


@pytest.mark.parametrize("st", APART)
def test_outputs_whose_elements_are_apart(anywhere, st):
    from ifd import _ops
    x = torch.zeros(8192).as_strided((2, 6, 4, 16), st)
    assert _ops.output(x, torch.zeros(2, 6, 4, 16), "out") is x
    one = torch.zeros(8192).as_strided((2, 1, 4, 16), (384, 0, 16, 1))  # a size of one: its stride says nothing
    assert _ops.output(one, torch.zeros(2, 1, 4, 16), "out") is one
    none = torch.zeros(8192).as_strided((2, 0, 4, 16), (0, 0, 0, 1))
    assert _ops.output(none, torch.zeros(2, 0, 4, 16), "out") is none


def test_places_agree_with_an_enumeration():
    """Every stride triple of a small set against the set of addresses: no shared place is let through, and what is refused
    either shares one or has strides that do not nest."""
    import itertools
    from ifd._ops import _apart
    n = (2, 3, 4)
    for st in itertools.product((1, 2, 3, 4, 6, 8, 9, 12), repeat=3):
        seen = [sum(i * s for i, s in zip(ix, st)) for ix in itertools.product(*map(range, n))]
        order = sorted(zip(st, n))
        nest = all(b[0] > sum((m - 1) * s for s, m in order[:i + 1]) for i, b in enumerate(order[1:]))
        assert _apart(torch.zeros(256).as_strided(n, st)) == nest
        assert not nest or len(set(seen)) == len(seen)


def test_forward_mode_tangents_are_refused(anywhere):
    """An operator that records nothing must not drop a tangent, under torch.no_grad() no more than without it."""
    import torch.autograd.forward_ad as fw
    from ifd.attention import attention, attention_bwd
    from ifd.rotary import qk_norm_rope, qk_norm_rope_bwd
    q, k, v = _qkv()
    w, lse = torch.ones(16), torch.zeros(2, 4, 6)
    with fw.dual_level():
        d = lambda t: fw.make_dual(t, torch.ones_like(t))  # noqa: E731
        calls = [lambda: attention(d(q), k, v), lambda: attention(q, d(k), v), lambda: attention(q, k, d(v)),
                 lambda: attention_bwd(d(q), q, k, v, q, lse), lambda: attention_bwd(q, q, k, v, d(q), lse),
                 lambda: attention_bwd(q, q, k, v, q, d(lse)), lambda: attention_bwd(q, q, k, d(v), q, lse),
                 lambda: qk_norm_rope(q, d(k)), lambda: qk_norm_rope(q, k, d(w)), lambda: qk_norm_rope_bwd(q, d(k), q, k)]
        for f in calls:
            with pytest.raises(ValueError, match="tangent"):
                f()
            with torch.no_grad(), pytest.raises(ValueError, match="tangent"):
                f()
        with pytest.raises(AssertionError, match="not refused"):  # no tangent: the call goes on
            attention(q, k, v)
    with pytest.raises(ValueError, match="tangent"):
        torch.func.jvp(lambda x: attention(x, k, v)[0], (q,), (q,))


def test_outputs_that_autograd_follows_are_refused(anywhere):
    """A caller's output that requires gradients or carries a tangent would be written behind autograd's back."""
    import torch.autograd.forward_ad as fw
    from ifd.attention import attention, attention_bwd
    from ifd.rotary import qk_norm_rope, qk_norm_rope_bwd
    q, k, v = _qkv()
    lse = torch.zeros(2, 4, 6)
    calls = lambda o: [lambda: attention(q, k, v, out=o), lambda: qk_norm_rope(q, k, q_out=o),  # noqa: E731
                       lambda: attention_bwd(q, q, k, v, q, lse, dq=o), lambda: qk_norm_rope_bwd(q, k, q, k, dq=o)]
    leaf = torch.zeros(2, 6, 4, 16, requires_grad=True)
    for o in (leaf, leaf * 2, leaf[:]):
        was = o._version
        for f in calls(o):
            with pytest.raises(ValueError, match="records no gradients"):
                f()
            assert o._version == was
            with torch.no_grad(), pytest.raises(AssertionError, match="not refused"):
                f()
            was = o._version
    with fw.dual_level():
        for f in calls(fw.make_dual(torch.zeros(2, 6, 4, 16), torch.ones(2, 6, 4, 16))):
            with torch.no_grad(), pytest.raises(ValueError, match="tangent"):
                f()


def test_optimizer_takes_no_tensor_for_a_list(anywhere):
    """A tensor walks over its rows: views of their own that never have a .grad. One tensor as a group's "params" is that
    tensor, as in torch.optim; in the list's place it is refused."""
    from ifd.optim import AdamW
    w = torch.nn.Parameter(torch.zeros(3, 4))
    assert AdamW([{"params": w}, {"params": [torch.zeros(5)]}]).params[0] is w
    with pytest.raises(ValueError, match="a list of tensors or of groups"):
        AdamW(w)
    assert len(AdamW(iter([w, torch.zeros(2)])).params) == 2


def test_group_options_are_not_ignored(anywhere):
    """betas, eps, max_norm and the rest belong to the optimizer: a group that sets one is refused, as are rates below 0 in a
    group and a group without parameters."""
    from ifd.optim import AdamW
    p = torch.zeros(5)
    for g, msg in (({"params": [p], "betas": (0.5, 0.9)}, "betas"), ({"params": [p], "eps": 1e-3}, "eps"),
                   ({"params": [p], "amsgrad": True}, "amsgrad"), ({"params": [p], "lr": -1.0}, "not negative"),
                   ({"params": [p], "weight_decay": float("nan")}, "not negative"), ({"lr": 1.0}, "params")):
        with pytest.raises(ValueError, match=msg):
            AdamW([g])
    o = AdamW([{"params": [p], "lr": 0.5, "weight_decay": 0.0}], lr=1.0, weight_decay=1.0)
    assert o.groups[0]["lr"] == 0.5 and o.groups[0]["weight_decay"] == 0.0


@pytest.mark.parametrize("bits", [8, 32])
def test_refused_states_change_nothing(anywhere, bits):
    """load_moments and load_state_dict look at every part before they copy one."""
    from ifd.optim import AdamW
    src, dst = AdamW([torch.zeros(300)], state_bits=bits, seed=3), AdamW([torch.zeros(300)], state_bits=bits)
    for t in (src.m, src.v, src.m_scale, src.v_scale):
        if t is not None:
            t.fill_(7)
    src.step_count = 9
    good = src.state_dict()
    bad = [{**good, "v": good["v"][:-1]}, {**good, "v": None}, {k: v for k, v in good.items() if k != "step"},
           {k: v for k, v in good.items() if k != "seed"}, {**good, "state_bits": 40 - bits}, {**good, "step": -1}]
    if bits == 8:
        bad += [{**good, "v_scale": None}, {**good, "v_scale": good["v_scale"].double()}]
    for d in bad:
        with pytest.raises((ValueError, KeyError)):
            dst.load_state_dict(d)
        assert dst.step_count == 0 and dst.seed == 0
        assert all((t == 0).all() for t in (dst.m, dst.v, dst.m_scale, dst.v_scale) if t is not None)
    dst.load_state_dict(good)
    assert dst.step_count == 9 and dst.seed == 3 and (dst.m == 7).all() and (dst.v == 7).all()
