"""Host side of clipping by the norm of all gradients: what minimize_step does with its parameters.
The device's work is replaced by a record of the calls, so these run without a GPU."""
import pytest


class Array:
    """stands for a one-element KnetArray"""

    class data:
        item = staticmethod(lambda: 1.5)


@pytest.fixture
def step(monkeypatch):
    """minimize_step with its differentiation, clipping and update recorded in `calls`."""
    from knet_sm100 import autograd, train
    calls = []

    def diff(f, *args):
        calls.append("diff")
        tape = autograd.Tape()
        tape.result = Array()
        return tape

    monkeypatch.setattr(autograd, "diff", diff)
    monkeypatch.setattr(train, "gclip_global_", lambda grads, c: calls.append(("clip", list(grads), c)))
    monkeypatch.setattr(train, "update_", lambda w, g, opt: calls.append(("update", w, g, opt.lr)))
    return autograd, train, calls


def params(autograd):
    ps = [autograd.Param(f"w{k}") for k in range(3)]
    for k in (0, 2):
        ps[k].grad = f"g{k}"
    return ps


def test_parameters_may_be_a_generator(step):
    """A generator of parameters, walked once for the clipping and once for the updates."""
    autograd, train, calls = step
    ps = params(autograd)
    assert autograd.minimize_step(None, (), train.SGD(lr=0.25), (p for p in ps), gclip_global=2.0) == 1.5
    assert calls == ["diff", ("clip", ["g0", "g2"], 2.0), ("update", "w0", "g0", 0.25), ("update", "w2", "g2", 0.25)]
