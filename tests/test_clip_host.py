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


def test_clipping_by_array_and_by_the_global_norm_is_refused(step):
    """As update_multi_ and MLP refuse it; nothing has been clipped or updated then, and what can be seen
    before the function is differentiated is seen before."""
    autograd, train, calls = step
    ps = params(autograd)
    with pytest.raises(ValueError, match="not both"):
        autograd.minimize_step(None, (), train.SGD(gclip=1.0), ps, gclip_global=2.0)
    ps[2].opt = train.Adam(gclip=0.5)
    with pytest.raises(ValueError, match="not both"):
        autograd.minimize_step(None, (), train.SGD(), iter(ps), gclip_global=2.0)
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="positive"):
            autograd.minimize_step(None, (), train.SGD(), ps, gclip_global=bad)
    assert calls == []
    autograd.minimize_step(None, (), train.SGD(gclip=1.0), ps)                 # by array alone: as ever
    assert [c[0] for c in calls[1:]] == ["update", "update"]


def test_a_parameter_met_on_the_tape_with_its_own_clipping_is_refused(step, monkeypatch):
    autograd, train, calls = step
    ps = params(autograd)
    ps[0].opt = train.SGD(gclip=1.0)
    monkeypatch.setattr(autograd, "params", lambda tape: ps)
    with pytest.raises(ValueError, match="not both"):
        autograd.minimize_step(None, (), train.SGD(), gclip_global=2.0)
    assert calls == ["diff"]


def cover(views):
    """how often each element of the buffer behind `views` is scaled"""
    import torch
    from knet_sm100 import train
    buf = torch.zeros(40)
    for v in train._disjoint([buf[a:b] for a, b in views]):
        v += 1
    return buf


@pytest.mark.parametrize("views", [[(0, 10), (5, 15)], [(5, 15), (0, 10), (0, 10)], [(0, 30), (3, 9), (8, 31)], [(0, 10), (10, 20)],
                                   [(7, 7), (3, 9), (3, 5), (4, 12), (30, 40)]], ids=str)
def test_overlapping_gradients_are_scaled_once(views):
    """Views of one buffer that share some of their elements: each of those is multiplied once, by one CTA."""
    want = [float(any(a <= i < b for a, b in views)) for i in range(40)]
    assert cover(views).tolist() == want


def test_arrays_that_share_part_of_an_element_are_refused():
    import torch
    from knet_sm100 import train
    raw = bytearray(64)
    with pytest.raises(ValueError, match="overlap"):
        train._disjoint([torch.frombuffer(raw, dtype=torch.float32, offset=o, count=8) for o in (0, 18)])


@pytest.mark.parametrize("views,shared", [([(0, 10), (5, 15)], True), ([(5, 15), (0, 30), (38, 39)], True), ([(0, 10), (10, 20)], False),
                                          ([(0, 10), (0, 10)], True), ([(0, 10), (4, 4)], False)], ids=str)
def test_a_plan_knows_whether_its_gradients_overlap(views, shared):
    """In a plan, whose table is used as it is, overlapping gradients cannot be clipped in place."""
    import torch
    from knet_sm100 import train
    buf = torch.zeros(40)
    plan = train.MultiTensorPlan([(torch.zeros(b - a), buf[a:b]) for a, b in views])
    assert plan.repeated == shared
