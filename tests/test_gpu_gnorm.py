"""The norm of all gradients as one vector, clipping by it in place, and the updates that apply it.

The norm is a Float64 sum of exact squares: n additions of positive terms, so its relative error is at
most n * 2^-53 / 2 + a few roundings, whatever the order.  The clipped gradient is lmul!(factor, g):
one Float64 product rounded once to the element type, which a host repeats bit for bit from the
factor it reads back."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

NPDT = {torch.float32: np.float32, torch.float64: np.float64}
SETS = [[1], [5, 3], [50176, 64, 640, 10], [8192, 8193, 1, 16384, 7], [3] * 300, [200_001, 100_000, 17]]


def flat_set(sizes, dtype, off, seed=0, std=1e-3):
    """gradients in one buffer that starts `off` elements in, with guards at both ends"""
    rng = np.random.default_rng(seed + len(sizes))
    host = [(rng.standard_normal(n) * std).astype(NPDT[dtype]) for n in sizes]
    buf = torch.full((off + sum(sizes) + 8,), 7.0, dtype=dtype, device="cuda")
    views, at = [], off
    for h in host:
        buf[at:at + h.size] = torch.from_numpy(h).cuda()
        views.append(buf[at:at + h.size])
        at += h.size
    return host, buf, views


def exact_norm(host, gscale):
    return abs(gscale) * float(np.sqrt(sum(float((h.astype(np.longdouble) ** 2).sum()) for h in host)))


def near(norm, want, host):
    n = sum(h.size for h in host)
    return abs(float(norm) - want) <= (n + 16) * 2.0 ** -53 * want


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("off", [0, 3])
@pytest.mark.parametrize("sizes", SETS, ids=lambda s: f"{len(s)}x{max(s)}")
def test_norm_and_clip_in_place(K, dtype, off, sizes):
    host, buf, views = flat_set(sizes, dtype, off)
    want = exact_norm(host, 0.5)
    plan = K.MultiTensorPlan([(v, v) for v in views])
    assert near(K.gnorm(plan, 0.5), want, host)
    assert near(K.gnorm([K.KnetArray(v) for v in views], -0.5), want, host)
    assert near(K.gclip_global_(plan, want * 1.5, 0.5), want, host)              # below the limit: nothing changes
    assert all(np.array_equal(v.cpu().numpy(), h) for v, h in zip(views, host))
    norm = K.gclip_global_(plan, want * 0.25, 0.5)
    assert near(norm, want, host)
    factor = (want * 0.25) / float(norm)
    for v, h in zip(views, host):
        np.testing.assert_array_equal(v.cpu().numpy(), (factor * h.astype(np.float64)).astype(NPDT[dtype]))
    assert bool((buf[:off] == 7).all()) and bool((buf[off + sum(sizes):] == 7).all())


@pytest.mark.parametrize("std", [1e-30, 1e25])
def test_squares_beyond_the_element_type(K, std):
    """Float32 squares would vanish or overflow here."""
    host, _, views = flat_set([1000, 70_000], torch.float32, 0, std=std)
    assert near(K.gnorm(views), exact_norm(host, 1.0), host)


def test_values_that_are_not_finite(K):
    host, _, views = flat_set([1000, 20_000], torch.float32, 0)
    views[1][77] = float("nan")
    kept = [v.clone() for v in views]
    assert np.isnan(float(K.gclip_global_(views, 1e-9)))
    assert all(torch.equal(a.nan_to_num(5.0), b.nan_to_num(5.0)) for a, b in zip(views, kept))
    views[1][77] = float("inf")
    assert float(K.gnorm(views)) == float("inf")
    K.gclip_global_(views, 1.0)                                               # inf * 0, as gclip! does
    assert not views[0].any() and bool(torch.isnan(views[1][77]))
    zero = [torch.zeros(100, device="cuda")]
    assert float(K.gclip_global_(zero, 1.0)) == 0 and not zero[0].any()


def test_one_array_listed_twice_is_scaled_once(K):
    g, h = torch.ones(100, device="cuda"), torch.ones(44, device="cuda")
    assert abs(float(K.gclip_global_([g, h, g], 1.0)) - np.sqrt(244)) < 1e-12
    assert torch.allclose(g, torch.full_like(g, 1 / np.sqrt(244)), rtol=1e-7, atol=0) and torch.equal(g[:44], h)
    with pytest.raises(ValueError):
        K.gclip_global_(K.MultiTensorPlan([(g, g), (h, h), (g, g)]), 1.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("name", ["sgd", "momentum", "adam"])
def test_update_applies_the_factor(K, dtype, name):
    """update_multi_(..., gclip_global=c) = clip a copy of the gradients in place, then update: the same bits."""
    sizes = [4096 * 3, 17, 8192, 1, 20001]
    opts = {"sgd": lambda: K.SGD(lr=0.1), "momentum": lambda: K.Momentum(lr=0.05, gamma=0.9), "adam": lambda: K.Adam()}[name]
    sides = []
    for fused in (True, False):
        _, _, g = flat_set(sizes, dtype, 3)
        _, _, w = flat_set(sizes, dtype, 3, seed=9, std=0.02)
        m, v = ([torch.zeros_like(a) for a in g] for _ in range(2))
        plan = K.MultiTensorPlan([t[:{"sgd": 2, "momentum": 3, "adam": 4}[name]] for t in zip(w, g, m, v)])
        opt, kept = opts(), [a.clone() for a in g]
        for step, limit in enumerate((1e-3, 100.0, 5e-2)):
            for a, b in zip(g, kept):
                a.copy_(b * (step + 1))
            if fused:
                norm = K.update_multi_(plan, opt, gclip_global=limit)
                assert all(torch.equal(a, b * (step + 1)) for a, b in zip(g, kept))       # gradients stay as they are
            else:
                norm = K.gclip_global_(plan, limit)
                assert K.update_multi_(plan, opt) is None
        sides.append([float(norm)] + [t.clone() for t in w + m + v])
    assert sides[0][0] == sides[1][0]
    assert all(torch.equal(a, b) for a, b in zip(sides[0][1:], sides[1][1:]))


def test_factor_with_gradient_scale(K):
    """With gscale the norm is that of gscale*g and the update sees gscale * lmul!(factor, g)."""
    host, _, g = flat_set([30_000, 9], torch.float32, 0)
    w = [torch.zeros_like(a) for a in g]
    want = exact_norm(host, 0.125)
    norm = K.update_multi_(K.MultiTensorPlan(list(zip(w, g))), K.SGD(lr=1.0), 0.125, gclip_global=want / 4)
    assert near(norm, want, host)
    f = (want / 4) / float(norm)
    for a, h in zip(w, host):
        np.testing.assert_array_equal(-a.cpu().numpy(), (f * h.astype(np.float64)).astype(np.float32) * np.float32(0.125))


def test_captured_step_and_two_streams(K):
    host, _, g = flat_set([40_000, 333, 8192], torch.float32, 0)
    plan = K.MultiTensorPlan([(a, a) for a in g])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = K.gclip_global_(plan, 0.01)
    for s in (1.0, 3.0):
        for a, h in zip(g, host):
            a.copy_(torch.from_numpy(h).cuda() * s)
        graph.replay()
        torch.cuda.synchronize()
        assert abs(float(norm) - s * exact_norm(host, 1.0)) < 1e-6 * s
        assert abs(float(K.gnorm(plan)) - 0.01) < 1e-8
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [None, None]
    want = float(K.gnorm(plan))
    torch.cuda.synchronize()
    for _ in range(5):
        for k in (0, 1):
            with torch.cuda.stream(streams[k]):
                got[k] = K.gnorm(plan)                       # the plan is shared, its scratch is not
    torch.cuda.synchronize()
    assert [float(t) for t in got] == [want, want]


def test_model_with_clipping_eager_captured_and_by_hand(K):
    sizes, B = [30, 16, 5], 20
    rng = np.random.default_rng(3)
    x = K.KnetArray(rng.standard_normal((30, B)).astype(np.float32))
    y = torch.from_numpy(rng.integers(1, 6, B).astype(np.int32)).cuda()
    plain = K.MLP(sizes, B, optimizer=K.Adam())
    clipped = K.MLP(sizes, B, optimizer=K.Adam(), gclip_global=0.05)
    graph = K.MLP(sizes, B, optimizer=K.Adam(), gclip_global=0.05).capture()
    for _ in range(4):
        plain.loss(plain.forward(x), y)
        plain.backward(x, y)
        norm = K.gclip_global_(plain.plan, 0.05)
        plain.update()
        plain.step_no += 1
        clipped.step(x, y)
        graph.step_graph(x, y)
        torch.cuda.synchronize()
        assert float(norm) == float(clipped.gnorm) == float(graph.gnorm) > 0.05
        assert torch.equal(plain.flat_w, clipped.flat_w) and torch.equal(plain.flat_w, graph.flat_w)
    with pytest.raises(ValueError):
        K.MLP(sizes, B, optimizer=K.Adam(gclip=1.0), gclip_global=0.05)
    with pytest.raises(ValueError):
        K.MLP(sizes, B, gclip_global=-1.0)


@pytest.mark.parametrize("limit", [0.3, 0.1])
def test_a_training_step_of_a_tied_model(K, limit):
    """The two operators as they are used together: embed tokens, score them with the same matrix,
    differentiate, clip by the global norm, update - against the same step written with the score
    matrix and numpy's clipping."""
    A = K.autograd
    V, H, N = 97, 24, 60
    rng = np.random.default_rng(5)
    e0 = np.asfortranarray(rng.standard_normal((H, V)) * 0.3)
    b0 = np.asfortranarray(rng.standard_normal(V) * 0.1)
    tokens = rng.integers(1, V + 1, N).tolist()
    labels = rng.integers(0, V + 1, N).astype(np.int32)
    params = []
    for fused in (True, False):
        e, b = A.Param(K.KnetArray(e0)), A.Param(K.KnetArray(b0))

        def loss():
            x = A.tanh(e[K.indexing.COLON, tokens])
            return A.linear_nll(e, x, labels, b, True) if fused else A.nll(A.At_mul_B(e, x) + b, labels)

        for step in range(3):
            if fused:
                A.minimize_step(loss, (), K.Adam(lr=0.01), gclip_global=limit)
            else:
                A.diff(loss)
                if e.opt is None:
                    e.opt, b.opt = K.Adam(lr=0.01), K.Adam(lr=0.01)
                ge, gb = e.grad.numpy(), b.grad.numpy()
                norm = np.sqrt((ge ** 2).sum() + (gb ** 2).sum())
                assert (norm > limit) == (limit == 0.1) or step > 0        # the smaller limit clips, the larger does not
                for p, g in ((e, ge), (b, gb)):
                    K.update_(p.value, K.KnetArray(np.asfortranarray(g * min(1.0, limit / norm))), p.opt)
        params.append((e.value.numpy(), b.value.numpy()))
    for p, q in zip(*params):
        np.testing.assert_allclose(p, q, rtol=1e-8, atol=1e-10)


def test_refusals(K):
    g = torch.ones(10, device="cuda")
    plan = K.MultiTensorPlan([(g, g)])
    for bad in (0, -1.0, float("nan")):
        with pytest.raises(ValueError):
            K.gclip_global_(plan, bad)
    with pytest.raises(ValueError):
        K.update_multi_(plan, K.SGD(gclip=1.0), gclip_global=1.0)
    with pytest.raises(ValueError):
        K.update_multi_(plan, K.SGD(), gclip_global=-1.0)
    with pytest.raises(TypeError):
        K.update_multi_(plan, K.Nesterov(), gclip_global=1.0)
    with pytest.raises(TypeError):
        K.gnorm([g, g.double()])
    with pytest.raises(TypeError):
        K.gnorm([g.half()])
    with pytest.raises(TypeError):
        K.gnorm([torch.ones(4, 4, device="cuda").t()[1:]])
    assert float(K.gnorm([])) == 0.0


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_overlapping_views_are_scaled_once(K, dtype):
    """Views that share part of their elements: each listed array counts in the norm, each element is
    multiplied once."""
    host, buf, (g,) = flat_set([50_000], dtype, 3)
    views = [g[20_000:], g[:30_000], K.KnetArray(g[100:200])]
    want = exact_norm([host[0][20_000:], host[0][:30_000], host[0][100:200]], 1.0)
    norm = K.gclip_global_(views, want / 8)
    assert near(norm, want, [host[0], host[0]])
    factor = (want / 8) / float(norm)
    np.testing.assert_array_equal(g.cpu().numpy(), (factor * host[0].astype(np.float64)).astype(NPDT[dtype]))
    with pytest.raises(ValueError):
        K.gclip_global_(K.MultiTensorPlan([(v, v) for v in (g[20_000:], g[:30_000])]), 1.0)


@pytest.mark.parametrize("off", [0, 1])
@pytest.mark.parametrize("stds", [(1e200, 1e200), (1e-200, 1e-200), (1e-309, 1e-309), (1e200, 1.0), (1.0, 1e-200), (1e-200, 1e-165),
                                  (1e-200, 1e-136), (1e152, 1e150), (1e200, 1e-200), (1e-200, 0.0)], ids=str)
def test_float64_squares_beyond_the_range(K, stds, off):
    """Finite gradients whose squares overflow or vanish in Float64, alone and beside ordinary arrays.  The root
    per chunk and its square add two roundings to each term, within the bound's 16."""
    sizes = [20_000, 9_000, 3]
    host, _, g = flat_set(sizes, torch.float64, off, std=1.0)
    for a, h, s in zip(g, host, stds + stds[:1]):
        h *= s
        a.copy_(torch.from_numpy(h).cuda())
    want = np.sqrt(sum((h.astype(np.longdouble) ** 2).sum() for h in host))       # 15 bits of exponent
    assert abs(float(K.gnorm(g)) - want) <= (sum(sizes) + 16) * 2.0 ** -53 * want
    norm = float(K.gclip_global_(g, float(want / 4)))
    for a, h in zip(g, host):
        np.testing.assert_array_equal(a.cpu().numpy(), (float(want / 4) / norm) * h)


def test_a_norm_beyond_float64(K):
    """Entries near the type's largest: their norm is inf, the clipped gradients have the norm asked for."""
    n = 30_000
    g = [torch.full((n,), 1.5e308, dtype=torch.float64, device="cuda"), torch.full((100,), -1.0, dtype=torch.float64, device="cuda")]
    assert float(K.gnorm(g)) == np.inf and abs(float(K.gnorm(g, 2.0 ** -20)) / (1.5e308 * 2.0 ** -20 * n ** 0.5) - 1) < 1e-11
    assert float(K.gclip_global_(g, 3.0)) == np.inf
    # a factor of about 2^-1031 has 43 bits left
    assert bool(((g[0] * n ** 0.5 / 3.0 - 1).abs() < 2.0 ** -41).all()) and bool((g[1].abs() < 1e-300).all())
    zero = [torch.zeros(20_000, dtype=torch.float64, device="cuda")]
    assert float(K.gclip_global_(zero, 1.0)) == 0 and not zero[0].any()
    zero[0][7] = float("inf")
    assert float(K.gnorm(zero)) == np.inf
    zero[0][8] = float("nan")
    assert np.isnan(float(K.gnorm(zero)))
