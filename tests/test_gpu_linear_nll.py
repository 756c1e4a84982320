"""linear_nll (nll of w*x .+ b without the scores) and its gradients against a plain evaluation in
64 bits.

Error bounds, entry by entry, with u the unit roundoff of the element type (2^-24, 2^-53):
  a sum of K products, in any order, by fused multiply-adds or by exact products of split operands
  added with truncation, is off by at most gamma(K) * sum |a||b|, gamma(K) = (K + 40) * 2u (a
  truncated addition loses up to 2u; the 40 covers what splitting operands leaves out);
  a score s = w.x + b:      ds <= gamma(H) * (|w|.|x|) + 2u (|s| + |b|)
  lse: the largest ds of its instance (d lse / d s are weights that add up to 1) + what exp, the
  sum of V exponentials and the logarithm do, (V/64 + 40) * 2u, + u |lse|
  p = exp(s - lse):         p * (exp(ds + dlse + 8u) - 1 + 8u); p - 1 rounds once more
  the gradients: that through the products' absolute values, + gamma of the product itself."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.float64: 2.0 ** -53}
SHAPES = [(1, 1, 1), (2, 3, 1), (10, 64, 100), (64, 64, 64), (65, 16, 257), (129, 65, 3), (128, 128, 128), (1000, 300, 33),
          (257, 515, 130), (300, 40, 513), (5003, 128, 70), (2500, 1025, 17),
          # few instances: one to eight vectors, several groups of eight, chunks of classes joined in either way
          (2100, 300, 1), (2101, 301, 2), (4300, 96, 4), (130, 2000, 7), (515, 517, 8), (5000, 64, 20), (100, 77, 31),
          # tensor-core tiles: sums cut because of few tiles (all three products), odd sizes, several rounds
          (300, 2000, 400), (40, 520, 5000), (1001, 260, 301), (1000, 256, 300), (3001, 515, 333), (129, 4099, 257)]


def gamma(k, u):
    return (k + 40) * 2 * u


class Case:
    """Inputs on the GPU and, in 64 bits, the results with their error bounds."""

    def __init__(self, V, H, N, dtype, trans, bias, skip, seed=0, std=2.0):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed + 17 * V + 5 * H + N)
        self.V, self.H, self.N, self.dtype, self.trans = V, H, N, dtype, trans
        self.ds_step = 0.0                  # absolute rounding of dS (without g)
        self.w = torch.randn((V, H), generator=g, device="cuda", dtype=dtype) * (std / math.sqrt(H))
        self.x = torch.randn((N, H), generator=g, device="cuda", dtype=dtype)
        self.b = torch.randn(V, generator=g, device="cuda", dtype=dtype) if bias else None
        self.labels = torch.randint(1, V + 1, (N,), generator=g, device="cuda", dtype=torch.int32)
        if skip:
            self.labels[torch.rand(N, generator=g, device="cuda") < 0.3] = 0
            self.labels[0] = 0

    def arrays(self, K):
        w = (self.w if self.trans else self.w.t()).contiguous().view(-1)
        kw = K.KnetArray(w, (self.H, self.V) if self.trans else (self.V, self.H))
        kx = K.KnetArray(self.x.reshape(-1), (self.H, self.N))
        return kw, kx, None if self.b is None else K.KnetArray(self.b, (self.V,))

    def matrix(self, dw):
        """a gradient of w, in w's layout, as (V, H)"""
        return dw.data.view(self.V, self.H) if self.trans else dw.data.view(self.H, self.V).t()

    def solve(self, average=True, dy=1.0):
        u, V, H, N = U[self.dtype], self.V, self.H, self.N
        w, x = self.w.double(), self.x.double()
        b = torch.zeros(V, device="cuda", dtype=torch.float64) if self.b is None else self.b.double()
        s = x @ w.t() + b                                                              # (N, V)
        fin = torch.where(torch.isfinite(b), b.abs(), torch.zeros_like(b))
        ds = gamma(H, u) * (x.abs() @ w.abs().t()) + 2 * u * (torch.nan_to_num(s, neginf=0.0).abs() + fin)
        lse = torch.logsumexp(s, 1)
        ds = torch.where(torch.exp(s - lse.unsqueeze(1)) > 0, ds, torch.zeros_like(ds))     # no share, no influence
        dlse = ds.max(1).values + (V / 64 + 40) * 2 * u
        used = self.labels != 0
        at = (self.labels.long() - 1).clamp_min(0).unsqueeze(1)
        per = torch.where(used, lse - s.gather(1, at).squeeze(1), torch.zeros_like(lse))
        dper = torch.where(used, dlse + ds.gather(1, at).squeeze(1) + 2 * u * per.abs(), torch.zeros_like(lse))
        self.lse, self.dlse = lse, dlse + 2 * u * lse.abs()
        self.per, self.dper = per, dper
        self.total, self.dtotal = float(per.sum()), float(dper.sum()) + 2 * u * float(per.abs().sum())
        self.count = int(used.sum())
        p = torch.exp(s - lse.unsqueeze(1))
        e = p * (torch.expm1(ds + dlse.unsqueeze(1) + 8 * u) + 8 * u) + 2 * u * p + self.ds_step
        p.scatter_add_(1, at, torch.full_like(lse, -1.0).unsqueeze(1))
        e.scatter_add_(1, at, torch.full_like(lse, 2 * u).unsqueeze(1))
        f = used.double().unsqueeze(1) * ((dy / self.count if self.count else 0.0) if average else dy)
        p, e = p * f, torch.where(f == 0, torch.zeros_like(e), e * f.abs() + 4 * u * (p * f).abs())     # skipped: exactly 0
        self.p, self.top = p, 1 + float(torch.nan_to_num(s, neginf=0.0).abs().max())
        self.dx, self.ddx = p @ w, e @ w.abs() + gamma(V, u) * (p.abs() @ w.abs())
        self.dw, self.ddw = p.t() @ x, e.t() @ x.abs() + gamma(N, u) * (p.abs().t() @ x.abs())
        self.db, self.ddb = p.sum(0), e.sum(0) + gamma(N, u) * p.abs().sum(0)
        return self


def within(got, want, bound, what):
    got = got.double()
    bad = ~((got - want).abs() <= bound + 1e-300)
    assert not bool(bad.any()), (what, int(bad.sum()), float((got - want).abs().max()), float(bound.max()))


def check(K, c, average=True, dy=1.0):
    kw, kx, kb = c.arrays(K)
    res = K.ops.linear_nll_device(kw, kx, c.labels, b=kb, trans=c.trans)
    dw, dx, db = K.ops.linear_nll_back(kw, kx, res, b=kb, trans=c.trans, average=average, dy=dy)
    c.solve(average, dy)
    assert int(res.count.item()) == c.count
    within(res.lse, c.lse, c.dlse, "lse")
    within(res.per_instance[:c.N], c.per, c.dper, "per_instance")
    assert abs(float(res.total.item()) - c.total) <= c.dtotal
    within(dx.data.view(c.N, c.H), c.dx, c.ddx, "dx")
    within(c.matrix(dw), c.dw, c.ddw, "dw")
    assert (db is None) == (kb is None)
    if db is not None:
        within(db.data, c.db, c.ddb, "db")
    return res, dw, dx, db


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_values_and_gradients(K, dtype, trans, shape):
    check(K, Case(*shape, dtype, trans, bias=shape[0] % 2 == 0, skip=shape[2] > 2))
    check(K, Case(*shape, dtype, trans, bias=shape[0] % 2 == 1, skip=False), average=False, dy=-0.75)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("trans", [False, True])
def test_several_pieces_of_the_vocabulary(K, trans, dtype):
    check(K, Case(9000, 96, 3000, dtype, trans, bias=True, skip=True))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_all_instances_skipped_and_none_at_all(K, dtype):
    c = Case(70, 20, 40, dtype, False, True, False)
    c.labels.zero_()
    res, dw, dx, db = check(K, c)
    assert float(res.total) == 0 and not dw.data.any() and not dx.data.any() and not db.data.any()
    kw, _, kb = c.arrays(K)
    none = K.KnetArray(torch.empty(0, dtype=dtype, device="cuda"), (20, 0))
    res = K.ops.linear_nll_device(kw, none, torch.empty(0, dtype=torch.int32, device="cuda"), b=kb)
    assert float(res.total) == 0 and int(res.count) == 0 and res.lse.numel() == 0
    dw, dx, db = K.ops.linear_nll_back(kw, none, res, b=kb)
    assert not dw.data.any() and not db.data.any() and len(dx) == 0


@pytest.mark.parametrize("shape", [(300, 40, 50), (1000, 128, 300), (1000, 256, 300), (5000, 100, 300), (300, 64, 8)], ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_masked_classes_and_bad_values(K, dtype, shape):
    """A bias of -inf takes a class out of every softmax; the type's lowest value does so too.  NaN or
    +inf in one instance stays in that instance's loss and dx."""
    c = Case(*shape, dtype, False, True, False)
    c.b[5:200] = -math.inf
    c.b[200] = torch.finfo(dtype).min
    c.labels.clamp_(1, 5)
    res, dw, dx, db = check(K, c)
    assert not c.matrix(dw)[5:201].any() and not db.data[5:201].any()
    c.labels[3] = 10                                                   # a masked label: infinite loss
    res = K.ops.linear_nll_device(*c.arrays(K)[:2], c.labels, b=c.arrays(K)[2])
    assert float(res.per_instance[3]) == math.inf and bool(torch.isfinite(res.per_instance[4:c.N]).all())
    c = Case(*shape, dtype, True, False, False)
    for bad in (math.nan, math.inf):
        c.x[7, 3] = bad
        kw, kx, _ = c.arrays(K)
        res = K.ops.linear_nll_device(kw, kx, c.labels, trans=True)
        dx = K.ops.linear_nll_back(kw, kx, res, trans=True)[1].data.view(c.N, c.H)
        ok = torch.ones(c.N, dtype=torch.bool, device="cuda")
        ok[7] = False
        assert bool(torch.isnan(res.per_instance[7])) and bool(torch.isnan(dx[7]).all())
        assert bool(torch.isfinite(res.per_instance[:c.N][ok]).all()) and bool(torch.isfinite(dx[ok]).all())
        c.labels[7] = 0                                                # skipped: its scores do not matter to the loss
        res = K.ops.linear_nll_device(kw, kx, c.labels, trans=True)
        assert bool(torch.isfinite(res.total))
        c.labels[7] = 1


@pytest.mark.parametrize("shape", [(300, 40, 50), (1000, 128, 300), (1000, 256, 300), (5000, 100, 300), (300, 64, 8)], ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_every_class_masked(K, dtype, shape):
    """Masked by the type's lowest value, the softmax is uniform and the loss log V, as the score
    matrix's logsoftmax gives; masked by -inf, NaN."""
    c = Case(*shape, dtype, False, True, False)
    c.b[:] = torch.finfo(dtype).min
    kw, kx, kb = c.arrays(K)
    res = K.ops.linear_nll_device(kw, kx, c.labels, b=kb)
    tol = 1e-6 if dtype == torch.float32 else 1e-14
    assert bool(((res.per_instance[:c.N] - math.log(c.V)).abs() <= tol * math.log(c.V)).all())
    db = K.ops.linear_nll_back(kw, kx, res, b=kb)[2].data.double()
    want = 1.0 / c.V - torch.bincount(c.labels.long() - 1, minlength=c.V).double() / c.N
    assert bool(((db - want).abs() <= (16 * c.N + 32) * 2 * U[dtype] * (1.0 / c.V + want.abs())).all())
    c.b[:] = -math.inf
    res = K.ops.linear_nll_device(kw, kx, c.labels, b=K.KnetArray(c.b, (c.V,)))
    assert bool(torch.isnan(res.per_instance[:c.N]).all())


def test_labels_out_of_range_make_the_loss_nan(K):
    for bad in (-1, 301, 2 ** 31 - 1):
        c = Case(300, 40, 50, torch.float32, False, False, False)
        c.labels[9] = bad
        kw, kx, _ = c.arrays(K)
        res = K.ops.linear_nll_device(kw, kx, c.labels)
        assert math.isnan(float(res.total)) and math.isnan(float(res.per_instance[9]))
        assert bool(torch.isfinite(res.per_instance[:9]).all())
        for g in K.ops.linear_nll_back(kw, kx, res)[:2]:
            assert bool(torch.isfinite(g.data).all())


@pytest.mark.parametrize("scale", [2.0 ** -70, 2.0 ** 60])
@pytest.mark.parametrize("shape", [(300, 40, 50), (1000, 256, 300)], ids=str)
def test_magnitudes_far_from_one(K, scale, shape):
    """Weights of a tiny and inputs of a huge magnitude (and the reverse): the products are ordinary."""
    c = Case(*shape, torch.float32, True, False, True)
    c.w *= scale
    c.x /= scale
    check(K, c)


def test_rows_of_very_different_magnitude(K):
    """Classes whose weights lie 2^-12 below the others', features 2^-10 below: bounds as everywhere."""
    c = Case(1000, 256, 300, torch.float32, False, True, False)
    c.w[::3] *= 2.0 ** -12
    c.x[:, 5::7] *= 2.0 ** -10
    check(K, c)


@pytest.mark.parametrize("off", [1, 3])
@pytest.mark.parametrize("shape", [(300, 40, 50), (1001, 130, 301), (1001, 260, 301), (1000, 256, 320), (2500, 100, 5)], ids=str)
def test_views_with_odd_offsets_and_guards(K, off, shape):
    """Operands and outputs that start `off` elements past an aligned address; what lies beside the
    outputs stays as it was."""
    c = Case(*shape, torch.float32, False, True, True)
    kw, kx, kb = c.arrays(K)

    def shifted(a):
        big = torch.full((len(a) + 16,), 7.0, device="cuda")
        big[off:off + len(a)] = a.data
        return big, K.KnetArray(big[off:off + len(a)], a.shape)

    (bw, sw), (bx, sx), (bb, sb) = (shifted(a) for a in (kw, kx, kb))
    (ow, gw), (ox, gx), (ob, gb) = (shifted(a) for a in (kw, kx, kb))
    ref = K.ops.linear_nll_device(kw, kx, c.labels, b=kb)
    res = K.ops.linear_nll_device(sw, sx, c.labels, b=sb)
    want = K.ops.linear_nll_back(kw, kx, ref, b=kb)
    got = K.ops.linear_nll_back(sw, sx, res, b=sb, out=(gw, gx, gb))
    for g, view, buf in zip(got, (gw, gx, gb), (ow, ox, ob)):
        assert g is view and bool((buf[:off] == 7).all()) and bool((buf[off + len(g):] == 7).all())
    if c.N > 32:                # the same order of additions at any alignment
        assert torch.equal(res.lse, ref.lse) and torch.equal(res.total, ref.total)
        assert all(torch.equal(w.data, g.data) for w, g in zip(want, got))
    c.solve()                   # few instances: aligned rows are added in packs of four, so within the bounds of any order
    within(res.lse, c.lse, c.dlse, "lse")
    within(c.matrix(gw), c.dw, c.ddw, "dw")
    within(gx.data.view(c.N, c.H), c.dx, c.ddx, "dx")
    within(gb.data, c.db, c.ddb, "db")


def test_need_leaves_gradients_out(K):
    c = Case(300, 40, 50, torch.float32, False, True, True)
    kw, kx, kb = c.arrays(K)
    res = K.ops.linear_nll_device(kw, kx, c.labels, b=kb)
    full = K.ops.linear_nll_back(kw, kx, res, b=kb)
    for k in range(3):
        need = tuple(i == k for i in range(3))
        part = K.ops.linear_nll_back(kw, kx, res, b=kb, need=need)
        for i in range(3):
            assert (part[i] is None) if i != k else torch.equal(part[i].data, full[i].data)
    assert K.ops.linear_nll_back(kw, kx, res, need=(False, False, True)) == (None, None, None)


def test_repeated_and_captured_and_two_streams(K):
    """Same bits on every run; a captured pass replays on new inputs; two streams at once."""
    cs = [Case(1000, 256, 300, torch.float32, True, True, True, seed=s) for s in (1, 2)]

    def step(c):
        kw, kx, kb = c.arrays(K)
        res = K.ops.linear_nll_device(kw, kx, c.labels, b=kb, trans=True)
        dw, dx, db = K.ops.linear_nll_back(kw, kx, res, b=kb, trans=True)
        return [res.total, res.lse, dw.data, dx.data, db.data]

    want = [[t.clone() for t in step(c)] for c in cs]
    for c, w in zip(cs, want):
        assert all(torch.equal(a, b) for a, b in zip(step(c), w))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [None, None]
    for _ in range(3):
        for k in (0, 1):
            with torch.cuda.stream(streams[k]):
                got[k] = step(cs[k])
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(g, w))
    box = Case(1000, 256, 300, torch.float32, True, True, True, seed=1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(box)
    for k in (1, 0, 1):
        for name in ("w", "x", "b", "labels"):
            getattr(box, name).copy_(getattr(cs[k], name))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[k]))


def test_agrees_with_the_composed_loss(K):
    """nll(w*x .+ b, labels) through the score matrix, and its gradients through the tape."""
    c = Case(500, 96, 64, torch.float64, False, True, True)
    kw, kx, kb = c.arrays(K)
    A = K.autograd
    grads = []
    for fused in (True, False):
        p, q, r = A.Param(kw.copy()), A.Param(kx.copy()), A.Param(kb.copy())
        f = (lambda: A.linear_nll(p, q, c.labels, r)) if fused else (lambda: A.nll(p @ q + r, c.labels))
        t = A.diff(f)
        grads.append([float(t.value().data.item())] + [v.grad.numpy() for v in (p, q, r)])
    for a, b in zip(*grads):
        np.testing.assert_allclose(a, b, rtol=1e-11, atol=1e-13)
    assert abs(K.linear_nll(kw, kx, c.labels, kb) - grads[0][0]) < 1e-12
    tot, cnt = K.linear_nll(kw, kx, c.labels, kb, average=False)
    assert abs(tot / cnt - grads[0][0]) < 1e-12


@pytest.mark.parametrize("trans", [False, True])
def test_gradients_against_differences(K, trans):
    A = K.autograd
    c = Case(30, 7, 11, torch.float64, trans, True, True)
    kw, kx, kb = c.arrays(K)
    for k, f in enumerate([lambda v: A.linear_nll(v, kx, c.labels, kb, trans), lambda v: A.linear_nll(kw, v, c.labels, kb, trans),
                           lambda v: A.linear_nll(kw, kx, c.labels, v, trans, average=False)]):
        assert A.gradcheck(f, (kw, kx, kb)[k].numpy())
    # gradients of gradients
    for k, f in enumerate([lambda v: A.linear_nll(v, kx, c.labels, kb, trans), lambda v: A.linear_nll(kw, v, c.labels, kb, trans)]):
        assert A.gradcheck(A.gradfun(f), (kw, kx)[k].numpy(), nsample=6)


def test_refusals(K):
    c = Case(30, 8, 11, torch.float32, False, True, False)
    kw, kx, kb = c.arrays(K)
    z = K.KnetArray
    for bad in (lambda: K.ops.linear_nll_device(kw, kx, c.labels, trans=True),                       # 30 features against 8
                lambda: K.ops.linear_nll_device(kw, kx, c.labels[:5]),
                lambda: K.ops.linear_nll_device(kw, kx, c.labels, b=z.zeros(29)),
                lambda: K.ops.linear_nll_device(kw.vec(), kx, c.labels)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        K.ops.linear_nll_device(kw, z.zeros((8, 11), torch.float64), c.labels)
    with pytest.raises(TypeError):
        K.ops.linear_nll_device(z(kw.data.half(), (30, 8)), z(kx.data.half(), (8, 11)), c.labels)
    res = K.ops.linear_nll_device(kw, kx, c.labels, b=kb)
    with pytest.raises(ValueError):
        K.ops.linear_nll_back(kw, z.zeros((8, 12)), res)
    with pytest.raises(ValueError):
        K.ops.linear_nll_back(kw, kx, res, out=(z.zeros((30, 9)), None, None))


# every form: few instances; FMA and FP64 tiles, the sum of dW whole and cut; tensor-core tiles, sums cut and whole;
# Float64 pieces
@pytest.mark.parametrize("shape", [(300, 64, 8), (300, 40, 50), (1000, 784, 400), (40, 70, 5000), (1000, 256, 300), (5000, 100, 3000),
                                   (9000, 96, 2100)], ids=str)
@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_skipped_instances_may_hold_anything(K, dtype, trans, shape):
    """What a padded batch has in a skipped instance changes no bit of the loss, the gradients or the used
    instances' lse."""
    c = Case(*shape, dtype, trans, True, True)
    skip = c.labels == 0

    def run():
        kw, kx, kb = c.arrays(K)
        res = K.ops.linear_nll_device(kw, kx, c.labels, b=kb, trans=trans)
        dw, dx, db = K.ops.linear_nll_back(kw, kx, res, b=kb, trans=trans)
        assert not dx.data.view(c.N, c.H)[skip].any()
        return [res.total, res.per_instance[:c.N], res.lse[~skip], dw.data, dx.data, db.data]

    c.x[skip] = 0
    want = run()
    for bad in (math.nan, math.inf, -math.inf, 1e30, torch.finfo(dtype).min):
        c.x[skip] = bad
        assert all(torch.equal(a, b) for a, b in zip(run(), want)), bad


@pytest.mark.parametrize("shape", [(10, 5, 20000), (33, 7, 30001), (70, 3, 150000), (300, 2, 70000)], ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_bias_gradient_over_many_instances(K, dtype, shape):
    check(K, Case(*shape, dtype, False, True, True))


@pytest.mark.parametrize("shape", [(4194240, 2, 5), (600001, 1, 33), (2, 4194240, 3), (3, 1048577, 40), (4, 3, 4194240), (5, 2, 4194240)], ids=str)
@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_longest_axes(K, dtype, trans, shape):
    """Each axis at its largest, few and many scores.  With millions of classes probabilities lie below 2^-16, and
    the tensor-core form's own rounding of dS shows: p 2^14 is held as two fp16 numbers, whose second is a multiple
    of fp16's smallest number 2^-24 (p < 2^-13 makes it that small), so p is off by half of that over 2^14, 2^-39."""
    c = Case(*shape, dtype, trans, True, True)
    V, H, N = shape
    c.ds_step = 2.0 ** -39 if dtype == torch.float32 and (N * V > 2 ** 24 or V * H * N >= 2 ** 26) else 0.0
    res, dw, dx, db = check(K, c)
    # The worst order of millions of roundings says little, so also: they come with either sign, an error beyond
    # 16 standard deviations of the longest sum's, sqrt(n) 2u of its largest value, is not rounding.
    t = 16 * math.sqrt(max(shape)) * 2 * U[dtype] * c.top
    used = c.labels != 0
    assert float((res.lse.double() - c.lse)[used].abs().max() if bool(used.any()) else 0.0) <= t
    # c.p holds the softmax minus one-hot; at the label the error is that of the softmax, at most t (|p - 1| + 1)
    hot = torch.zeros_like(c.p).scatter_(1, (c.labels.long() - 1).clamp_min(0).unsqueeze(1), 1.0)
    x, w, p = c.x.double().abs(), c.w.double().abs(), (c.p.abs() + (hot + c.ds_step) / max(c.count, 1)) * used.unsqueeze(1)
    within(c.matrix(dw), c.dw, t * (p.t() @ x) + c.ds_step * x.sum(0), "dw")
    within(dx.data.view(N, H), c.dx, t * (p @ w) + c.ds_step * w.sum(0) * used.unsqueeze(1), "dx")
    within(db.data, c.db, t * p.sum(0) + c.ds_step, "db")
