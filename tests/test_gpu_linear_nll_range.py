"""linear_nll where magnitudes differ widely inside one call: every form holds the entries that an ordinary Float32
composition holds, whatever another instance, another class or a likelier class contains.  Bounds as in
test_gpu_linear_nll.py, whose inputs and evaluation in 64 bits are used."""
import math

import pytest
import torch

from test_gpu_linear_nll import Case, U, check, gamma, within

pytestmark = pytest.mark.gpu

# few instances; FMA tiles; tensor-core tiles with cut sums, with whole ones, with several pieces of the vocabulary
FORMS = [(300, 64, 8), (300, 40, 50), (1000, 256, 300), (1001, 260, 301), (3001, 515, 700), (9000, 96, 3000)]


@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("shape", FORMS, ids=str)
def test_classes_that_are_never_hit(K, trans, shape):
    """Two thirds of the classes have probabilities from 2^-24 down to 2^-90 of the others': their rows of dW and
    entries of db are as exact, relative to themselves, as those of any class (a score of the size of its bias
    rounds to 2u |b|, which the bound of its exponential has)."""
    c = Case(*shape, torch.float32, trans, True, True)
    for k, bits in enumerate((24, 36, 44, 60, 90)):
        c.b[c.V // 3 + k::8] -= bits * math.log(2.0)
    c.labels[c.labels != 0] = c.labels[c.labels != 0].clamp_max(c.V // 3)
    _, dw, _, db = check(K, c)
    for k in range(5):
        assert bool(c.matrix(dw)[c.V // 3 + k::8].any()) and bool((db.data[c.V // 3 + k::8] > 0).all())


class Wide(Case):
    """A Case whose instance `big` and class `masked` have values 2^k times the others'.  Instance `big` is 2^k times
    the weights of class `top`, whose score in it is then far above any other; class `masked` has the score -4 * 2^k
    in every instance, of which its remaining weights move a tenth.  Their shares of the softmax are exactly 1 and 0
    and do not feel the rounding of those scores.

    Tensor-core forms hold a row of an operand in two fp16 terms, the second a multiple of 2^-24 where the row's
    largest entry lies in [2^14, 2^15): an entry is off by 2^-25 / 2^14 = 2^-39 of the power of two m at or below that
    largest one, which is all that tells for entries below 2^-16 m (class `masked` has some, labelled in instance 1).
    So a term p w of dx is off by 2^-39 |p| m(w) and, as p m(w) / m with m that of the instance's largest |p| m(w),
    by 2^-39 m |w| / m(w) <= 2^-38 max(|p| |w|max) |w| / |w|max; terms of dW likewise."""

    def __init__(self, V, H, N, trans, bias, k):
        super().__init__(V, H, N, torch.float32, trans, bias, True)
        self.big, self.masked, self.top = N // 2, V // 2, 3
        s = 2.0 ** k
        self.x[:, 1] = 1.0
        self.w[self.masked] *= s * 0.05
        self.w[self.masked, 1] = -4.0 * s
        self.w[self.top, 1] = 1.0                                     # so that the two meet with the score -4 * 4^k
        self.x[self.big] = self.w[self.top] * s
        self.labels[self.big] = 1
        self.labels[self.labels == self.masked + 1] = 1
        self.labels[1] = self.masked + 1                              # one instance is labelled with it: a loss of about 4 * 2^k

    def solve(self):
        u, V, H, N = U[self.dtype], self.V, self.H, self.N
        w, x = self.w.double(), self.x.double()
        b = torch.zeros(V, device="cuda", dtype=torch.float64) if self.b is None else self.b.double()
        s = x @ w.t() + b
        ds = gamma(H, u) * (x.abs() @ w.abs().t()) + 2 * u * (s.abs() + b.abs())
        lse = torch.logsumexp(s, 1)
        p = torch.exp(s - lse.unsqueeze(1))
        sure = (p == 0) | (p == 1)                                     # beyond any rounding, as is checked here:
        gap = (s - s.max(1, keepdim=True).values).abs()
        alone = torch.zeros_like(sure)
        alone[self.big] = True
        alone[:, self.masked] = True
        assert bool(sure[alone].all())
        far = gap - ds - ds.gather(1, s.argmax(1, keepdim=True))
        assert bool((far[alone & (p == 0)] > 200).all())
        de = torch.where(alone, torch.zeros_like(ds), ds)              # what reaches the softmax
        dlse = de.max(1).values + (V / 64 + 40) * 2 * u
        used = self.labels != 0
        at = (self.labels.long() - 1).clamp_min(0).unsqueeze(1)
        top = ds.gather(1, s.argmax(1, keepdim=True)).squeeze(1)
        per = torch.where(used, lse - s.gather(1, at).squeeze(1), torch.zeros_like(lse))
        self.lse, self.dlse = lse, dlse + torch.maximum(top, dlse) + 2 * u * lse.abs()
        self.per, self.dper = per, torch.where(used, self.dlse + ds.gather(1, at).squeeze(1) + 2 * u * per.abs(), torch.zeros_like(lse))
        e = p * (torch.expm1(de + dlse.unsqueeze(1) + 8 * u) + 8 * u) + 2 * u * p
        p = p.scatter_add(1, at, torch.full_like(lse, -1.0).unsqueeze(1))
        e = e.scatter_add(1, at, torch.full_like(lse, 2 * u).unsqueeze(1))
        f = used.double().unsqueeze(1) / int(used.sum())
        p, e = p * f, e * f + 4 * u * (p * f).abs()
        self.p = p
        self.dx, self.ddx = p @ w, e @ w.abs() + gamma(V, u) * (p.abs() @ w.abs())
        self.dw, self.ddw = p.t() @ x, e.t() @ x.abs() + gamma(N, u) * (p.abs().t() @ x.abs())
        self.db, self.ddb = p.sum(0), e.sum(0) + gamma(N, u) * p.abs().sum(0)
        if V * H * N >= 2 ** 26 or V * N > 2 ** 24:
            wm, xm, q = w.abs().max(1, keepdim=True).values, x.abs().max(1, keepdim=True).values, p.abs()
            self.ddx += 2.0 ** -39 * (q @ wm) + 2.0 ** -38 * (q * wm.t()).max(1, keepdim=True).values * (w.abs() / wm).sum(0)
            self.ddw += 2.0 ** -39 * (q.t() @ xm) + 2.0 ** -38 * (q * xm).max(0).values.unsqueeze(1) * (x.abs() / xm).sum(0)
        return self


# the last two: weights that the forward splits at once and the backward in two pieces, with sums cut for want of tiles.
# A score of 2^22 rounds to 1/4: the backward's has to be the forward's bit for bit, or its exponential is not 1.
@pytest.mark.parametrize("k", [20, 40, 60])
@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("shape", FORMS + [(5830, 9093, 60), (800, 50496, 40)], ids=str)
def test_one_instance_and_one_class_far_above_the_others(K, trans, shape, k):
    """A finite outlier reaches its own instance or class only: the losses, lse, dx of the other instances and dW, db
    of the other classes are as exact as without it."""
    c = Wide(*shape, trans, shape[0] % 2 == 0, k).solve()
    kw, kx, kb = c.arrays(K)
    res = K.ops.linear_nll_device(kw, kx, c.labels, b=kb, trans=trans)
    dw, dx, db = K.ops.linear_nll_back(kw, kx, res, b=kb, trans=trans)
    within(res.lse, c.lse, c.dlse, "lse")
    within(res.per_instance[:c.N], c.per, c.dper, "per_instance")
    others = torch.ones(c.N, dtype=torch.bool, device="cuda")
    others[[c.big, 1]] = False
    loss = res.per_instance[:c.N].double()
    assert float((loss - c.per)[others].abs().max()) < 1e-2
    within(dx.data.view(c.N, c.H), c.dx, c.ddx, "dx")
    within(c.matrix(dw), c.dw, c.ddw, "dw")
    if db is not None:
        within(db.data, c.db, c.ddb, "db")


@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("shape", [(1000, 256, 300), (3001, 515, 700), (1000, 2100, 300), (2000, 9000, 130)], ids=str)
def test_magnitudes_of_every_size(K, trans, shape):
    """Each instance and each class with a power of two of its own: instances from 2^-39 to 2, classes from 2^-30
    to 4."""
    c = Case(*shape, torch.float32, trans, True, True)
    c.w *= 2.0 ** -torch.arange(c.V, device="cuda").remainder(33).sub(2).float().unsqueeze(1)
    c.x *= 2.0 ** -torch.arange(c.N, device="cuda").remainder(41).sub(1).float().unsqueeze(1)
    check(K, c)


@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("scales", [(2.0 ** 100, 2.0 ** -110), (2.0 ** -100, 2.0 ** 110), (2.0 ** -120, 2.0 ** 100), (2.0 ** 124, 2.0 ** -126)],
                         ids=str)
def test_magnitudes_at_the_ends_of_the_type(K, trans, scales):
    """Scores far below the type's largest value from operands close to it and to its smallest."""
    c = Case(1000, 256, 300, torch.float32, trans, False, True, std=0.5)
    c.w *= scales[0]
    c.x *= scales[1]
    kw, kx, _ = c.arrays(K)
    res = K.ops.linear_nll_device(kw, kx, c.labels, trans=trans)
    c.solve()
    within(res.lse, c.lse, c.dlse, "lse")
    within(res.per_instance[:c.N], c.per, c.dper, "per_instance")


@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("shape", [(1000, 1024, 300), (3001, 2048, 700), (20000, 256, 2000)], ids=str)
def test_terms_of_one_sign(K, trans, shape):
    """Operands without negative entries, as after relu: every truncated addition of the tensor core then errs in
    the same direction.  An accumulator takes 8 blocks of 32 summed indices, 3 products of 2 steps each, so at most 48
    additions that each lose less than 2^-23 of the sum, of which the epilogue gives back 6 * 2^-23; what the split
    leaves out is 3 * 2^-22 and the additions of chunks in Float32 lose n / 256 times 2^-24: below 2^-17 of the
    sum, far inside gamma(n) from n = 256 on.  The scores here are shifted so that the softmax is not one-hot."""
    c = Case(*shape, torch.float32, trans, True, True)
    c.w.abs_()
    c.x.abs_()
    c.w *= 0.25
    res, dw, dx, db = check(K, c)
    # lse within 2^-17 of the scores' size, the gradients within that of the sums of absolute values and
    # what the error of the scores, at most 2 * 2^-17 of them, does to the probabilities
    t = 2.0 ** -17
    top = float((c.x.double() @ c.w.double().t()).max()) + float(c.b.abs().max())
    used = c.labels != 0
    assert float((res.lse.double() - c.lse)[used].abs().max()) <= t * top
    hot = torch.zeros_like(c.p).scatter_(1, (c.labels.long() - 1).clamp_min(0).unsqueeze(1), 1.0 / c.count) * used.unsqueeze(1)
    p = c.p.abs() + hot
    within(c.matrix(dw), c.dw, t * (2 * top + 2) * (p.t() @ c.x.double()), "dw")
    within(dx.data.view(c.N, c.H), c.dx, t * (2 * top + 2) * (p @ c.w.double()), "dx")


@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("shape", [(1, 8192, 8192), (3001, 515, 700), (9000, 96, 3000), (2000, 4096, 500)], ids=str)
def test_roundings_of_either_sign_mostly_cancel(K, trans, shape):
    """The worst order of n roundings would hide the loss of a few of an operand's bits.  Of a product's terms t each
    is off by less than 3 * 2^-23 |t| (the two splits and the product of the second terms), with either sign; an accumulator's 48
    truncated additions, their mean made up for, by 2^-23 (48 / 12)^0.5 of a partial sum each in the mean square,
    a partial sum being about |t|_2, the root of the sum of squares: about 2^-21.5 |t|_2 together.  Beyond 8 of those
    standard deviations, 2^-18.5 |t|_2, is not rounding.  To the gradients adds what the probabilities' own error
    does, a common factor per instance: as much as the scores' and lse's error together, with the sign of one."""
    c = Case(*shape, torch.float32, trans, False, True, std=1.0)
    kw, kx, _ = c.arrays(K)
    res = K.ops.linear_nll_device(kw, kx, c.labels, trans=trans)
    dw, dx, _ = K.ops.linear_nll_back(kw, kx, res, trans=trans)
    c.solve()
    t = 2.0 ** -18.5
    w, x, p = c.w.double(), c.x.double(), c.p
    score = t * ((x * x) @ (w * w).t()).sqrt() + 2.0 ** -24 * (x @ w.t()).abs()
    if c.V == 1:                                                       # lse is the score
        within(res.lse, c.lse, score[:, 0] + 2.0 ** -24, "lse")
        return
    ds = 2 * float(score.max()) + 2.0 ** -21                           # exponential, logarithm, lse's own rounding
    within(res.lse, c.lse, torch.full_like(c.lse, ds), "lse")
    hot = torch.zeros_like(p).scatter_(1, (c.labels.long() - 1).clamp_min(0).unsqueeze(1), 1.0 / c.count) * (c.labels != 0).unsqueeze(1)
    soft = p + hot
    within(dx.data.view(c.N, c.H), c.dx, t * ((p * p) @ (w * w)).sqrt() + ds * (soft @ w.abs()), "dx")
    within(c.matrix(dw), c.dw, t * ((p * p).t() @ (x * x)).sqrt() + ds * (soft.t() @ x.abs()), "dw")


@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("shape", [(1001, 260, 301), (9000, 96, 3000)], ids=str)
def test_gradients_one_at_a_time(K, trans, shape):
    """dS is split for dx and for dW only where they are asked for; either alone has the bits that it has with the
    others."""
    c = Case(*shape, torch.float32, trans, True, True)
    kw, kx, kb = c.arrays(K)
    res = K.ops.linear_nll_device(kw, kx, c.labels, b=kb, trans=trans)
    full = K.ops.linear_nll_back(kw, kx, res, b=kb, trans=trans)
    for k in range(3):
        part = K.ops.linear_nll_back(kw, kx, res, b=kb, trans=trans, need=tuple(i == k for i in range(3)))
        assert [g is None for g in part] == [i != k for i in range(3)] and torch.equal(part[k].data, full[k].data)


@pytest.mark.parametrize("shape", [(1000, 256, 300), (5001, 700, 400)], ids=str)
def test_weights_in_columns_captured_and_on_two_streams(K, shape):
    """The clusters that split W by columns, replayed on new inputs and side by side."""
    cs = [Case(*shape, torch.float32, False, True, True, seed=s) for s in (1, 2)]
    held = [c.arrays(K) for c in cs]

    def step(c, arrays):
        res = K.ops.linear_nll_device(*arrays[:2], c.labels, b=arrays[2])
        return [res.total, res.lse] + [g.data for g in K.ops.linear_nll_back(*arrays[:2], res, b=arrays[2])]

    want = [[t.clone() for t in step(c, a)] for c, a in zip(cs, held)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [None, None]
    for _ in range(4):
        for k in (0, 1):
            with torch.cuda.stream(streams[k]):
                got[k] = step(cs[k], held[k])
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(g, w))
    box = Case(*shape, torch.float32, False, True, True, seed=1)
    arrays = box.arrays(K)
    graphs, outs = [], []
    for _ in range(2):                                                 # two graphs of one set of inputs
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step(box, arrays))
    for k, g in ((1, 0), (0, 1), (1, 1), (0, 0)):
        for to, of in zip(arrays, held[k]):
            to.data.copy_(of.data)
        box.labels.copy_(cs[k].labels)
        graphs[g].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs[g], want[k]))


@pytest.mark.parametrize("off", [0, 1])
@pytest.mark.parametrize("shape", [(1000, 256, 300), (1001, 260, 301), (3000, 2000, 300), (2501, 1100, 200), (9000, 96, 3000)], ids=str)
def test_maxima_handed_to_the_backward_or_not(K, shape, off):
    """With W's maxima from the forward the backward reads W once, without them it finds them again: the same bits, at
    any alignment of W."""
    c = Case(*shape, torch.float32, False, True, True)
    kw, kx, kb = c.arrays(K)
    big = torch.zeros(len(kw) + 4, device="cuda")
    big[off:off + len(kw)] = kw.data
    kw = K.KnetArray(big[off:off + len(kw)], kw.shape)
    res = K.ops.linear_nll_device(kw, kx, c.labels, b=kb)
    top = c.w.abs().max(1).values
    assert torch.equal(res.class_max, top)
    got = [g.data.clone() for g in K.ops.linear_nll_back(kw, kx, res, b=kb)]
    assert torch.equal(res.class_max, top)                             # read, not written
    res.class_max = None
    assert all(torch.equal(g, h.data) for g, h in zip(got, K.ops.linear_nll_back(kw, kx, res, b=kb)))
    c.solve()
    within(c.matrix(K.KnetArray(got[0], kw.shape)), c.dw, c.ddw, "dw")
    within(got[1].view(c.N, c.H), c.dx, c.ddx, "dx")


@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("shape", [(70000, 1, 1000), (40000, 3, 700), (3000, 73, 400), (2000, 300, 200), (700, 700, 200), (1000, 1352, 100),
                                   (301, 2049, 150), (300, 5169, 60), (33, 9001, 250)], ids=str)
def test_rows_of_every_length_and_alignment(K, trans, shape):
    """W and x that start 0 to 3 values past a 16-byte word, with NaN just before and behind them: each row has its own
    offset in a word, and what lies beside an array is not read into it."""
    c = Case(*shape, torch.float32, trans, True, True)
    kw, kx, kb = c.arrays(K)
    res = K.ops.linear_nll_device(kw, kx, c.labels, b=kb, trans=trans)
    want = [res.total, res.lse] + [g.data for g in K.ops.linear_nll_back(kw, kx, res, b=kb, trans=trans)]
    c.solve()
    within(res.lse, c.lse, c.dlse, "lse")
    within(c.matrix(K.KnetArray(want[2], kw.shape)), c.dw, c.ddw, "dw")
    within(want[3].view(c.N, c.H), c.dx, c.ddx, "dx")
    for off in (1, 2, 3):
        views = []
        for a in (kw, kx):
            buf = torch.full((len(a) + 16,), float("nan"), device="cuda")
            buf[4 + off:4 + off + len(a)] = a.data
            views.append(K.KnetArray(buf[4 + off:4 + off + len(a)], a.shape))
        res = K.ops.linear_nll_device(*views, c.labels, b=kb, trans=trans)
        got = [res.total, res.lse] + [g.data for g in K.ops.linear_nll_back(*views, res, b=kb, trans=trans)]
        assert all(torch.equal(g, w) for g, w in zip(got, want)), off
