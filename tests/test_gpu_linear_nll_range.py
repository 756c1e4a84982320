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
