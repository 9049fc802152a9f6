"""The few-token layer where one width is below a load's four columns and the other is not:
both projections then take the element-by-element path, over many column tiles."""

import pytest

from tests.test_gpu_few_tokens import TYPES, _check, _inputs

pytestmark = pytest.mark.gpu

SHAPES = [  # T, d, f, E, k
    (12, 3, 800, 4, 2), (64, 1, 1000, 4, 2), (40, 2, 64, 2, 1), (9, 700, 2, 3, 1), (20, 130, 3, 4, 2),
    (33, 65, 1, 8, 2), (5, 2, 130, 8, 3), (3, 3, 4096, 2, 1), (1, 1000, 1, 2, 1),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ffn", ["swiglu", "gelu"])
@pytest.mark.parametrize("T,d,f,E,k", SHAPES)
def test_one_narrow_width(ext, dtype, ffn, T, d, f, E, k):
    x, router, weights = _inputs(T, d, f, E, TYPES[dtype], ffn, T * d + f)
    _check(x, router, None, weights, k)
