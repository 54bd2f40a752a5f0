"""losses.distill_top of a teacher's values that are no log probabilities: their rows are NaN throughout, the others as they
would be without them."""
from __future__ import annotations

from importlib import import_module

import pytest

from conftest import gpu_case
from test_gpu_losses import INF, NAN, TYPES, check_distill, rows_of, teacher_of

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,V", [(12, 3000), (12, 70001), (300, 3000)])
@pytest.mark.parametrize("rest", [True, False])
def test_values_that_are_not_finite(pkg, dtype, R, V, rest):
    losses = import_module(pkg.__name__ + ".losses")
    x, _ = rows_of(R, V, dtype, V, 1, 1)
    ids, v, w = teacher_of(x, 6, V)
    w = w + 0.1
    v[1, 0], v[2, 3], v[4, 5] = INF, NAN, INF
    v[5, 1], ids[5, 1] = INF, -1                                     # (none, with its value)
    bad = [1, 2, 4]
    if rest:
        v[6, 2] = 100.0                                              # (e^100 is past float32)
        bad.append(6)
    gpu_case(f"distill {dtype} R={R} V={V} rest={rest} with values that are not finite")
    loss, grad = losses.distill_top_grad(x, ids, v, w, rest=rest)
    torch.cuda.synchronize()
    assert loss[bad].isnan().all() and grad[bad].isnan().all()
    fine = [r for r in range(R) if r not in bad + [5]]
    check_distill(loss[fine], grad[fine], x[fine], ids[fine], v[fine], w[fine], rest)
    keep = [0, 2, 3, 4, 5]
    check_distill(loss[5:6], grad[5:6], x[5:6], ids[5:6, keep], v[5:6, keep], w[5:6], rest)
