"""Requests that share what they begin with, without a GPU: what is refused, and how."""
import pytest

from scriptling_llm_lib_b200.engine.generate import plan_batches


@pytest.mark.parametrize("n", [1, 3])
def test_a_request_that_does_not_fit_is_refused_with_its_pages_and_tokens(n):
    with pytest.raises(ValueError, match=r"request 0 needs 4 cache pages \(209 tokens\); the cache has 3"):
        plan_batches([200] * n, 10, 8, 3, 1000, n=n)
    with pytest.raises(ValueError, match=r"request 0 needs 10 cache pages \(640 tokens\); the cache has 9"):
        plan_batches([5000] * n, 10, 8, 9, 640, n=n)


def test_a_plan_knows_how_many_pages_its_layout_reaches():
    """Of the rows that it has, whatever else the table is wide, and after it has taken another layout."""
    import numpy as np
    from scriptling_llm_lib_b200.cache import PlanCapacity, SharePlan, TileShape
    table, shape = np.arange(60, dtype=np.int32).reshape(3, 20), TileShape(64, 10)
    table[1, :6] = table[0, :6]
    build = lambda held, new, **more: SharePlan.build(table, held, new, 4, 2, shape, None, **more)      # noqa: E731
    assert build([400, 500, 3], [1, 1, 1]).width == 8 and build([447, 448, 0], [1, 1, 1]).width == 8 and build([1000, 2, 3], [0, 1, 1]).width == 1
    assert build([400, 10, 0], [0, 0, 0]).width == 0 and build([0, 0, 0], [1280, 1, 0]).width == 20
    cap = PlanCapacity.of_decode(3, 4, 2, shape)
    plan = build([400, 500, 3], [1, 1, 1], capacity=cap)
    plan.again(build([400, 1000, 3], [1, 1, 1], capacity=cap))
    assert plan.width == 16
