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


def test_a_copy_that_fails_leaves_forks_and_writers_as_they_were(monkeypatch):
    """The copies' ids find no memory: no slot is taken, no page is held for nothing, and the writers hold the pages that they shared."""
    from test_share_cpu import _cache, _check, _consistent, _write
    c = _cache()
    a = c.open()
    _write(c, a, list(range(1, 151)))
    b, d = c.fork(a, 2)
    copy = c._copy

    def fails(*args, **kw):
        raise MemoryError("no memory")
    before = [(g.pool.n_held, g.pool.n_shared, {s: list(p) for s, p in g.pages.items()}, g.table.copy()) for g in c.groups]

    def unchanged():
        return all((g.pool.n_held, g.pool.n_shared, {s: list(p) for s, p in g.pages.items()}) == was[:3] and (g.table == was[3]).all()
                   for g, was in zip(c.groups, before))
    monkeypatch.setattr(c, "_copy", fails)
    with pytest.raises(MemoryError):
        c.fork(a, 3)
    assert c.slots.n_held == 3 and unchanged()
    for growth in ([(b, 1)], [(a, 2), (b, 1), (d, 70)]):
        with pytest.raises(MemoryError):
            c.reserve(growth)
        assert unchanged()
    monkeypatch.setattr(c, "_copy", copy)
    for s, t in ((a, 7), (b, 8), (d, 9)):
        _write(c, s, [t])
        _check(c, s, list(range(1, 151)) + [t])
    _consistent(c)
    for s in (a, b, d):
        c.close(s)
    assert all(g.pool.n_held == 0 for g in c.groups)
