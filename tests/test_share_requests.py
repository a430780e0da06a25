"""Requests that share what they begin with, without a GPU: what is refused, and how."""
import pytest

from scriptling_llm_lib_b200.engine.generate import plan_batches


@pytest.mark.parametrize("n", [1, 3])
def test_a_request_that_does_not_fit_is_refused_with_its_pages_and_tokens(n):
    with pytest.raises(ValueError, match=r"request 0 needs 4 cache pages \(209 tokens\); the cache has 3"):
        plan_batches([200] * n, 10, 8, 3, 1000, n=n)
    with pytest.raises(ValueError, match=r"request 0 needs 10 cache pages \(640 tokens\); the cache has 9"):
        plan_batches([5000] * n, 10, 8, 9, 640, n=n)
