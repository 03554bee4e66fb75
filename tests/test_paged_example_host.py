"""Host side of examples/paged_batch.py: requests that cannot be served are refused before any step or
page is taken."""
import importlib.util
import os
import types

import pytest

pytest.importorskip("torch")

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def batch(n_pages=24, page_size=16, max_positions=512):
    spec = importlib.util.spec_from_file_location("paged_batch_host", os.path.join(ROOT, "examples", "paged_batch.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)

    def step(*_):
        raise RuntimeError("a step")

    return m.Batch(types.SimpleNamespace(n_pages=n_pages, page_size=page_size, max_positions=max_positions, step=step,
                                         dev="cpu"), slots=4)


@pytest.mark.parametrize("request_,pool", [
    (([1] * 380, 20), {}),                    # more than all the pages hold
    (([1] * 500, 20), {"n_pages": 99}),       # more than there are positions
    (([], 5), {}), (([1, 2], 0), {}), (([1, 2], -3), {})])
def test_requests_that_do_not_fit_are_refused(request_, pool):
    b = batch(**pool)
    with pytest.raises(ValueError, match="request 7"):
        b.generate({3: ([1, 2, 3], 2), 7: request_})
    assert sorted(b.free) == list(range(b.model.n_pages)) and not (b.table >= 0).any() and b.run == [None] * 4


@pytest.mark.parametrize("request_", [([1] * 383, 1), ([1], 383)])
def test_requests_that_just_fit_are_taken_up(request_):
    with pytest.raises(RuntimeError, match="a step"):
        batch().generate({0: request_})
