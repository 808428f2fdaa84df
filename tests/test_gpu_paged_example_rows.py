"""The paged decoding example row by row: one wrong row among several shows."""
import pytest
import torch

from test_gpu_paged_example import TOL, example  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("top", [0, 64])
def test_each_row_matches_a_model_without_a_cache(example, top):  # noqa: F811
    """The rounding errors that the tolerance counts are independent from value to value, so a row's bound is the whole's."""
    model, history, logits = example.run(steps=24, top=top)
    ref = example.reference_logits(model, history)
    err = (logits.float() - ref).norm(dim=-1) / ref.norm(dim=-1)
    assert bool((err <= TOL).all()), err.tolist()
