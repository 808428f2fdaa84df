"""The paged decoding example: compressed weights, plan, rotary write and
attention together in a CUDA graph, against fp32 without a cache."""
import os
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    import paged_decode
    return paged_decode


# Each of the 2 layers rounds to bf16 (2^-9 rms at most of its value) some six
# times on the residual's way and the head once more; the errors are independent:
# sqrt(13) * 2^-9 < 0.8%, doubled for what the layers amplify.
TOL = 0.016


@pytest.mark.parametrize("top", [0, 64])
def test_paged_decode_matches_a_model_without_a_cache(example, top):
    """All pages, and a choice of 64 pages where no row has more."""
    model, history, logits = example.run(steps=24, top=top)
    ref = example.reference_logits(model, history)
    assert [len(h) for h in history] == [33 + 5 + 12, 120 + 24, 7 + 24]
    err = float((logits.float() - ref).norm() / ref.norm())
    assert err <= TOL, err


def test_paged_decode_sparse_runs(example):
    model, history, logits = example.run(steps=24, top=3)
    assert bool(logits.isfinite().all())
