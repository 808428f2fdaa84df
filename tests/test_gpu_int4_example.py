"""The decoding example over a 4-bit cache, and with sampling: plan, quantising write, read
back, attention over the codes and sampling together in a CUDA graph."""
import pytest
import torch

from test_gpu_paged_example import TOL, example  # noqa: F401

pytestmark = pytest.mark.gpu

# Beside the roundings that TOL counts, codes differ where they move a value across the middle
# of two codes: values are off by up to TOL of their size, a step is some 0.31 of it (a range
# of 4.7 in 15 steps), so one code in 30 is off by a step, an error of sqrt(1 / 30) 0.31 < 6%
# of a value's size. Scores (128 terms of q and k of size 1, times 128^-1/2) are off by as
# much, weights too, and outputs by both: 8.5% of the attention's, of which each of two
# independent layers adds at most all to the residual: 12%.
TOL4 = 0.12 + TOL


@pytest.mark.parametrize("settings", [dict(), dict(temperature=0.8, top_k=50, top_p=0.95)])
def test_a_4_bit_cache_matches_a_model_with_quantised_keys_and_values(example, settings):  # noqa: F811
    model, history, logits = example.run(steps=24, bits=4, **settings)
    ref = example.reference_logits(model, history, bits=4)
    err = (logits.float() - ref).norm(dim=-1) / ref.norm(dim=-1)
    assert bool((err <= TOL4).all()), err.tolist()


def test_sampled_tokens_are_the_logits_own(example):  # noqa: F811
    """Rows that sampling filled still match the model without a cache; another seed's random
    numbers give other tokens, top_k = 1 the largest logits' ones."""
    model, history, logits = example.run(steps=12, temperature=1.0)
    ref = example.reference_logits(model, history)
    assert float((logits.float() - ref).norm() / ref.norm()) <= TOL
    greedy = example.run(steps=12)[1]
    assert greedy != history
    assert example.run(steps=12, temperature=1.0, top_k=1)[1] == greedy
    assert example.run(steps=12, temperature=1.0)[1] == history


def test_pages_can_not_be_chosen_in_a_4_bit_cache(example):  # noqa: F811
    with pytest.raises(RuntimeError):
        example.run(steps=2, bits=4, top=3)
