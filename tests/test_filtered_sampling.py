"""Filters of a draw: what a request may ask, and the restatement the kernel is tested against."""
import numpy as np
import pytest

import plain_operators as plain
from lucciola_b200 import SamplingParams


@pytest.mark.parametrize("bad", [dict(top_k=-1), dict(top_k=2 ** 31), dict(top_p=0.0), dict(top_p=1.5), dict(top_p=float("nan")), dict(min_p=-0.1),
                                 dict(min_p=1.01), dict(min_p=float("nan"))])
def test_parameters_out_of_range_are_refused(bad):
    with pytest.raises(ValueError):
        SamplingParams(temperature=1.0, **bad).validate()


def test_parameters_in_range():
    for ok in (dict(), dict(top_k=5), dict(top_p=1.0), dict(top_p=1e-6), dict(min_p=1.0)):
        SamplingParams(temperature=1.0, **ok).validate()
    assert not SamplingParams(temperature=0.0, top_k=5).filtered           # greedy
    assert not SamplingParams(temperature=1.0).filtered
    assert SamplingParams(temperature=1.0, min_p=0.1).filtered


def test_kept_tokens_by_hand():
    x = np.log(np.array([0.1, 0.4, 0.2, 0.2, 0.1]))
    assert plain.kept_tokens(x, 1.0, 0, 1.0, 0.0).tolist() == [1, 2, 3, 0, 4]
    assert plain.kept_tokens(x, 1.0, 3, 1.0, 0.0).tolist() == [1, 2, 3]
    assert plain.kept_tokens(x, 1.0, 0, 0.5, 0.0).tolist() == [1, 2]
    assert plain.kept_tokens(x, 1.0, 3, 0.49, 0.0).tolist() == [1]            # 0.4 of the 0.8 that three tokens make up is more than 0.49
    assert plain.kept_tokens(x, 1.0, 0, 1.0, 0.4).tolist() == [1, 2, 3]
    assert plain.kept_tokens(x, 1.0, 0, 1e-9, 1.0).tolist() == [1]


def test_numbers_are_those_of_the_other_restatement():
    import plain_qwen3
    u = plain.uniforms(0x1234567890ABCDEF, 7, 50)
    assert [float(plain_qwen3.hash_uniform(0x1234567890ABCDEF, 7, i)) for i in range(50)] == u.tolist()
