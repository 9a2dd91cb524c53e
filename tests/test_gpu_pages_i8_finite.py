"""The cases of test_gpu_pages_i8.py once more, with a NaN in place of a finite output an error: max(worst, nan) there is worst, so
that a bound alone does not show one."""
import math

import pytest

import test_gpu_pages_i8 as cases

pytestmark = pytest.mark.gpu


def no_nan(*args, **kw):
    for x in args:
        assert not (isinstance(x, float) and math.isnan(x)), "NaN where the result is finite"
    return max(*args, **kw)


@pytest.fixture(autouse=True)
def strict(monkeypatch):
    monkeypatch.setattr(cases, "max", no_nan, raising=False)


def listed(test):
    return next(m.args[1] for m in test.pytestmark if m.name == "parametrize")


@pytest.mark.parametrize("case", listed(cases.test_decode))
def test_decode(ctx, nnhip, case):
    cases.check_decode(ctx, nnhip, **case)


@pytest.mark.parametrize("case", listed(cases.test_prompt) + listed(cases.test_prompt_few_queries))
def test_prompt(ctx, nnhip, case):
    cases.prompt_case(ctx, nnhip, **case)


def test_edges(ctx, nnhip):
    cases.test_decode_edges(ctx, nnhip)
    cases.test_prompt_edges(ctx, nnhip)
    cases.test_prompt_few_queries_edges(ctx, nnhip)


@pytest.mark.parametrize("cap", [0.0, 20.0])
@pytest.mark.parametrize("dk", [64, 128])
def test_whole_tiles_edges(ctx, nnhip, dk, cap):
    cases.test_prompt_whole_tiles_edges(ctx, nnhip, dk, cap)


def test_a_nan_is_seen():
    with pytest.raises(AssertionError):
        cases.max(0.0, float("nan"))
