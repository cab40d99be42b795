"""The forms of h3x_cross_sdpa_bf16 (keys cut into pieces or not, one or two query tiles per CTA, the kernel for any shape)
against the formula in 64 bits and against one another."""
import numpy as np
import pytest

from adapter_case import cross_reference, wide
from test_gpu_cross import Case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pkg():
    import __graft_entry__ as entry
    return entry.load_package()


@pytest.fixture(scope="module")
def gpu(pkg):
    g = pkg.Gpu(0)
    yield g
    g.close()


# ------------------------------------------------------------------ keys whose scores are all -inf

LOW, NAN, INF = 0xFF80, 0x7FC0, 0x7F80


def hopeless_keys(dim, keys, first, count, heads=4):
    """Positive queries; the keys [first, first + count) of one segment have a component of -inf, so that every score of
    theirs is -inf and every probability exactly 0."""
    case = Case([[0, 1, 0, keys]], heads, heads, dim)
    case.q &= 0x7FFF
    case.q[case.q == 0] = 0x3F80
    case.k.reshape(keys, heads, dim)[first:first + count, :, 0] = LOW
    return case


def results(gpu, case, monkeypatch):
    """Cut into pieces (one row of few heads over long states), and uncut (the kernel that walks all keys of a row)."""
    cut = wide(case.run(gpu, case.dim ** -0.5))
    monkeypatch.setenv("H3B_SDPA_SIMT", "1")
    whole = wide(case.run(gpu, case.dim ** -0.5))
    monkeypatch.delenv("H3B_SDPA_SIMT")
    return cut, whole


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("first,count", [(0, 2048), (1024, 1024), (0, 4096)])
@pytest.mark.parametrize("word", [NAN, INF])
def test_a_probability_of_zero_times_a_value_that_is_not_finite(gpu, monkeypatch, dim, first, count, word):
    """0 * inf and 0 * NaN are NaN in softmax(s) . v, wherever the keys of a segment are cut."""
    case = hopeless_keys(dim, 4096, first, count)
    case.v.reshape(4096, -1)[first:first + count, ::2] = word
    for name, got in zip(("cut", "whole"), results(gpu, case, monkeypatch)):
        assert np.isnan(got[::2]).all(), name
        assert np.isfinite(got[1::2]).all(), name


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("first,count", [(0, 2048), (1024, 1024), (0, 4096)])
def test_pieces_without_a_score_above_minus_infinity(gpu, monkeypatch, dim, first, count):
    """Finite values: such keys add nothing, and a row that has no others is zero."""
    case = hopeless_keys(dim, 4096, first, count)
    rest = np.r_[0:first, first + count:4096]
    q, k, v = (wide(bits).reshape(-1, 4, dim) for bits in (case.q, case.k, case.v))
    # the others alone: what is added for these keys are zeros, which round nothing
    want, tol = cross_reference(q, k[rest], v[rest], [[0, 1, 0, rest.size]], dim ** -0.5, np.zeros((1, 4, dim)))
    for name, got in zip(("cut", "whole"), results(gpu, case, monkeypatch)):
        assert (np.abs(got.reshape(want.shape) - want) <= tol).all(), name
