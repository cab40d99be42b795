"""The forms of h3x_linear_lora_bf16 (few rows, lone and paired tiles, a last round split along k, several passes of rows)
against the formula in 64 bits, and what an adapter that is not finite costs the others."""
import numpy as np
import pytest

from adapter_case import assert_within, wide
from test_gpu_lora import Case

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


def check_beside_infinities(gpu, pkg, case, word=0x7F80):
    """`up` of adapter 1 all infinities (or `word`): the rows of the others are right, its own are not finite."""
    want, tol = case.reference()
    case.up = case.up.copy()
    case.up.reshape(case.adapters, -1)[1] = word
    got = case.run(gpu, pkg).reshape(case.rows, case.n)
    own = case.map == 1
    assert own.any() and not own.all()
    assert_within(got[~own], want[~own], tol[~own], f"beside adapter 1 {case.sizes()}")
    assert not np.isfinite(wide(got[own])).any()


@pytest.mark.parametrize("word", [0x7F80, 0x7FC0])
@pytest.mark.parametrize("rows,k,n,adapters,rank", [
    (5, 7168, 1032, 3, 16), (12, 7168, 520, 4, 12), (100, 7168, 520, 3, 16), (400, 7168, 768, 3, 16), (300, 2688, 2056, 2, 20),
    (129, 1032, 776, 3, 8), (257, 1024, 5376, 3, 64)])
def test_an_adapter_of_nothing_but_infinities(gpu, pkg, rows, k, n, adapters, rank, word):
    check_beside_infinities(gpu, pkg, Case(rows, k, n, adapters, rank, kind="random"), word)


@pytest.mark.parametrize("rows,k,n", [(400, 1024, 38400), (12, 1024, 38400)])
def test_an_adapter_of_infinities_holds_up_no_wait(pkg, rows, k, n):
    """Several tiles per CTA, each with something to repair, under a wait budget of half a millisecond (the call itself
    takes a tenth of that): the repair is behind the last of the kernel's waits, whatever it takes."""
    gpu = pkg.Gpu(0)
    try:
        assert gpu.lib.h3x_set_wait_budget_cycles(gpu.handle, 1_000_000, 0) == 1
        check_beside_infinities(gpu, pkg, Case(rows, k, n, 3, 16, kind="random"))
    finally:
        gpu.close()
