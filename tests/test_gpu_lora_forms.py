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


# ------------------------------------------------------------------ the last round of tiles split along k
# 1,003 rows x 5,376 columns are 84 tiles of 256 x 256 on 74 pairs of SMs, or 168 of 128 x 256 on 148: what is left over
# after a round is cut along k into as many slices as there are 8 K blocks of 64, four at most, and the last slice
# carries the adapters. 400 rows x 38,400 are 300 pair tiles: four whole rounds in front.

SPLIT = [(1003, 2048, 5376, 16, 12), (1003, 1536, 5376, 5, 64), (1003, 1024, 5376, 3, 100), (400, 1024, 38400, 3, 16)]


@pytest.mark.parametrize("pairs", [True, False])
@pytest.mark.parametrize("kind", ["runs", "each", "none"])
@pytest.mark.parametrize("rows,k,n,adapters,rank", SPLIT)
def test_the_split_last_round(gpu, pkg, monkeypatch, rows, k, n, adapters, rank, kind, pairs):
    if not pairs:
        monkeypatch.setenv("H3B_NO_CTA_PAIRS", "1")
    case = Case(rows, k, n, adapters, rank, kind=kind)
    want, tol = case.reference()
    got = case.run(gpu, pkg)
    assert_within(got, want, tol, f"{case.sizes()}")
    assert np.array_equal(got, case.run(gpu, pkg))
    # other sums in another order: this shape did split, and without it the same holds
    monkeypatch.setenv("H3B_NO_SPLIT_K", "1")
    whole = case.run(gpu, pkg)
    assert_within(whole, want, tol, f"whole {case.sizes()}")
    assert not np.array_equal(got, whole)


@pytest.mark.parametrize("pairs", [True, False])
@pytest.mark.parametrize("rows,k,n,adapters,rank", [SPLIT[0], SPLIT[2]])
def test_the_split_last_round_beside_infinities(gpu, pkg, monkeypatch, rows, k, n, adapters, rank, pairs):
    if not pairs:
        monkeypatch.setenv("H3B_NO_CTA_PAIRS", "1")
    check_beside_infinities(gpu, pkg, Case(rows, k, n, adapters, rank, kind="each"))


@pytest.mark.parametrize("rows,pairs,rank", [(17001, False, 256), (17001, False, 250), (9001, True, 256), (9001, True, 250)])
def test_low_rank_rows_in_several_passes(gpu, pkg, monkeypatch, rows, pairs, rank):
    """Low-rank rows beyond 1 GiB. A tile of 128 rows has room for 128 entries of 128 x 256 columns, 8 MiB: 133 tiles are
    128 and 5. One of 256 rows has room for 256 of 256 x 256, 32 MiB: 36 tiles are 32 and 4. (Rank 250 is stored as 256,
    with up copied to rows of 256 in front of the first pass.)"""
    if pairs:
        monkeypatch.setenv("H3B_CTA_PAIRS_ALWAYS", "1")
    case = Case(rows, 64, 64, 256, rank, kind="random")
    got = case.run(gpu, pkg)
    assert_within(got, *case.reference(), f"{rows} rows, rank {rank}")
    assert np.array_equal(got, case.run(gpu, pkg))
