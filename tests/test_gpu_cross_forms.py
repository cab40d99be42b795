"""The forms of h3x_cross_sdpa_bf16 (keys cut into pieces or not, one or two query tiles per CTA, the kernel for any shape)
against the formula in 64 bits and against one another."""
import numpy as np
import pytest

from adapter_case import assert_within, cross_reference, wide
from test_gpu_cross import RAGGED, Case

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


# ------------------------------------------------------------------ two query tiles per CTA
# The form of every call is read from the op profile, so that a rule that moves fails here instead of leaving the
# kernel for many rows without a test.

@pytest.fixture(scope="module")
def profiled(pkg):
    with pytest.MonkeyPatch.context() as patch:
        patch.setenv("H3_PROFILE", "2")
        g = pkg.Gpu(0)
    yield g
    g.close()


@pytest.fixture
def form(profiled, monkeypatch, capfd):
    """form(): the form of the calls since the last time, which all have to have the same."""
    def read():
        monkeypatch.setenv("H3_PROFILE", "2")
        profiled.lib.h3_gpu_profile_mark(profiled.handle, b"calls")
        names = [line for line in capfd.readouterr().err.splitlines() if "launches" in line and "cross_sdpa_bf16" in line]
        assert len(names) == 1, names
        return names[0].split("cross_sdpa_bf16, ")[1].split("  ")[0].strip()
    return read


def packed(*lengths, gap=0):
    """Segments of (query rows, keys), one behind the other, `gap` rows and keys in between."""
    out, q, k = [], gap, gap
    for a, b in lengths:
        out.append([q, a, k, b])
        q, k = q + a + gap, k + b + gap
    return out


def check(gpu, case, form, want_form="two tiles", **kw):
    scale = case.dim ** -0.5
    got = case.run(gpu, scale, **kw)
    assert form() == want_form
    want, tol = case.reference(scale)
    if kw.get("in_place"):                                       # rows of no segment hold the query
        nobody = np.ones(case.query_rows, bool)
        for q0, qn, _, _ in case.segments:
            nobody[q0:q0 + qn] = False
        want[nobody] = wide(case.q).reshape(want.shape)[nobody]
    assert_within(got, want, tol, f"{want_form} {case.sizes()}")
    return got


@pytest.mark.parametrize("dim,heads", [(128, 56), (64, 112), (128, 24), (64, 56)])
@pytest.mark.parametrize("queries,keys", [(700, 300), (1283, 128), (1500, 77), (1409, 257), (1281, 1)])
def test_one_segment_of_many_rows(profiled, form, dim, heads, queries, keys):
    pairs, sms = (queries // 256 + 1) * heads, 148
    case = Case([[0, queries, 0, keys]], heads, heads, dim)
    check(profiled, case, form, "two tiles" if (pairs > 2 * sms if dim == 64 else 2 * pairs > sms) else "one tile")


@pytest.mark.parametrize("dim", [64, 128])
def test_a_ragged_batch_of_many_heads(profiled, form, dim):
    """Segments of one to 256 rows: whole tiles, tiles in part, a second tile of the pair that is dead."""
    case = Case(RAGGED, 56, 56, dim, query_rows=800, key_rows=776)
    first = check(profiled, case, form)
    for _ in range(3):
        assert np.array_equal(first, case.run(profiled, dim ** -0.5))
    form()
    check(profiled, Case([RAGGED[i] for i in (3, 0, 5, 4, 2, 1)], 56, 56, dim, query_rows=800, key_rows=776), form)


@pytest.mark.parametrize("dim", [64, 128])
def test_padding_of_nan_beside_many_rows(profiled, form, dim):
    """Unused keys and values hold infinities and NaN, behind every kind of last key tile; some rows are nobody's."""
    segments, q = [], 3
    for i, (a, b) in enumerate(zip([160, 31, 312, 1, 80, 256, 300, 129, 257], [51, 7, 333, 129, 0, 256, 1, 200, 383])):
        segments.append([q, a, i * 390, b])
        q += a + i
    check(profiled, Case(segments, 56, 56, dim, query_rows=q + 5, key_rows=390 * 9).spoil_gaps(), form)


@pytest.mark.parametrize("dim,heads,kv_heads,rows", [
    (128, 32, 8, 900), (64, 32, 8, 2500), (128, 16, 2, 1500), (64, 16, 2, 5000), (128, 32, 1, 700), (64, 32, 1, 2500),
    (128, 64, 1, 400), (64, 64, 1, 1300), (128, 128, 1, 200), (64, 128, 1, 700), (128, 28, 4, 700), (64, 28, 4, 2900),
    (128, 24, 4, 1700), (64, 24, 4, 3300), (128, 12, 4, 1700)])
def test_shared_key_heads_of_many_rows(profiled, form, dim, heads, kv_heads, rows):
    """2, 4, 8, 16 and more heads in a tile's rows, and groups of 3, 6 and 7 heads."""
    check(profiled, Case(packed((rows - 131, 200), (130, 333), gap=1), heads, kv_heads, dim, query_rows=rows + 9, key_rows=700)
          .spoil_gaps(), form)


@pytest.mark.parametrize("dim,heads,kv_heads", [(128, 56, 56), (64, 112, 112), (128, 56, 14), (64, 56, 56)])
def test_many_rows_in_place_of_the_query(profiled, form, dim, heads, kv_heads):
    case = Case(packed((300, 200), (3, 900), (140, 0), (700, 129), gap=2), heads, kv_heads, dim, query_rows=1400, key_rows=1300)
    check(profiled, case, form, in_place=True)


@pytest.mark.parametrize("dim,heads,kv_heads,lengths", [
    (128, 30, 30, [(300, 4000), (40, 96)]), (128, 56, 56, [(150, 4000), (150, 96)]), (128, 64, 16, [(300, 8000), (9, 0), (100, 130)]),
    (64, 56, 56, [(500, 6001), (1, 1), (60, 130), (7, 64), (130, 0), (180, 300)]), (64, 112, 112, [(258, 4500), (40, 96)])])
def test_many_rows_over_keys_that_are_cut(profiled, form, dim, heads, kv_heads, lengths):
    """A segment of long states beside short ones is cut into pieces whose results are joined."""
    segments = packed(*lengths, gap=3)
    case = Case(segments, heads, kv_heads, dim, query_rows=segments[-1][0] + segments[-1][1] + 4,
                key_rows=segments[-1][2] + segments[-1][3] + 130).spoil_gaps()
    first = check(profiled, case, form, "two tiles, cut")
    assert np.array_equal(first, case.run(profiled, dim ** -0.5))
    form()


@pytest.mark.parametrize("dim", [64, 128])
def test_peaked_scores_of_many_rows(profiled, form, dim):
    """Scores far apart, growing along the keys: both groups raise their reference many times."""
    case = Case([[0, 1300, 0, 900]], 56, 56, dim, spread=6.0)
    order = np.argsort(wide(case.k).reshape(900, 56, dim)[:, 0, 0])
    case.k = np.ascontiguousarray(case.k.reshape(900, -1)[order]).reshape(-1)
    got = case.run(profiled, 0.5)
    assert form() == "two tiles"
    assert_within(got, *case.reference(0.5), f"peaked {dim}")


@pytest.mark.parametrize("dim", [64, 128])
def test_values_spoiled_inside_a_segment_of_many_rows_stay_there(profiled, form, dim):
    case = Case(RAGGED, 56, 56, dim, query_rows=800, key_rows=776)
    want, tol = case.reference(dim ** -0.5)
    case.v.reshape(776, -1)[60, :] = NAN                         # a key row of the third segment
    got = case.run(profiled, dim ** -0.5).reshape(want.shape)
    assert form() == "two tiles"
    clean = np.ones(800, bool)
    clean[191:403] = False
    assert_within(got[clean], want[clean], tol[clean], "other segments")
    assert np.isnan(wide(got[191:403])).all()


@pytest.mark.parametrize("dim", [64, 128])
def test_rows_of_queries_that_are_not_finite_stay_alone(profiled, form, dim):
    """The rows between and behind the segments too: they share tiles with rows that count."""
    segments = packed((300, 200), (130, 300), (500, 77), (400, 129), gap=5)
    case = Case(segments, 56, 56, dim, query_rows=1400, key_rows=800)
    want, tol = case.reference(dim ** -0.5)
    used = np.zeros(1400, bool)
    for q0, qn, _, _ in segments:
        used[q0:q0 + qn] = True
    rows = case.q.reshape(1400, -1)
    rows[~used] = NAN
    rows[[7, 340, 600]] = INF                                    # of three segments
    got = case.run(profiled, dim ** -0.5).reshape(want.shape)
    assert form() == "two tiles"
    clean = np.ones(1400, bool)
    clean[[7, 340, 600]] = False
    assert_within(got[clean], want[clean], tol[clean], "the other rows")


def test_one_tile_and_two_tiles_in_two_contexts_at_once(pkg):
    """Calls of both forms and of the adapter projection in two contexts on two streams, interleaved without a wait."""
    import torch
    contexts, streams = [pkg.Gpu(0), pkg.Gpu(0)], [torch.cuda.Stream(), torch.cuda.Stream()]
    cases = [Case(RAGGED, 56, 56, 128, query_rows=800, key_rows=776), Case([[0, 1, 0, 3000]], 8, 8, 128),
             Case(packed((900, 300), (130, 77)), 32, 8, 128), Case(packed((300, 4000), (40, 96)), 30, 30, 128),
             Case([[0, 1500, 0, 200]], 56, 56, 64)]
    try:
        for gpu, stream in zip(contexts, streams):
            gpu.set_stream(stream.cuda_stream)
        alone = [[c.run(gpu, 0.1) for c in cases] for gpu in contexts]
        sets = [[(c, c.tensors(gpu), gpu.bf16(np.full(c.q.size, 0x4248, np.uint16))) for c in cases] for gpu in contexts]
        for gpu in contexts:
            gpu.begin()
        for turn in range(20):
            for i in range(len(cases)):
                for n, gpu in enumerate(contexts):
                    c, tensors, out = sets[n][(i + 2 * n + turn) % len(cases)]
                    gpu.op("h3x_cross_sdpa_bf16", out, *tensors, *c.sizes(), 0.1)
        for gpu in contexts:
            gpu.submit()
        for n in range(2):
            for (c, _, out), bits in zip(sets[n], alone[n]):
                assert np.array_equal(out.read(), bits), c.sizes()
    finally:
        for gpu in contexts:
            gpu.close()


@pytest.mark.parametrize("lengths", [[(700, 300), (131, 77)], [(300, 4000), (40, 96)]])
def test_many_rows_captured(pkg, lengths):
    """Two graphs, replayed side by side; one table is written between capture and replay."""
    import torch
    gpu, stream = pkg.Gpu(0), torch.cuda.Stream()
    try:
        gpu.set_stream(stream.cuda_stream)
        sets = []
        for seed in (1, 2):
            c = Case(packed(*lengths), 30, 30, 128, seed=seed)
            table = torch.tensor(c.segments, dtype=torch.int32, device="cuda").reshape(-1)
            sets.append((c, c.tensors(gpu)[:3] + [gpu.wrap(table.data_ptr(), 8, pkg.U32)], table, gpu.bf16(np.full(c.q.size, 0x4248, np.uint16))))
        torch.cuda.synchronize()
        graphs = []
        gpu.begin()
        for c, tensors, _, out in sets:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                gpu.op("h3x_cross_sdpa_bf16", out, *tensors, *c.sizes(), 0.1)
            graphs.append(graph)
        gpu.submit()
        sets[0][0].segments = [[s[0], s[1], s[2] + 3, s[3] - 60] for s in sets[0][0].segments]
        sets[0][2].copy_(torch.tensor(sets[0][0].segments, dtype=torch.int32).reshape(-1))
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        for _ in range(3):
            with torch.cuda.stream(stream):
                graphs[0].replay()
            with torch.cuda.stream(side):
                graphs[1].replay()
        torch.cuda.synchronize()
        for c, _, _, out in sets:
            assert_within(out.read(), *c.reference(0.1), "replayed")
        del graphs
    finally:
        gpu.close()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lengths,heads,want_form", [
    ([(1, 4096)], 4, "one tile, cut"), ([(300, 500)], 4, "one tile"), ([(1000, 500)], 112, "two tiles"),
    ([(258, 4500), (40, 96)], 112, "two tiles, cut")])
@pytest.mark.parametrize("first", [0, 100, 372])
def test_hopeless_keys_in_every_form(profiled, form, dim, lengths, heads, want_form, first):
    """128 keys of the first segment without a score above -inf: a column of values with a NaN among them is NaN, the
    other columns are those of the other keys."""
    segments = packed(*lengths)
    case = Case(segments, heads, heads, dim)
    case.q &= 0x7FFF
    case.q[case.q == 0] = 0x3F80
    k, v = (bits.reshape(-1, heads, dim) for bits in (case.k, case.v))
    k[first:first + 128, :, 0] = LOW
    v[first:first + 128, :, ::2] = NAN
    got = case.run(profiled, dim ** -0.5).reshape(-1, heads, dim)
    assert form() == want_form
    rows, keys = lengths[0]
    rest = np.r_[0:first, first + 128:keys]
    q = wide(case.q).reshape(-1, heads, dim)[:rows]
    sample = np.unique(np.r_[0:rows:37, rows - 1])                       # some rows for the reference
    want, tol = cross_reference(q[sample], wide(k)[rest], wide(v)[rest], [[0, sample.size, 0, rest.size]], dim ** -0.5,
                                np.zeros((sample.size, heads, dim)))
    assert np.isnan(wide(got[:rows, :, ::2])).all()
    assert_within(got[sample][:, :, 1::2], want[:, :, 1::2], tol[:, :, 1::2], want_form)
    assert np.isfinite(wide(got[rows:])).all()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lengths,heads,want_form", [
    ([(1, 4096)], 4, "one tile, cut"), ([(300, 500)], 4, "one tile"), ([(1000, 500)], 112, "two tiles")])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_of_two_to_the_28(profiled, form, dim, lengths, heads, want_form, sign):
    """Queries and keys whose scores are exact in F32, up to 2^28 in magnitude with steps of 2^21: the largest takes all.
    The kernel's reference is off from it by up to half a step of 2^29 (2^-24 of it: 32), which has to cancel."""
    (rows, keys), = lengths
    case = Case([[0, rows, 0, keys]], heads, heads, dim)
    exact = lambda values: (values.astype(np.float32).view(np.uint32) >> 16).astype(np.uint16)
    case.q = exact(np.full(case.q.size, sign * 4096.0))
    rng = np.random.default_rng(keys)
    c = np.r_[np.arange(keys - 1) % 127 + 1, 128] * (2.0 ** 16 / dim / 128)      # dot: 4096 * dim * c = 2^21 * (1 .. 128)
    if sign < 0:                                                               # the largest score is the smallest in magnitude
        c = np.where(np.arange(keys) == keys - 1, 64.0, 64 + np.arange(keys) % 64 + 1) * (2.0 ** 16 / dim / 128)
    order = rng.permutation(keys)
    case.k = exact(np.repeat(c[order], heads * dim))
    got = wide(case.run(profiled, 1.0)).reshape(rows, heads, dim)
    assert form() == want_form
    want = wide(case.v).reshape(keys, heads, dim)[np.argmax(order)]
    # the probability is rounded to BF16, its sum is not; the result is rounded to BF16
    assert (np.abs(got - want) <= (2.0 ** -8 + 2.0 ** -8 + 2.0 ** -16 + 2.0 ** -20) * np.abs(want)).all()
