"""h3x_cross_sdpa_bf16 against the formula in 64 bits: lengths from zero and one up, ragged and padded
batches, shared key heads, what padding holds, refusals, and the calls a host can make around it."""
import numpy as np
import pytest

import h3_oracle as o
from adapter_case import assert_within, cross_reference, wide

pytestmark = pytest.mark.gpu

MARK = 0x4248          # 50.0: what output rows hold before a call


@pytest.fixture(scope="module")
def pkg():
    import __graft_entry__ as entry
    return entry.load_package()


@pytest.fixture(scope="module")
def gpu(pkg):
    g = pkg.Gpu(0)
    yield g
    g.close()


class Case:
    """segments: list of [first query row, query rows, first key row, key rows], or None."""

    def __init__(self, segments, heads, kv_heads, dim, *, query_rows=None, key_rows=None, seed=1, spread=1.0):
        self.segments = segments
        self.query_rows = query_rows if query_rows is not None else max(s[0] + s[1] for s in segments)
        self.key_rows = key_rows if key_rows is not None else max(s[2] + s[3] for s in segments)
        self.heads, self.kv_heads, self.dim = heads, kv_heads, dim
        rng = np.random.default_rng([seed, self.query_rows, self.key_rows, heads, kv_heads, dim])
        bits = lambda rows, h, std=1.0: o.to_bf16((rng.standard_normal(rows * h * dim) * std).astype(np.float32))
        self.q = bits(self.query_rows, heads, spread)
        self.k, self.v = bits(self.key_rows, kv_heads), bits(self.key_rows, kv_heads)

    def spoil_gaps(self):
        """Key and value rows that no segment uses hold infinities and NaN."""
        used = np.zeros(self.key_rows, bool)
        for _, _, k0, kn in self.segments:
            used[k0:k0 + kn] = True
        for name, word in (("k", 0x7FC0), ("v", 0xFF80)):
            rows = getattr(self, name).reshape(self.key_rows, -1)
            rows[~used, ::2], rows[~used, 1::2] = word, 0x7FC0
        return self

    def reference(self, scale):
        shape = lambda bits, rows, h: wide(bits).reshape(rows, h, self.dim)
        q = shape(self.q, self.query_rows, self.heads)
        segments = self.segments if self.segments is not None else [[0, self.query_rows, 0, self.key_rows]]
        return cross_reference(q, shape(self.k, self.key_rows, self.kv_heads), shape(self.v, self.key_rows, self.kv_heads),
                               segments, scale, np.full(q.shape, 50.0))

    def tensors(self, gpu):
        table = gpu.u32(np.array(self.segments, np.uint32).reshape(-1)) if self.segments is not None else None
        return [gpu.bf16(self.q), gpu.bf16(self.k), gpu.bf16(self.v), table]

    def sizes(self):
        return (len(self.segments) if self.segments is not None else 0, self.query_rows, self.key_rows, self.heads,
                self.kv_heads, self.dim)

    def run(self, gpu, scale, in_place=False):
        tensors = self.tensors(gpu)
        out = tensors[0] if in_place else gpu.bf16(np.full(self.query_rows * self.heads * self.dim, MARK, np.uint16))
        gpu.begin()
        gpu.op("h3x_cross_sdpa_bf16", out, *tensors, *self.sizes(), float(scale))
        gpu.submit()
        got = out.read()
        for t in {id(t): t for t in [out, *tensors] if t is not None}.values():
            t.free()
        return got


def check(gpu, case, name="", scale=None, **kw):
    scale = scale if scale is not None else case.dim ** -0.5
    assert_within(case.run(gpu, scale, **kw), *case.reference(scale), name or str(case.segments))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("queries,keys", [
    (1, 1), (1, 77), (2, 128), (5, 129), (127, 64), (128, 128), (129, 255), (130, 256), (200, 257), (255, 3), (256, 384),
    (257, 511), (300, 640), (511, 130), (700, 1000)])
def test_one_segment(gpu, dim, queries, keys):
    check(gpu, Case([[0, queries, 0, keys]], 3, 3, dim))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(8, 8), (8, 2), (8, 1), (7, 1), (12, 4), (14, 2), (20, 4)])
def test_shared_key_heads(gpu, dim, heads, kv_heads):
    check(gpu, Case([[0, 150, 0, 200], [150, 9, 200, 333]], heads, kv_heads, dim).spoil_gaps(), f"{heads}/{kv_heads}")


RAGGED = [[0, 160, 0, 51], [160, 31, 51, 7], [191, 212, 58, 333], [403, 1, 391, 129], [404, 80, 520, 0], [484, 256, 520, 256]]


@pytest.mark.parametrize("dim", [64, 128])
def test_ragged_batch(gpu, dim):
    check(gpu, Case(RAGGED, 5, 5, dim, query_rows=800, key_rows=776))


@pytest.mark.parametrize("dim", [64, 128])
def test_padded_batch_whose_padding_holds_nan(gpu, dim):
    lengths, pad = [51, 7, 333, 129, 0, 256, 1], 333
    queries = [160, 31, 212, 1, 80, 256, 300]
    segments, q = [], 3                                          # rows before the first segment, gaps between them
    for i, (a, b) in enumerate(zip(queries, lengths)):
        segments.append([q, a, i * pad, b])
        q += a + i
    check(gpu, Case(segments, 4, 4, dim, query_rows=q + 5, key_rows=pad * len(lengths)).spoil_gaps())


def test_many_small_segments_and_shared_keys(gpu):
    segments = [[3 * i, 1 + i % 3, 11 * (i % 7), 1 + 5 * (i % 9)] for i in range(150)]
    check(gpu, Case(segments, 2, 2, 128, query_rows=460, key_rows=150).spoil_gaps(), "150 segments")


def test_segments_in_any_order(gpu):
    check(gpu, Case([RAGGED[i] for i in (3, 0, 5, 4, 2, 1)], 3, 3, 128, query_rows=800, key_rows=776), "shuffled")


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lengths", [[(1, 2048)], [(1, 4100), (1, 77), (1, 1)], [(4, 3000), (2, 0), (16, 1500)]])
def test_few_queries_over_long_states(gpu, dim, lengths):
    segments, q, k = [], 0, 0
    for a, b in lengths:
        segments.append([q, a, k, b])
        q, k = q + a, k + b
    check(gpu, Case(segments, 4, 2, dim))


@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 2, 128), (8, 2, 64), (16, 2, 128)])
@pytest.mark.parametrize("lengths", [
    [(1, 100), (1, 4000), (1, 0), (2, 129), (1, 2047)], [(130, 1500), (1, 12000), (700, 10), (3, 0)], [(1, 20001)]])
def test_segments_cut_into_different_numbers_of_pieces(gpu, heads, kv_heads, dim, lengths):
    segments, q, k = [], 2, 1
    for a, b in lengths:
        segments.append([q, a, k, b])
        q, k = q + a + 1, k + b + 3
    case = Case(segments, heads, kv_heads, dim, query_rows=q + 1, key_rows=k + 130).spoil_gaps()
    check(gpu, case, f"{lengths}")


@pytest.mark.parametrize("dim", [8, 32, 40, 80, 96, 100, 256, 512, 1])
def test_other_head_sizes(gpu, dim):
    check(gpu, Case([[0, 9, 0, 51], [9, 20, 60, 140]], 4, 2, dim).spoil_gaps(), f"dim {dim}")


@pytest.mark.parametrize("scale", [0.0, -0.1, 1.0])
def test_other_scales(gpu, scale):
    check(gpu, Case([[0, 70, 0, 200]], 2, 2, 64), f"scale {scale}", scale=scale)


def test_peaked_scores(gpu):
    """Scores far apart: the running maximum has to be raised many times."""
    for dim in (64, 128):
        case = Case([[0, 140, 0, 900]], 2, 2, dim, spread=6.0)
        order = np.argsort(wide(case.k).reshape(900, 2, dim)[:, 0, 0])          # growing along the keys
        case.k = np.ascontiguousarray(case.k.reshape(900, -1)[order]).reshape(-1)
        check(gpu, case, "peaked", scale=0.5)


def test_without_a_table_and_without_keys(gpu):
    check(gpu, Case(None, 3, 3, 128, query_rows=300, key_rows=200), "no table")
    check(gpu, Case(None, 3, 3, 64, query_rows=30, key_rows=0), "no keys")
    check(gpu, Case([[0, 5, 9, 0], [7, 0, 0, 9]], 3, 3, 128, query_rows=20, key_rows=9), "empty segments")


def test_rows_past_the_tensors_are_ignored(gpu):
    check(gpu, Case([[0, 40, 0, 70], [40, 1000, 70, 1 << 31], [90, 0xFFFFFFFF, 0xFFFFFFFF, 5]], 3, 3, 128,
                    query_rows=80, key_rows=100), "past the end")


@pytest.mark.parametrize("dim", [64, 128, 40])
def test_output_in_place_of_the_query(gpu, dim):
    case = Case([[0, 300, 0, 200], [300, 3, 200, 900]], 3, 3, dim)
    assert_within(case.run(gpu, dim ** -0.5, in_place=True), *case.reference(dim ** -0.5), "in place")


def test_equals_the_joint_attention_of_equal_lengths(gpu, pkg):
    """The sibling operator on the same rows, inside both operators' tolerances."""
    case = Case(None, 4, 4, 128, query_rows=500, key_rows=500)
    want, tol = case.reference(128 ** -0.5)
    tensors, out = case.tensors(gpu), gpu.new(500 * 4 * 128, pkg.BF16)
    gpu.begin()
    gpu.op("sdpa_bf16", out, *tensors[:3], 500, 4, 128, 128 ** -0.5)
    gpu.submit()
    assert_within(out.read(), want, tol, "joint")
    assert_within(case.run(gpu, 128 ** -0.5), want, tol, "cross")


def test_values_spoiled_inside_a_segment_stay_there(gpu):
    for dim in (64, 128):
        case = Case(RAGGED, 3, 3, dim, query_rows=800, key_rows=776)
        want, tol = case.reference(dim ** -0.5)
        case.v.reshape(776, -1)[60, :] = 0x7FC0                  # a key row of the third segment
        got = case.run(gpu, dim ** -0.5).reshape(800, 3, dim)
        clean = np.ones(800, bool)
        clean[191:403] = False
        assert_within(got[clean], want[clean], tol[clean], "other segments")
        assert np.isnan(wide(got[191:403])).all()


def test_the_same_call_twice_gives_the_same_bits(gpu):
    for case in (Case(RAGGED, 3, 3, 128), Case([[0, 1, 0, 3000]], 4, 4, 128)):
        first = case.run(gpu, 0.1)
        for _ in range(5):
            assert np.array_equal(first, case.run(gpu, 0.1))


def test_statistics_count_an_attention_call(gpu):
    before = gpu.stats().mps_sdpa_dispatches
    Case([[0, 3, 0, 1000]], 4, 4, 128).run(gpu, 0.1)
    assert gpu.stats().mps_sdpa_dispatches - before == 1


def test_refusals(gpu, pkg):
    case = Case([[0, 8, 0, 9]], 4, 2, 64)
    q, k, v, table = case.tensors(gpu)
    out, small, f32 = gpu.new(8 * 4 * 64, pkg.BF16), gpu.new(16, pkg.BF16), gpu.new(8 * 4 * 64, pkg.F32)
    good = [out, q, k, v, table, 1, 8, 9, 4, 2, 64, 0.125]
    assert not gpu.try_op("h3x_cross_sdpa_bf16", *good) and "no active command" in gpu.error()
    gpu.begin()
    try:
        def refused(changes, text):
            args = list(good)
            for place, value in changes.items():
                args[place] = value
            assert not gpu.try_op("h3x_cross_sdpa_bf16", *args), text
            assert text in gpu.error(), gpu.error()
        for place, label in ((0, "output"), (1, "query"), (2, "key"), (3, "value")):
            refused({place: None}, label)
            refused({place: f32}, "wrong dtype")
            refused({place: small}, "too small")
        refused({4: f32}, "segments")
        refused({5: 2}, "too small")
        refused({4: None}, "segments")
        for place in (8, 9, 10):
            refused({place: 0}, "empty")
        refused({8: 5}, "divide")
        refused({10: 513}, "too large")
        refused({0: k, 6: 2, 8: 2}, "overlaps")
        refused({0: v, 6: 2, 8: 2}, "overlaps")
        shifted = gpu.wrap(q.pointer + 64 * 4 * 2, 7 * 4 * 64, pkg.BF16)
        refused({0: shifted, 6: 7}, "overlaps part")
        assert gpu.try_op("h3x_cross_sdpa_bf16", *good)
    finally:
        gpu.submit()


def test_unaligned_tensors(gpu, pkg):
    case = Case([[0, 70, 0, 90]], 2, 2, 64)
    tensors = case.tensors(gpu)
    whole = gpu.bf16(np.concatenate([np.zeros(1, np.uint16), case.k]))
    tensors[1] = gpu.wrap(whole.pointer + 2, case.k.size, pkg.BF16)
    out = gpu.new(70 * 2 * 64, pkg.BF16)
    gpu.begin()
    gpu.op("h3x_cross_sdpa_bf16", out, *tensors, *case.sizes(), 0.125)
    gpu.submit()
    assert_within(out.read(), *case.reference(0.125), "unaligned")


@pytest.mark.parametrize("segments", [[[0, 300, 0, 200]], [[0, 1, 0, 3000]]])
def test_on_another_stream_and_captured(pkg, segments):
    """Captured twice on a caller's stream, replayed side by side; the table is read at replay."""
    import torch
    gpu = pkg.Gpu(0)
    stream = torch.cuda.Stream()
    try:
        gpu.set_stream(stream.cuda_stream)
        sets, tables = [], [torch.tensor(segments[0], dtype=torch.int32, device="cuda") for _ in range(2)]
        for seed, table in zip((1, 2), tables):
            c = Case(segments, 4, 4, 128, seed=seed)
            tensors = c.tensors(gpu)[:3] + [gpu.wrap(table.data_ptr(), 4, pkg.U32)]
            sets.append((c, tensors, gpu.new(c.query_rows * 512, pkg.BF16)))
        torch.cuda.synchronize()
        for c, t, out in sets:
            gpu.begin()
            gpu.op("h3x_cross_sdpa_bf16", out, *t, *c.sizes(), 0.1)
            gpu.submit()
        graphs = []
        gpu.begin()
        for c, t, out in sets:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                gpu.op("h3x_cross_sdpa_bf16", out, *t, *c.sizes(), 0.1)
            graphs.append(graph)
        gpu.submit()
        # the first request's states are shorter at replay
        sets[0][0].segments = [[0, segments[0][1], 5, segments[0][3] - 70]]
        tables[0].copy_(torch.tensor(sets[0][0].segments[0], dtype=torch.int32))
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        for _ in range(3):
            with torch.cuda.stream(stream):
                graphs[0].replay()
            with torch.cuda.stream(side):
                graphs[1].replay()
        torch.cuda.synchronize()
        for c, _, out in sets:
            assert_within(out.read(), *c.reference(0.1), "replayed")
        del graphs
    finally:
        gpu.close()
