"""h3x_linear_lora_bf16 against the formula in 64 bits: shapes around every tile boundary, row maps of
every kind, odd sizes and ranks, refusals, and the calls a host can make around it."""
import numpy as np
import pytest

import h3_oracle as o
from adapter_case import NONE, assert_within, lora_reference, wide

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


class Case:
    def __init__(self, rows, k, n, adapters, rank, *, bias=True, scale=True, kind="runs", seed=1):
        rng = np.random.default_rng([seed, rows, k, n, adapters, rank])
        bits = lambda *shape, std=1.0: o.to_bf16((rng.standard_normal(shape) * std).astype(np.float32).reshape(-1))
        self.rows, self.k, self.n, self.adapters, self.rank = rows, k, n, adapters, rank
        self.x, self.w = bits(rows, k), bits(n, k, std=max(1, k) ** -0.5)
        self.bias = bits(n) if bias else None
        self.down, self.up = bits(adapters, rank, k, std=max(1, k) ** -0.5), bits(adapters, n, rank, std=rank ** -0.5)
        self.scale = (rng.random(adapters) * 2 - 0.5).astype(np.float32) if scale else None
        r = np.arange(rows)
        self.map = {
            "runs": r * (adapters + 1) // max(1, rows),             # contiguous, the last run without an adapter
            "each": r % adapters,                                   # every row another one than its neighbour
            "none": np.full(rows, NONE),
            "one": np.zeros(rows),
            "random": rng.integers(0, adapters + 2, rows),          # some beyond the last adapter
            "default": None,                                        # NULL: adapter 0
        }[kind]
        if self.map is not None:
            self.map = self.map.astype(np.uint32)

    def reference(self):
        row_adapter = self.map if self.map is not None else np.zeros(self.rows, np.uint32)
        scale = self.scale.astype(np.float64) if self.scale is not None else np.ones(self.adapters)
        return lora_reference(wide(self.x).reshape(self.rows, self.k), wide(self.w).reshape(self.n, self.k),
                              wide(self.bias) if self.bias is not None else None,
                              wide(self.down).reshape(self.adapters, self.rank, self.k),
                              wide(self.up).reshape(self.adapters, self.n, self.rank), scale, row_adapter)

    def tensors(self, gpu):
        return [gpu.bf16(self.x), gpu.bf16(self.w), gpu.bf16(self.bias) if self.bias is not None else None,
                gpu.bf16(self.down), gpu.bf16(self.up), gpu.f32(self.scale) if self.scale is not None else None,
                gpu.u32(self.map) if self.map is not None else None]

    def sizes(self):
        return self.rows, self.k, self.n, self.adapters, self.rank

    def run(self, gpu, pkg):
        tensors, out = self.tensors(gpu), gpu.bf16(np.full(self.rows * self.n, 0x7FC0, np.uint16))   # NaN where unwritten
        gpu.begin()
        gpu.op("h3x_linear_lora_bf16", out, *tensors, *self.sizes())
        gpu.submit()
        got = out.read()
        for t in [out, *tensors]:
            if t is not None:
                t.free()
        return got


@pytest.mark.parametrize("kind", ["runs", "each", "none", "one", "random", "default"])
@pytest.mark.parametrize("rows,k,n,adapters,rank", [
    (1, 256, 264, 3, 16), (7, 512, 1000, 2, 8), (33, 640, 520, 5, 12), (130, 1024, 768, 3, 64), (300, 328, 1288, 9, 20),
    (513, 576, 512, 4, 128)])
def test_maps_and_sizes(gpu, pkg, kind, rows, k, n, adapters, rank):
    case = Case(rows, k, n, adapters, rank, kind=kind)
    assert_within(case.run(gpu, pkg), *case.reference(), f"{kind} {case.sizes()}")


@pytest.mark.parametrize("rows,k,n,adapters,rank", [
    (1, 1, 1, 1, 1), (2, 3, 5, 2, 1), (65, 100, 131, 3, 7), (129, 257, 96, 2, 5), (40, 1001, 77, 4, 33),
    (200, 512, 520, 2, 7), (200, 512, 520, 2, 256), (96, 256, 512, 1, 255)])
def test_odd_sizes(gpu, pkg, rows, k, n, adapters, rank):
    for bias, scale, kind in ((True, True, "random"), (False, False, "runs")):
        case = Case(rows, k, n, adapters, rank, bias=bias, scale=scale, kind=kind)
        assert_within(case.run(gpu, pkg), *case.reference(), f"{case.sizes()}")


@pytest.mark.parametrize("rows", [1, 2, 8, 9, 16, 17, 31, 32, 33, 47, 63, 64, 65, 96, 127, 128, 129, 255, 256, 257])
def test_every_row_count_around_a_tile(gpu, pkg, rows):
    case = Case(rows, 1152, 1032, 3, 24, kind="random")
    assert_within(case.run(gpu, pkg), *case.reference(), f"rows {rows}")


@pytest.mark.parametrize("rows,k,n,adapters,rank,kind", [
    (1, 7168, 5376, 4, 16, "one"), (42, 2688, 5376, 2, 32, "runs"), (1664, 1024, 5376, 3, 64, "runs"),
    (2122, 5376, 1536, 16, 16, "each"), (800, 2048, 5376, 8, 128, "runs")])
def test_model_sizes(gpu, pkg, rows, k, n, adapters, rank, kind):
    case = Case(rows, k, n, adapters, rank, kind=kind, bias=False)
    assert_within(case.run(gpu, pkg), *case.reference(), f"{case.sizes()}")


@pytest.mark.parametrize("rows,k,n,adapters,rank,kind", [
    (300, 328, 520, 256, 64, "each"), (700, 1024, 256, 1024, 16, "random"), (260, 512, 520, 40, 200, "each"),
    (100, 512, 520, 100, 48, "each"), (2000, 512, 256, 300, 16, "runs")])
def test_more_adapters_than_are_computed_side_by_side(gpu, pkg, rows, k, n, adapters, rank, kind):
    case = Case(rows, k, n, adapters, rank, kind=kind)
    assert_within(case.run(gpu, pkg), *case.reference(), f"{case.sizes()}")


@pytest.mark.parametrize("rows,k,n,adapters,rank", [
    (1, 264, 50008, 3, 12), (9, 328, 38000, 4, 16), (16, 128, 100008, 2, 8), (17, 128, 100008, 2, 8), (2, 2816, 12552, 3, 24),
    (1, 8, 2_200_000, 2, 8), (3, 8, 8_400_000, 2, 8)])
def test_few_rows_of_a_wide_projection(gpu, pkg, rows, k, n, adapters, rank):
    case = Case(rows, k, n, adapters, rank, kind="random")
    assert_within(case.run(gpu, pkg), *case.reference(), f"{case.sizes()}")


@pytest.mark.parametrize("rank", [256, 250])
def test_low_rank_rows_beyond_a_gigabyte(gpu, pkg, rank):
    """256 entries of 256 rows in every tile: the rows are taken in several passes."""
    case = Case(9001, 64, 64, 256, rank, kind="random")
    assert_within(case.run(gpu, pkg), *case.reference(), f"rank {rank}")


@pytest.mark.parametrize("rows,k,n,rank,pairs", [(9_000_001, 8, 8, 8, False), (9_000_001, 8, 8, 8, True), (4_300_001, 3, 3, 2, False)])
def test_more_rows_than_a_grid_dimension_holds(gpu, pkg, monkeypatch, rows, k, n, rank, pairs):
    """On the tensor cores, with tiles of 128 and of 256 rows, and on the kernels for any shape; the input repeats a base
    block of rows."""
    if pairs:
        monkeypatch.setenv("H3B_CTA_PAIRS_ALWAYS", "1")
    base = Case(1009, k, n, 3, rank, kind="random")
    want, tol = base.reference()
    tensors = base.tensors(gpu)
    tensors[0].free()
    tensors[6].free()
    tensors[0] = gpu.bf16(np.resize(base.x, rows * k))
    tensors[6] = gpu.u32(np.resize(base.map, rows))
    out = gpu.bf16(np.full(rows * n, 0x7FC0, np.uint16))
    gpu.begin()
    gpu.op("h3x_linear_lora_bf16", out, *tensors, rows, k, n, 3, rank)
    gpu.submit()
    got = wide(out.read()).reshape(rows, n)
    for t in [out, *tensors]:
        t.free()
    for row0 in range(0, rows, 1009):
        count = min(1009, rows - row0)
        assert (np.abs(got[row0:row0 + count] - want[:count]) <= tol[:count]).all(), row0


@pytest.mark.parametrize("rows,k,n", [(5, 264, 272), (48, 512, 1024), (200, 512, 520), (400, 1024, 768)])
def test_an_adapter_of_infinities_stays_with_its_own_rows(gpu, pkg, rows, k, n):
    """Rows of other adapters and rows without one are finite and right, whatever adapter 1 holds."""
    case = Case(rows, k, n, 3, 16, kind="random")
    want, tol = case.reference()
    for name in ("down", "up"):
        other = Case(rows, k, n, 3, 16, kind="random")
        values = getattr(other, name).reshape(3, -1)
        values[1, ::3], values[1, 1::3] = 0x7F80, 0x7FC0          # infinity, NaN
        got = other.run(gpu, pkg).reshape(rows, n)
        at = case.map != 1
        assert_within(got[at], want[at], tol[at], f"{name} of another adapter")
    # a NaN in one row's input stays in that row
    other = Case(rows, k, n, 3, 16, kind="random")
    other.x.reshape(rows, k)[1, 5] = 0x7FC0
    got = other.run(gpu, pkg).reshape(rows, n)
    at = np.arange(rows) != 1
    assert_within(got[at], want[at], tol[at], "input of another row")
    assert np.isnan(wide(got[1])).all()


def test_without_adapters_it_is_the_plain_projection(gpu, pkg):
    case = Case(300, 512, 768, 2, 16, kind="none")
    tensors = case.tensors(gpu)
    plain, got = gpu.new(300 * 768, pkg.BF16), gpu.new(300 * 768, pkg.BF16)
    gpu.begin()
    gpu.op("linear_bf16", plain, tensors[0], tensors[1], tensors[2], 300, 512, 768)
    gpu.op("h3x_linear_lora_bf16", got, tensors[0], tensors[1], tensors[2], None, None, None, None, 300, 512, 768, 0, 0)
    gpu.submit()
    assert np.array_equal(plain.read(), got.read())


def test_the_same_call_twice_gives_the_same_bits(gpu, pkg):
    for shape in ((3, 2048, 1024, 4, 16), (200, 2048, 1024, 4, 64)):
        case = Case(*shape, kind="random")
        first = case.run(gpu, pkg)
        for _ in range(5):
            assert np.array_equal(first, case.run(gpu, pkg))


def test_statistics_count_a_projection(gpu, pkg):
    for rows, want in ((4, (1, 0)), (64, (0, 1))):
        case = Case(rows, 256, 256, 2, 8)
        before = gpu.stats()
        case.run(gpu, pkg)
        after = gpu.stats()
        assert (after.direct_dispatches - before.direct_dispatches,
                after.mps_linear_dispatches - before.mps_linear_dispatches) == want


def test_refusals(gpu, pkg):
    rows, k, n, adapters, rank = 8, 64, 64, 2, 8
    case = Case(rows, k, n, adapters, rank)
    x, w, bias, down, up, scale, row_map = case.tensors(gpu)
    out, small, f32 = gpu.new(rows * n, pkg.BF16), gpu.new(16, pkg.BF16), gpu.new(rows * k, pkg.F32)
    good = [out, x, w, bias, down, up, scale, row_map, rows, k, n, adapters, rank]
    assert not gpu.try_op("h3x_linear_lora_bf16", *good) and "no active command" in gpu.error()
    gpu.begin()
    try:
        def refused(place, value, text):
            args = list(good)
            args[place] = value
            assert not gpu.try_op("h3x_linear_lora_bf16", *args), text
            assert text in gpu.error(), gpu.error()
        for place, label in ((0, "output"), (1, "input"), (2, "weight"), (4, "down"), (5, "up")):
            refused(place, None, label)
            refused(place, f32, "wrong dtype")
            refused(place, small, "too small")
        refused(3, f32, "bias")
        refused(3, small, "too small")
        refused(6, small, "scale")
        refused(7, f32, "row adapter")
        refused(11, 1025, "adapters must be")
        refused(12, 0, "rank 1..256")
        refused(12, 257, "rank 1..256")
        refused(0, x, "overlaps")
        assert gpu.try_op("h3x_linear_lora_bf16", *good)
    finally:
        gpu.submit()


def test_no_rows_and_no_columns(gpu, pkg):
    case = Case(4, 64, 64, 2, 8)
    tensors, out = case.tensors(gpu), gpu.bf16(np.full(4 * 64, 7, np.uint16))
    gpu.begin()
    gpu.op("h3x_linear_lora_bf16", out, *tensors, 0, 64, 64, 2, 8)
    gpu.op("h3x_linear_lora_bf16", out, *tensors, 4, 64, 0, 2, 8)
    gpu.submit()
    assert (out.read() == 7).all()


def test_unaligned_tensors(gpu, pkg):
    """Views that start two bytes into a block: the kernels for any alignment serve them."""
    case = Case(70, 256, 264, 2, 16, kind="random")
    tensors = case.tensors(gpu)
    holders = []
    for i, bits in ((0, case.x), (4, case.up)):
        whole = gpu.bf16(np.concatenate([np.zeros(1, np.uint16), bits]))
        holders.append(whole)
        tensors[i] = gpu.wrap(whole.pointer + 2, bits.size, pkg.BF16)
    out = gpu.new(70 * 264, pkg.BF16)
    gpu.begin()
    gpu.op("h3x_linear_lora_bf16", out, *tensors, *case.sizes())
    gpu.submit()
    assert_within(out.read(), *case.reference(), "unaligned")


@pytest.mark.parametrize("rows,rank", [(3, 16), (300, 16), (3, 12), (300, 12)])
def test_on_another_stream_and_captured(pkg, rows, rank):
    """The op on a caller's stream, captured twice into graphs whose replays use inputs written later;
    a larger call in between may grow the context's workspace."""
    import torch
    gpu = pkg.Gpu(0)
    stream = torch.cuda.Stream()
    try:
        gpu.set_stream(stream.cuda_stream)
        cases = [Case(rows, 1024, 1024, 3, rank, kind="random", seed=s) for s in (1, 2)]
        sets = [(c, c.tensors(gpu), gpu.new(rows * 1024, pkg.BF16)) for c in cases]
        big = Case(900, 1024, 520, 8, 128, kind="each")
        big_set = (big.tensors(gpu), gpu.new(900 * 520, pkg.BF16))
        gpu.begin()
        for c, t, out in sets:                       # once outside a graph
            gpu.op("h3x_linear_lora_bf16", out, *t, *c.sizes())
        gpu.submit()
        want = [out.read() for _, _, out in sets]
        graphs = []
        gpu.begin()
        for c, t, out in sets:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                gpu.op("h3x_linear_lora_bf16", out, *t, *c.sizes())
            graphs.append(graph)
        gpu.op("h3x_linear_lora_bf16", big_set[1], *big_set[0], *big.sizes())
        gpu.submit()
        assert_within(big_set[1].read(), *big.reference(), "between the graphs")
        for c, t, out in sets:
            out.write(np.zeros(out.elements, np.uint16))
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        for _ in range(3):
            with torch.cuda.stream(stream):
                graphs[0].replay()
            with torch.cuda.stream(side):
                graphs[1].replay()
        torch.cuda.synchronize()
        # a graph may split its sums differently from an eager call: each is right by itself
        for (c, _, out), eager in zip(sets, want):
            assert_within(out.read(), *c.reference(), "replayed")
            assert_within(eager, *c.reference(), "eager")
        del graphs
    finally:
        gpu.close()
