"""Host logic of adapters and conditioning, no GPU: the op sequence of a block with them, the refusals of the
segment table and of combinations, and what stays as it was without them."""
import numpy as np
import pytest


@pytest.fixture(scope="module")
def pkg():
    import __graft_entry__ as entry
    return entry.load_package()


class FakeTensor:
    def __init__(self, name):
        self.name = name

    def __repr__(self):
        return self.name


class FakeGpu:
    def __init__(self):
        self.log, self.uploads = [], []

    def new(self, n, dtype):
        return FakeTensor(f"new{n}")

    def upload(self, values):
        self.uploads.append(np.asarray(values))
        return FakeTensor(f"upload{len(self.uploads) - 1}")

    bf16 = u32 = f32 = upload

    def flush(self):
        self.log.append(("flush",))

    def op(self, name, *args):
        self.log.append((name,) + args)

    def names(self):
        return [entry[0] for entry in self.log]


def shape(pkg):
    return pkg.DitShape(hidden=64, heads=2, head_dim=128, ffn=32, blocks=2)


def weights(pkg):
    return pkg.BlockWeights(**{n: FakeTensor(n) for n in ("norm1", "norm2", "qkv", "q_norm", "k_norm", "out", "fc1", "fc2",
                                                          "modulation")})


def pair(name):
    return FakeTensor(name + "_down"), FakeTensor(name + "_up")


PLAIN = ["adaln_bf16", "grouped_qkv_linear_rope_bf16", "sdpa_bf16", "linear_bf16", "gate_adaln_bf16", "mlp_bf16", "gate_bf16"]


def test_a_block_without_them_is_as_before(pkg):
    gpu = FakeGpu()
    dit = pkg.Dit(gpu, shape(pkg), 10)
    dit.run_block(weights(pkg), *[FakeTensor(n) for n in ("map", "cos", "sin")], False, None)
    assert gpu.names() == PLAIN
    gpu.log.clear()
    dit.run_block(weights(pkg), *[FakeTensor(n) for n in ("map", "cos", "sin")], False, None,
                  pkg.BlockAdapters(adapters=1, rank=4))
    assert gpu.names() == PLAIN


def test_every_projection_with_adapters_and_conditioning(pkg):
    gpu, s = FakeGpu(), shape(pkg)
    dit = pkg.Dit(gpu, s, 10)
    rows, scale = FakeTensor("row_adapter"), FakeTensor("scale")
    adapters = pkg.BlockAdapters(adapters=3, rank=4, row_adapter=rows, scale=scale, qkv=pair("qkv"), out=pair("out"),
                                 fc1=pair("fc1"), fc2=pair("fc2"))
    cond = pkg.Conditioning(gpu, s, rows=10, states=7, segments=[(2, 8, 0, 7)])
    for _ in range(2):
        cond.add_block(FakeTensor("states"), 48, FakeTensor("wk"), FakeTensor("wv"), adapters, pair("k"), None)
    assert gpu.names() == ["h3x_linear_lora_bf16", "linear_bf16"] * 2
    gpu.log.clear()
    dit.run_block(weights(pkg), *[FakeTensor(n) for n in ("map", "cos", "sin")], False, None, adapters, cond, 1)
    assert gpu.names() == ["adaln_bf16", "h3x_linear_lora_bf16", "grouped_qkv_rope_bf16", "sdpa_bf16", "h3x_cross_sdpa_bf16",
                           "add_bf16", "h3x_linear_lora_bf16", "gate_adaln_bf16", "h3x_linear_lora_bf16", "swiglu_bf16",
                           "h3x_linear_lora_bf16", "gate_bf16"]
    lora = [entry[1:] for entry in gpu.log if entry[0] == "h3x_linear_lora_bf16"]
    assert [str(a[2]) for a in lora] == ["qkv", "out", "fc1", "fc2"]
    assert [(str(a[4]), str(a[5])) for a in lora] == [(n + "_down", n + "_up") for n in ("qkv", "out", "fc1", "fc2")]
    assert [a[8:] for a in lora] == [(10, 64, 768, 3, 4), (10, 256, 64, 3, 4), (10, 64, 64, 3, 4), (10, 32, 64, 3, 4)]
    assert all(a[3] is None and a[6] is scale and a[7] is rows for a in lora)
    cross = next(entry[1:] for entry in gpu.log if entry[0] == "h3x_cross_sdpa_bf16")
    assert cross[1] is dit.query and cross[2:4] == cond.blocks[1] and cross[4] is cond.segments
    assert cross[5:] == (1, 10, 7, 2, 2, 128, s.scale)
    add = next(entry[1:] for entry in gpu.log if entry[0] == "add_bf16")
    assert add == (dit.attention_heads, dit.attention_heads, cond.heads, 10 * 256)
    assert not gpu.uploads[1].any() and gpu.uploads[1].size == 10 * 256      # rows of no segment add zeros


def test_adapters_on_one_projection_of_the_mlp(pkg):
    for given, want in (("fc1", ["h3x_linear_lora_bf16", "swiglu_bf16", "linear_bf16"]),
                        ("fc2", ["h3x_linear_swiglu_bf16", "h3x_linear_lora_bf16"])):
        gpu = FakeGpu()
        dit = pkg.Dit(gpu, shape(pkg), 10)
        adapters = pkg.BlockAdapters(adapters=1, rank=4, **{given: pair(given)})
        dit.run_block(weights(pkg), *[FakeTensor(n) for n in ("map", "cos", "sin")], True, None, adapters)
        names = gpu.names()
        assert names[names.index("gate_adaln_bf16") + 1:names.index("gate_bf16")] == want


def test_run_blocks_hands_every_block_its_own(pkg):
    gpu, s = FakeGpu(), shape(pkg)
    dit = pkg.Dit(gpu, s, 10)
    cond = pkg.Conditioning(gpu, s, rows=10, states=7, segments=[(0, 10, 0, 7)], kv_heads=1)
    for i in range(2):
        cond.add_block(FakeTensor("states"), 48, FakeTensor("wk"), FakeTensor("wv"))
    adapters = [None, pkg.BlockAdapters(adapters=1, rank=4, out=pair("second"))]
    gpu.log.clear()
    dit.run_blocks([weights(pkg), weights(pkg)], *[FakeTensor(n) for n in ("map", "cos", "sin")], adapters=adapters,
                   conditioning=cond)
    crosses = [entry[1:] for entry in gpu.log if entry[0] == "h3x_cross_sdpa_bf16"]
    assert [c[2:4] for c in crosses] == cond.blocks and [c[9] for c in crosses] == [1, 1]
    assert [str(entry[5]) for entry in gpu.log if entry[0] == "h3x_linear_lora_bf16"] == ["second_down"]
    maps = [FakeTensor(n) for n in ("map", "cos", "sin")]
    with pytest.raises(ValueError, match="one entry per block"):
        dit.run_blocks([weights(pkg)], *maps, adapters=adapters)
    with pytest.raises(ValueError, match="every block"):
        dit.run_blocks([weights(pkg)] * 3, *maps, conditioning=cond)
    with pytest.raises(ValueError, match="token reduction"):
        dit.run_blocks([weights(pkg)] * 2, *maps, reduction=object(), adapters=adapters)


def test_not_with_sequence_parallelism(pkg):
    class Two:
        world, rank = 2, 0
    dit = pkg.Dit(FakeGpu(), shape(pkg), 10, Two())
    with pytest.raises(ValueError, match="sequence parallelism"):
        dit.run_block(weights(pkg), *[FakeTensor(n) for n in ("map", "cos", "sin")], False, None,
                      pkg.BlockAdapters(adapters=1, rank=4))


@pytest.mark.parametrize("segments,text", [
    ([(0, 11, 0, 1)], "past"), ([(0, 1, 0, 8)], "past"), ([(-1, 1, 0, 1)], "past"), ([(0, 5, 0, 1), (4, 2, 0, 1)], "overlap"),
    ([(5, 5, 0, 1), (0, 6, 1, 1)], "overlap")])
def test_segment_tables_that_are_refused(pkg, segments, text):
    with pytest.raises(ValueError, match=text):
        pkg.Conditioning(FakeGpu(), shape(pkg), rows=10, states=7, segments=segments)


def test_segment_tables_that_are_not(pkg):
    gpu = FakeGpu()
    cond = pkg.Conditioning(gpu, shape(pkg), rows=10, states=7, segments=[(5, 5, 0, 7), (0, 5, 0, 7), (3, 0, 2, 0)])
    assert cond.segment_count == 3 and gpu.uploads[0].dtype == np.uint32
    with pytest.raises(ValueError, match="divide"):
        pkg.Conditioning(gpu, shape(pkg), rows=10, states=7, segments=[], kv_heads=3)
