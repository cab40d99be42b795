"""Calls of the block driver with adapters and conditioning, no GPU: single blocks on rows that are not those they were made
for, and a denoise step that has them."""
import pytest

from test_adapters_host import FakeGpu, FakeTensor, pair, shape, weights


@pytest.fixture(scope="module")
def pkg():
    import __graft_entry__ as entry
    return entry.load_package()


def maps():
    return [FakeTensor(n) for n in ("map", "cos", "sin")]


def conditioning(pkg, gpu, rows, blocks):
    cond = pkg.Conditioning(gpu, shape(pkg), rows=rows, states=7, segments=[(0, rows, 0, 7)])
    for _ in range(blocks):
        cond.add_block(FakeTensor("states"), 48, FakeTensor("wk"), FakeTensor("wv"))
    gpu.log.clear()
    return cond


def test_a_block_with_conditioning_of_other_rows_is_refused(pkg):
    """Its attention would read and add rows that the block does not have."""
    for rows in (9, 11):
        gpu = FakeGpu()
        dit, cond = pkg.Dit(gpu, shape(pkg), 10), conditioning(pkg, gpu, rows, 1)
        with pytest.raises(ValueError, match="these rows"):
            dit.run_block(weights(pkg), *maps(), False, None, None, cond)
        assert gpu.log == []


def test_a_block_without_keys_of_its_own_is_refused_before_anything_runs(pkg):
    gpu = FakeGpu()
    dit, cond = pkg.Dit(gpu, shape(pkg), 10), conditioning(pkg, gpu, 10, 2)
    for block in (2, -1):
        with pytest.raises(ValueError, match="this block"):
            dit.run_block(weights(pkg), *maps(), False, None, None, cond, block)
    assert gpu.log == []


def test_a_single_block_on_the_reduced_rows_is_refused(pkg):
    """Token reduction pools rows: the row map of the adapters and the segments are of other rows then."""
    gpu = FakeGpu()
    dit, cond = pkg.Dit(gpu, shape(pkg), 10), conditioning(pkg, gpu, 10, 1)
    dit.active_rows = dit.active_sequence = 6
    for given in (dict(adapters=pkg.BlockAdapters(adapters=1, rank=4, out=pair("out"))), dict(conditioning=cond)):
        with pytest.raises(ValueError, match="token reduction"):
            dit.run_block(weights(pkg), *maps(), False, None, **given)
    assert gpu.log == []
    dit.run_block(weights(pkg), *maps(), False, None)


def test_a_denoise_step_hands_both_to_every_block(pkg):
    gpu, s = FakeGpu(), shape(pkg)
    dit, cond = pkg.Dit(gpu, s, 10), conditioning(pkg, gpu, 10, 2)
    names = ("patch_weight", "patch_bias", "text_hidden", "final_norm", "final_modulation", "final_weight", "final_bias", "row_map",
             "final_row_map", "rope_cos", "rope_sin")
    step = pkg.DenoiseStep(dit, [weights(pkg), weights(pkg)], video_rows=7, text_rows=3, **{n: FakeTensor(n) for n in names})
    step.forward()
    plain = gpu.names()
    assert not any("lora" in n or "cross" in n for n in plain)
    gpu.log.clear()
    step.adapters = [pkg.BlockAdapters(adapters=1, rank=4, out=pair("first")), pkg.BlockAdapters(adapters=2, rank=8, out=pair("second"))]
    step.conditioning = cond
    step.forward()
    lora = [entry[1:] for entry in gpu.log if entry[0] == "h3x_linear_lora_bf16"]
    assert [str(a[4]) for a in lora] == ["first_down", "second_down"] and [a[-2:] for a in lora] == [(1, 4), (2, 8)]
    assert [entry[3:5] for entry in gpu.log if entry[0] == "h3x_cross_sdpa_bf16"] == cond.blocks
    rest = [n for n in gpu.names() if n not in ("h3x_linear_lora_bf16", "h3x_cross_sdpa_bf16", "add_bf16")]
    assert rest == [n for i, n in enumerate(plain) if not (n == "linear_bf16")]
