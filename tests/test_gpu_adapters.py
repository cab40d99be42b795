"""A block with adapters beside every projection and conditioning on an encoder's states, through the host driver,
against the same block composed of the oracle's ops and the two operators' formulas in 64 bits."""
import numpy as np
import pytest

import h3_oracle as o
from adapter_case import NONE, cross_reference, lora_reference, wide
from block_case import make_block_case, upload_block
from parity import assert_block_close

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pkg():
    import __graft_entry__ as entry
    return entry.load_package()


def bits(rng, *shape, std=1.0):
    return o.to_bf16((rng.standard_normal(shape) * std).astype(np.float32).reshape(-1))


def lora_bits(x, w, pair, rows, k, n, rank, scale, row_adapter):
    y, _ = lora_reference(wide(x).reshape(rows, k), wide(w).reshape(n, k), None, wide(pair[0]).reshape(-1, rank, k),
                          wide(pair[1]).reshape(-1, n, rank), scale.astype(np.float64), row_adapter)
    return o.to_bf16(y.astype(np.float32).reshape(-1))


@pytest.mark.parametrize("rows,text_rows,heads,kv_heads", [(320, 64, 4, 4), (200, 72, 4, 2)])
def test_block_with_adapters_and_conditioning(pkg, rows, text_rows, heads, kv_heads):
    case = make_block_case(rows=rows, text_rows=text_rows, heads=heads, hidden=512, ffn=768, seed=3)
    hidden, ffn, inner, rank, adapters, states, width = 512, 768, heads * 128, 12, 3, 77 + 129, 256
    rng = np.random.default_rng(rows)
    row_adapter = np.where(np.arange(rows) < text_rows, NONE, np.arange(rows) // 50 % adapters).astype(np.uint32)
    scale = np.array([1.0, 0.5, 2.0], np.float32)
    dims = {"qkv": (hidden, 3 * inner), "out": (inner, hidden), "fc1": (hidden, 2 * ffn), "fc2": (ffn, hidden)}
    pairs = {n: (bits(rng, adapters, rank, k, std=k ** -0.5), bits(rng, adapters, m, rank, std=0.02)) for n, (k, m) in dims.items()}
    encoder = bits(rng, states, width)
    wk, wv = bits(rng, kv_heads * 128, width, std=width ** -0.5), bits(rng, kv_heads * 128, width, std=width ** -0.5)
    middle = text_rows + (rows - text_rows) // 2
    segments = [(text_rows, middle - text_rows, 0, 77), (middle, rows - middle, 77, 129)]

    gpu = pkg.Gpu(0)
    try:
        shape = pkg.DitShape(hidden=hidden, heads=heads, ffn=ffn, blocks=1)
        dit = pkg.Dit(gpu, shape, rows)
        block = pkg.BlockAdapters(adapters=adapters, rank=rank, row_adapter=gpu.u32(row_adapter), scale=gpu.f32(scale),
                                  **{n: (gpu.bf16(d), gpu.bf16(u)) for n, (d, u) in pairs.items()})
        cond = pkg.Conditioning(gpu, shape, rows=rows, states=states, segments=segments, kv_heads=kv_heads)
        w = upload_block(pkg, gpu, case)
        tables = gpu.u32(case.row_map), gpu.bf16(case.rope_cos), gpu.bf16(case.rope_sin)
        dit.hidden.write(case.hidden)
        gpu.begin()
        cond.add_block(gpu.bf16(encoder), width, gpu.bf16(wk), gpu.bf16(wv))
        dit.run_blocks([w], *tables, adapters=[block], conditioning=cond)
        gpu.submit()
        got = dit.hidden.read()
        # the same driver without them afterwards: nothing of them is left behind
        dit.hidden.write(case.hidden)
        gpu.begin()
        dit.run_block(w, *tables, False, None)
        gpu.submit()
        plain = dit.hidden.read()
    finally:
        gpu.close()

    c = case.weights
    mod = o.adaln_bf16(case.hidden, c["norm1"], c["modulation"], case.row_map, rows, hidden, 6, 0, 1)
    qkv = lora_bits(mod, c["qkv_weight"], pairs["qkv"], rows, hidden, 3 * inner, rank, scale, row_adapter)
    q, k, v = o.qkv_rope_bf16(qkv, c["q_norm"], c["k_norm"], case.rope_cos, case.rope_sin, rows, heads, 128, 48)
    joint = o.sdpa_bf16(q, k, v, rows, heads, 128, 128 ** -0.5, round_p=1)
    ks = o.linear_bf16(encoder, wk, None, states, width, kv_heads * 128)
    vs = o.linear_bf16(encoder, wv, None, states, width, kv_heads * 128)
    extra, _ = cross_reference(wide(q).reshape(rows, heads, 128), wide(ks).reshape(states, kv_heads, 128),
                               wide(vs).reshape(states, kv_heads, 128), segments, 128 ** -0.5, np.zeros((rows, heads, 128)))
    mixed = o.add_bf16(joint, o.to_bf16(extra.astype(np.float32).reshape(-1)))
    out = lora_bits(mixed, c["out_weight"], pairs["out"], rows, inner, hidden, rank, scale, row_adapter)
    gated, mod = o.gate_adaln_bf16(case.hidden, out, c["norm2"], c["modulation"], c["modulation"], case.row_map, rows, hidden, 6,
                                   2, 3, 4)
    fused = lora_bits(mod, c["fc1_weight"], pairs["fc1"], rows, hidden, 2 * ffn, rank, scale, row_adapter)
    branch = lora_bits(o.swiglu_bf16(fused, rows, ffn), c["fc2_weight"], pairs["fc2"], rows, ffn, hidden, rank, scale, row_adapter)
    want = o.gate_bf16(gated, branch, c["modulation"], case.row_map, rows, hidden, 6, 5)
    assert_block_close(got, want, "block with adapters and conditioning")
    without = o.dit_block(case.hidden, c, case.row_map, case.rope_cos, case.rope_sin, rows=rows, width=hidden, heads=heads,
                          head_dim=128, ffn=ffn, rope_half=48, round_p=1)
    assert_block_close(plain, without, "the plain block afterwards")


def test_conditioning_without_requests_adds_nothing(pkg):
    gpu = pkg.Gpu(0)
    try:
        shape = pkg.DitShape(hidden=64, heads=2, ffn=32, blocks=1)
        cond = pkg.Conditioning(gpu, shape, rows=5, states=3, segments=[])
        rng = np.random.default_rng(1)
        query, heads = gpu.bf16(bits(rng, 5 * 256)), bits(rng, 5 * 256)
        out = gpu.bf16(heads)
        gpu.begin()
        cond.add_block(gpu.bf16(bits(rng, 3, 32)), 32, gpu.bf16(bits(rng, 256, 32)), gpu.bf16(bits(rng, 256, 32)))
        cond.attend(0, query, out)
        gpu.submit()
        assert np.array_equal(out.read(), heads)
    finally:
        gpu.close()


@pytest.mark.parametrize("rows,rank", [(1, 16), (70, 12), (640, 16)])
def test_a_chain_of_calls_equals_the_calls_one_by_one(pkg, rows, rank):
    """Every call reads what the one in front of it wrote (their launches may begin before it has ended), the table
    and the row map included: the same bits as with the stream drained in between."""
    heads, adapters, states, steps = 8, 3, 700, 12
    width = heads * 128
    rng = np.random.default_rng([rows, rank])
    gpu = pkg.Gpu(0)
    try:
        w, down, up = (gpu.bf16(bits(rng, width, width, std=width ** -0.5)), gpu.bf16(bits(rng, adapters, rank, width, std=width ** -0.5)),
                       gpu.bf16(bits(rng, adapters, width, rank, std=0.1)))
        key, value = gpu.bf16(bits(rng, states, width)), gpu.bf16(bits(rng, states, width))
        start = bits(rng, rows, width)
        maps = [gpu.u32(rng.integers(0, adapters + 1, rows).astype(np.uint32)) for _ in range(steps)]
        tables = [gpu.u32(np.array([[0, rows, 0, 1 + 17 * i], [0, 0, 0, 0]], np.uint32).reshape(-1)) for i in range(steps)]
        row_map, table = gpu.u32(np.zeros(rows, np.uint32)), gpu.u32(np.zeros(8, np.uint32))
        x, y, z = (gpu.new(rows * width, pkg.BF16) for _ in range(3))
        words = lambda t: gpu.wrap(t.pointer, t.elements, pkg.F32)          # for the copies

        def run(drain):
            x.write(start)
            gpu.begin()

            def op(*args):
                gpu.op(*args)
                if drain:
                    gpu.submit()
                    gpu.begin()
            for i in range(steps):
                op("copy_f32", words(row_map), 0, words(maps[i]), 0, rows)
                op("h3x_linear_lora_bf16", y, x, w, None, down, up, None, row_map, rows, width, width, adapters, rank)
                op("copy_f32", words(table), 0, words(tables[i]), 0, 8)
                op("h3x_cross_sdpa_bf16", z, y, key, value, table, 2, rows, states, heads, heads, 128, 128 ** -0.5)
                op("h3x_cross_sdpa_bf16", y, z, key, value, table, 2, rows, states, heads, heads, 128, 128 ** -0.5)
                op("h3x_linear_lora_bf16", z, y, w, None, down, up, None, row_map, rows, width, width, adapters, rank)
                op("add_bf16", x, x, z, rows * width)
            gpu.submit()
            return x.read()
        want = run(True)
        for _ in range(3):
            assert np.array_equal(run(False), want)
    finally:
        gpu.close()


def test_two_contexts_at_once(pkg):
    """Calls of every kind in two contexts on two streams, interleaved without a wait: the bits of each on its own."""
    import torch
    rng = np.random.default_rng(5)
    contexts = [pkg.Gpu(0), pkg.Gpu(0)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    try:
        calls = []          # per context: (name, arguments, output)
        for gpu, stream in zip(contexts, streams):
            gpu.set_stream(stream.cuda_stream)
            mine = []
            for rows, k, n, adapters, rank in ((640, 1024, 1536, 3, 16), (3, 1024, 1024, 3, 8), (100, 2048, 1024, 3, 64), (300, 1000, 520, 2, 12)):
                out = gpu.new(rows * n, pkg.BF16)
                mine.append(("h3x_linear_lora_bf16", (out, gpu.bf16(bits(rng, rows, k)), gpu.bf16(bits(rng, n, k, std=k ** -0.5)), None,
                                                      gpu.bf16(bits(rng, adapters, rank, k, std=k ** -0.5)),
                                                      gpu.bf16(bits(rng, adapters, n, rank, std=0.1)), None,
                                                      gpu.u32(rng.integers(0, adapters + 1, rows).astype(np.uint32)), rows, k, n,
                                                      adapters, rank), out))
            for segments, heads, kv_heads, dim in (([[0, 700, 0, 300], [700, 90, 300, 77]], 8, 8, 128), ([[0, 1, 0, 2000], [1, 1, 40, 5]], 8, 2, 128),
                                                   ([[0, 400, 0, 260]], 6, 6, 64)):
                rows, keys = max(s[0] + s[1] for s in segments), max(s[2] + s[3] for s in segments)
                out = gpu.new(rows * heads * dim, pkg.BF16)
                mine.append(("h3x_cross_sdpa_bf16", (out, gpu.bf16(bits(rng, rows, heads * dim)), gpu.bf16(bits(rng, keys, kv_heads * dim)),
                                                     gpu.bf16(bits(rng, keys, kv_heads * dim)),
                                                     gpu.u32(np.array(segments, np.uint32).reshape(-1)), len(segments), rows, keys, heads,
                                                     kv_heads, dim, dim ** -0.5), out))
            calls.append(mine)
        want = []
        for gpu, mine in zip(contexts, calls):
            gpu.begin()
            for name, args, _ in mine:
                gpu.op(name, *args)
            gpu.submit()
            want.append([out.read() for _, _, out in mine])
        for gpu in contexts:
            gpu.begin()
        for turn in range(30):
            for i in range(len(calls[0])):
                for c, gpu in enumerate(contexts):
                    name, args, _ = calls[c][(i + 3 * c + turn) % len(calls[c])]
                    gpu.op(name, *args)
        for gpu in contexts:
            gpu.submit()
        for c in range(2):
            for (name, _, out), bits_alone in zip(calls[c], want[c]):
                assert np.array_equal(out.read(), bits_alone), name
    finally:
        for gpu in contexts:
            gpu.close()
