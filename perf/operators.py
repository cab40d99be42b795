"""What is measured of the adapter and conditioning operators.

  lora   low-rank adapters of many requests beside a shared projection (h3x_linear_lora_bf16)
  cross  attention of query rows to an encoder's states of another length (h3x_cross_sdpa_bf16)

`run` computes an operator in its plain form from elementary torch operations, or, where `own` is
true, through the framework's entry points.
"""
import math
import random

import torch

own = False

NONE = -1          # as a U32 row map entry: 0xffffffff, a row without an adapter


# ------------------------------------------------------------------------------------ the cases

def listed():
    return [
        # one row: the smallest call there is, a single conditioning token through an output projection
        dict(name="lora one row", op="lora", rows=1, k=7168, n=5376, adapters=4, rank=16, runs=1, bias=True),
        # time rows of a 20-step schedule through one block's modulation projection
        dict(name="lora time rows", op="lora", rows=42, k=2688, n=96768, adapters=2, rank=32, runs=3, bias=True),
        # text rows of sixteen requests through the projection into the model width
        dict(name="lora text rows", op="lora", rows=1003, k=5120, n=5376, adapters=16, rank=12, runs=17, bias=True),
        # output projection of one small video, three customers' adapters in one batch
        dict(name="lora out projection", op="lora", rows=1664, k=7168, n=5376, adapters=3, rank=64, runs=5, bias=False),
        # the MLP's second projection at one rank's share of an eight-way sharded video
        dict(name="lora mlp share", op="lora", rows=800, k=14336, n=5376, adapters=8, rank=128, runs=2, bias=False),
        # QKV projection of a whole video with two adapters and rows that have none
        dict(name="lora qkv", op="lora", rows=6400, k=5376, n=21504, adapters=2, rank=64, runs=3, bias=False),
        # single rows of four requests over states of several lengths
        dict(name="cross single rows", op="cross", queries="1,1,1,1", keys="512,77,2048,1", pad=0,
             heads=56, kv_heads=56, dim=128),
        # narrow heads that share keys, states of one short prompt
        dict(name="cross shared keys", op="cross", queries="1797", keys="77", pad=0, heads=32, kv_heads=8, dim=64),
        # image states of one small video
        dict(name="cross image states", op="cross", queries="1664", keys="257", pad=0, heads=24, kv_heads=24, dim=128),
        # a ragged batch over states padded to one length, one request without states
        dict(name="cross ragged batch", op="cross", queries="1600,301,2122,1,800,640", keys="512,77,333,129,0,256",
             pad=512, heads=56, kv_heads=56, dim=128),
        # a whole video over the states of a long prompt
        dict(name="cross video", op="cross", queries="6400", keys="512", pad=0, heads=56, kv_heads=56, dim=128),
        # the long video
        dict(name="cross long video", op="cross", queries="50476", keys="512", pad=0, heads=56, kv_heads=56, dim=128),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    if rng.random() < 0.5:
        most = 6400 * 5376 * 21504
        while True:
            k, n = rng.choice([(5376, 21504), (7168, 5376), (5376, 28672), (14336, 5376), (5120, 5376), (2688, 10752),
                               (8 * _log(rng, 32, 1024), 8 * _log(rng, 32, 1024))])
            rows = _log(rng, 1, 6400)
            if rows * k * n <= most:
                break
        rank = rng.choice([4, 7, 8, 12, 16, 20, 32, 48, 64, 100, 128])
        return dict(op="lora", rows=rows, k=k, n=n, adapters=rng.randint(1, 16), rank=rank,
                    runs=rng.randint(1, min(rows, 24)), bias=rng.random() < 0.5)
    while True:
        count = rng.randint(1, 10)
        queries = [_log(rng, 1, 8000) if rng.random() < 0.8 else rng.randint(1, 4) for _ in range(count)]
        keys = [0 if rng.random() < 0.05 else _log(rng, 1, 2048) for _ in range(count)]
        heads, kv_heads = rng.choice([(56, 56), (24, 24), (32, 8), (32, 32), (16, 2), (28, 4), (12, 4)])
        if max(keys) and count * max(queries) * max(keys) * heads <= 50476 * 512 * 56:
            break
    return dict(op="cross", queries=",".join(map(str, queries)), keys=",".join(map(str, keys)),
                pad=max(keys) if rng.random() < 0.5 else 0, heads=heads, kv_heads=kv_heads, dim=rng.choice([64, 128]))


# ----------------------------------------------------------------------------------- their data

def _row_adapters(case):
    """Contiguous runs of rows, one per request: run i has adapter i, the one after the last has none."""
    rows, runs, adapters = case["rows"], case["runs"], case["adapters"]
    cuts = sorted(random.Random(rows * 31 + runs).sample(range(1, rows), runs - 1)) if runs > 1 else []
    edges = [0] + cuts + [rows]
    out = []
    for i in range(runs):
        which = i % (adapters + 1)
        out += [which if which < adapters else NONE] * (edges[i + 1] - edges[i])
    return out


def _segments(case):
    """[first query row, query rows, first key row, key rows] of every request, packed query rows; key
    rows packed, or (pad) every request's states padded to one length."""
    out, q, k = [], 0, 0
    for a, b in zip(map(int, case["queries"].split(",")), map(int, case["keys"].split(","))):
        out.append([q, a, k, b])
        q += a
        k += case["pad"] or b
    return out, q, max(1, k)


_context = None


def _gpu():
    """The program's one context, with its command open."""
    global _context
    if _context is None:
        from __graft_entry__ import load_package
        package = load_package()
        _context = package, package.Gpu(0)
        _context[1].begin()
    return _context


def _normal(generator, *shape, std=1.0):
    return (torch.randn(shape, device="cuda", generator=generator) * std).to(torch.bfloat16)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "lora":
        rows, k, n, adapters, rank = (case[v] for v in ("rows", "k", "n", "adapters", "rank"))
        s = dict(case=case, x=_normal(g, rows, k), weight=_normal(g, n, k, std=0.02),
                 bias=_normal(g, n, std=0.1) if case["bias"] else None,
                 down=_normal(g, adapters, rank, k, std=k ** -0.5), up=_normal(g, adapters, n, rank, std=0.05),
                 scale=torch.rand(adapters, device="cuda", generator=g) + 0.5,
                 row_adapter=torch.tensor(_row_adapters(case), dtype=torch.int32, device="cuda"),
                 out=torch.empty(rows, n, dtype=torch.bfloat16, device="cuda"))
        kinds = dict(scale="F32", row_adapter="U32")
    else:
        segments, q_rows, k_rows = _segments(case)
        heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
        # one row more than there are: where the plain form puts what belongs nowhere
        s = dict(case=case, q=_normal(g, q_rows, heads, dim), key=_normal(g, k_rows, kv_heads, dim),
                 value=_normal(g, k_rows, kv_heads, dim), segments=torch.tensor(segments, dtype=torch.int32, device="cuda"),
                 out=torch.zeros(q_rows + 1, heads, dim, dtype=torch.bfloat16, device="cuda"),
                 most_queries=max(a[1] for a in segments), most_keys=max(a[3] for a in segments), count=len(segments))
        kinds = dict(segments="U32")
    if own:
        package, gpu = _gpu()
        s["gpu"] = gpu
        s["tensors"] = {name: gpu.wrap(t.data_ptr(), t.numel(), getattr(package, kinds.get(name, "BF16")))
                        for name, t in s.items() if isinstance(t, torch.Tensor)}
    return s


# ------------------------------------------------------------------------------------ one pass

def _lora_plain(s):
    x, own_adapter = s["x"].float(), s["row_adapter"].long()
    adapters, rank, k = s["down"].shape
    y = x @ s["weight"].float().T
    if s["bias"] is not None:
        y = y + s["bias"].float()
    low = (x @ s["down"].float().reshape(adapters * rank, k).T).view(-1, adapters, rank)
    mine = own_adapter[:, None] == torch.arange(adapters, device=x.device)
    low = low * (mine * s["scale"]).unsqueeze(2)
    y = y + low.reshape(-1, adapters * rank) @ s["up"].float().permute(0, 2, 1).reshape(adapters * rank, -1)
    s["out"].copy_(y)
    return s["out"]


def _cross_plain(s):
    q, key, value, seg = s["q"].float(), s["key"].float(), s["value"].float(), s["segments"].long()
    q_rows, heads, dim = q.shape
    group = heads // key.shape[1]
    at_q = torch.arange(s["most_queries"], device=q.device)
    at_k = torch.arange(s["most_keys"], device=q.device)
    live_q, live_k = at_q < seg[:, 1:2], at_k < seg[:, 3:4]
    rows_q = torch.where(live_q, seg[:, 0:1] + at_q, q_rows)
    rows_k = torch.where(live_k, seg[:, 2:3] + at_k, 0)
    qs = q[rows_q.clamp(max=q_rows - 1)].transpose(1, 2)                     # [segment][head][row][dim]
    ks = key[rows_k].transpose(1, 2).repeat_interleave(group, 1)
    vs = value[rows_k].transpose(1, 2).repeat_interleave(group, 1)
    scores = qs @ ks.transpose(2, 3) * dim ** -0.5
    dead = ~live_k[:, None, None, :]
    scores = scores.masked_fill(dead, -math.inf)
    most = scores.amax(3, keepdim=True)
    weights = torch.exp(scores - torch.where(most == -math.inf, 0.0, most))
    total = weights.sum(3, keepdim=True)
    result = (weights @ vs) / torch.where(total == 0, 1.0, total)
    s["out"][rows_q] = result.transpose(1, 2).to(torch.bfloat16)
    return s["out"][:q_rows]


def run(state):
    case = state["case"]
    if not own:
        return _lora_plain(state) if case["op"] == "lora" else _cross_plain(state)
    gpu, t = state["gpu"], state["tensors"]
    if case["op"] == "lora":
        gpu.op("h3x_linear_lora_bf16", t["out"], t["x"], t["weight"], t.get("bias"), t["down"], t["up"], t["scale"],
               t["row_adapter"], case["rows"], case["k"], case["n"], case["adapters"], case["rank"])
        return state["out"]
    q_rows, k_rows = state["q"].shape[0], state["key"].shape[0]
    gpu.op("h3x_cross_sdpa_bf16", t["out"], t["q"], t["key"], t["value"], t["segments"], state["count"], q_rows, k_rows,
           case["heads"], case["kv_heads"], case["dim"], case["dim"] ** -0.5)
    return state["out"][:q_rows]


def work(case):
    if case["op"] == "lora":
        rows, k, n, rank = (case[v] for v in ("rows", "k", "n", "rank"))
        which = _row_adapters(case)
        used = len({a for a in which if a != NONE})
        with_one = sum(a != NONE for a in which)
        return dict(bytes=2 * (rows * k + n * k + rows * n + used * rank * (k + n) + (n if case["bias"] else 0)) + 4 * rows,
                    flops=2 * rows * k * n + 2 * with_one * rank * (k + n))
    segments, q_rows, _ = _segments(case)
    keys = sum(a[3] for a in segments)
    pairs = sum(a[1] * a[3] for a in segments)
    return dict(bytes=2 * case["dim"] * (2 * q_rows * case["heads"] + 2 * keys * case["kv_heads"]),
                flops=4 * pairs * case["heads"] * case["dim"])


# ------------------------------------------------------------------------- the definition, 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "lora":
        out = torch.empty(case["rows"], case["n"], dtype=torch.float64, device="cuda")
        weight = s["weight"].double()
        which = s["row_adapter"].tolist()
        for r0 in range(0, case["rows"], 1024):                 # the projection, some rows at a time
            out[r0:r0 + 1024] = torch.matmul(s["x"][r0:r0 + 1024].double(), weight.t())
        if s["bias"] is not None:
            out += s["bias"].double()
        for a in sorted(set(which) - {NONE}):                   # every adapter on the rows that have it
            at = torch.tensor([r for r, b in enumerate(which) if b == a], device="cuda")
            low = torch.matmul(s["x"][at].double(), s["down"][a].double().t())
            out[at] += torch.matmul(low, s["up"][a].double().t()) * s["scale"][a].double()
        return out
    segments, q_rows, _ = _segments(case)
    heads, group = case["heads"], case["heads"] // case["kv_heads"]
    out = torch.zeros(q_rows, heads, case["dim"], dtype=torch.float64, device="cuda")
    for q0, queries, k0, keys in segments:
        if not keys:
            continue
        for h in range(heads):
            k64, v64 = (s[name][k0:k0 + keys, h // group].double() for name in ("key", "value"))
            for r0 in range(q0, q0 + queries, 16384):
                r1 = min(r0 + 16384, q0 + queries)
                weights = torch.softmax(s["q"][r0:r1, h].double() @ k64.t() / math.sqrt(case["dim"]), dim=1)
                out[r0:r1, h] = weights @ v64
    return out
