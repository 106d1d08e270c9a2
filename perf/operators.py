"""The operators that a decoder graph adds to this package's encoders, as cases that can be timed and compared.

  linear  MatMulNBits            rows times a matrix that is held in 4 bits with a scale for each group of inputs
  append  OxiPagedCacheAppend    rotates the new tokens' queries and keys by their positions and puts keys and values
                                 into the pages of a cache
  attend  OxiPagedAttention      causal attention of packed sequences' new tokens over the pages of such a cache

`own` false computes them from elementary torch operations, true through planned sessions whose inputs and outputs are
bound to device buffers and which are enqueued on the caller's stream.
"""
import math
import random

import numpy as np
import torch

own = False

TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def listed():
    return [
        # one token of a decoding program through a feed-forward layer: nothing but the weights to read
        {"name": "linear one token", "op": "linear", "rows": 1, "k": 4096, "n": 16384, "group": 128, "type": "bfloat16", "zero_points": True, "bias": False, "mix": 0},
        # a few rows through an odd layer of a float graph, the last group of a row half empty
        {"name": "linear odd f32", "op": "linear", "rows": 5, "k": 1000, "n": 1111, "group": 32, "type": "float32", "zero_points": True, "bias": True, "mix": 0},
        # a token of each of 32 streams, weights around a fixed zero point
        {"name": "linear 32 streams", "op": "linear", "rows": 32, "k": 4096, "n": 4096, "group": 32, "type": "float16", "zero_points": False, "bias": False, "mix": 0},
        # the rows of a prompt
        {"name": "linear prompt", "op": "linear", "rows": 2048, "k": 4096, "n": 4096, "group": 128, "type": "bfloat16", "zero_points": False, "bias": True, "mix": 0},
        # one decoding step of 64 streams
        {"name": "append 64 streams", "op": "append", "sequences": 64, "tokens": 64, "past": 4000, "heads": 32, "kv_heads": 8, "size": 128, "rotary": 128,
         "interleaved": False, "page": 16, "type": "bfloat16", "packed": False, "mix": 1},
        # the prompts of six streams out of one product, a rotation of half of each head
        {"name": "append prompts", "op": "append", "sequences": 6, "tokens": 8100, "past": 500, "heads": 16, "kv_heads": 16, "size": 64, "rotary": 32,
         "interleaved": True, "page": 64, "type": "float16", "packed": True, "mix": 2},
        # a decoding step of four short streams: latency
        {"name": "attend 4 short streams", "op": "attend", "sequences": 4, "tokens": 4, "past": 700, "heads": 12, "kv_heads": 12, "size": 64, "page": 16,
         "type": "float16", "mix": 3},
        # a decoding step of 64 streams of very different lengths
        {"name": "attend 64 streams", "op": "attend", "sequences": 64, "tokens": 64, "past": 8100, "heads": 32, "kv_heads": 8, "size": 128, "page": 64,
         "type": "bfloat16", "mix": 4},
        # a decoding step of one stream with a long past
        {"name": "attend one long stream", "op": "attend", "sequences": 1, "tokens": 1, "past": 131000, "heads": 32, "kv_heads": 8, "size": 128, "page": 128,
         "type": "bfloat16", "mix": 5},
        # a batch of prompts, packed
        {"name": "attend packed prompts", "op": "attend", "sequences": 7, "tokens": 8000, "past": 0, "heads": 32, "kv_heads": 8, "size": 128, "page": 16,
         "type": "bfloat16", "mix": 6},
        # one long prompt
        {"name": "attend one prompt", "op": "attend", "sequences": 1, "tokens": 8192, "past": 0, "heads": 32, "kv_heads": 8, "size": 128, "page": 64,
         "type": "bfloat16", "mix": 7},
        # prompts that are taken in pieces: new tokens behind a past; five heads share a key head, heads of 96
        {"name": "attend pieces of prompts", "op": "attend", "sequences": 3, "tokens": 1500, "past": 6000, "heads": 20, "kv_heads": 4, "size": 96, "page": 32,
         "type": "float16", "mix": 8},
    ]


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "append", "attend", "attend", "attend"])
    mix = rng.randrange(1 << 20)
    if op == "linear":
        kind = rng.choice(["float32", "float16", "float16", "bfloat16", "bfloat16"])
        k = _log(rng, 64, 8192)
        n = _log(rng, 64, min(16384, 33_000_000 // k))
        rows = _log(rng, 1, 64 if kind == "float32" else 2048)
        if rng.random() < 0.5:
            k, n = -(-k // 64) * 64, -(-n // 64) * 64
        return {"op": op, "rows": rows, "k": k, "n": n, "group": rng.choice([16, 32, 32, 64, 128, 128]), "type": kind, "zero_points": rng.random() < 0.5,
                "bias": rng.random() < 0.3, "mix": mix}
    size = rng.choice([64, 64, 80, 96, 128, 128, 128])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 4, 5, 8])
    page = rng.choice([16, 16, 32, 64, 128])
    case = {"op": op, "heads": heads, "kv_heads": kv_heads, "size": size, "page": page, "type": rng.choice(["float16", "bfloat16"]), "mix": mix}
    if op == "append":
        sequences = _log(rng, 1, 64)
        tokens = sequences if rng.random() < 0.4 else _log(rng, sequences, 8000)
        return {**case, "sequences": sequences, "tokens": tokens, "past": rng.choice([0, _log(rng, 1, 4000)]), "rotary": rng.choice([size, size, size // 2]),
                "interleaved": rng.random() < 0.5, "packed": rng.random() < 0.5}
    kind = rng.choice(["steps", "steps", "prompts", "pieces"])
    if kind == "steps":  # a token of each stream, at times two or three that were guessed ahead
        sequences = _log(rng, 1, 64)
        return {**case, "sequences": sequences, "tokens": sequences * rng.choice([1, 1, 1, 2, 3]), "past": _log(rng, 16, min(60000, 400_000 // sequences))}
    sequences = _log(rng, 1, 8)
    tokens = _log(rng, sequences * 4, 4000)
    return {**case, "sequences": sequences, "tokens": tokens, "past": 0 if kind == "prompts" else _log(rng, 16, 4000)}


def _lengths(case):
    """New tokens of each sequence, and how many it has with them: both follow from the case alone."""
    rng = random.Random(case["mix"])
    count, tokens = case["sequences"], case["tokens"]
    if tokens % count == 0 and tokens // count < 4:
        new = [tokens // count] * count
    else:
        share = [rng.uniform(0.1, 1.0) for _ in range(count)]
        new = [1 + int((tokens - count) * s / sum(share)) for s in share]
        new[0] += tokens - sum(new)
    past = [case["past"]] + [int(case["past"] * rng.uniform(0.05, 1.0)) for _ in range(count - 1)]
    return new, [n + p for n, p in zip(new, past)]


def work(case):
    if case["op"] == "linear":
        rows, k, n, size = case["rows"], case["k"], case["n"], TYPES[case["type"]].itemsize
        groups = n * -(-k // case["group"])
        weights = n * k // 2 + 2 * groups + (groups // 2 if case["zero_points"] else 0) + (4 * n if case["bias"] else 0)
        return {"bytes": weights + rows * (k + n) * size, "flops": 2 * rows * k * n}
    new, total = _lengths(case)
    heads, kv_heads, size = case["heads"], case["kv_heads"], case["size"]
    if case["op"] == "append":
        tokens = case["tokens"]
        return {"bytes": 2 * tokens * (heads + 2 * kv_heads) * size * 2 + tokens * case["rotary"] * 4, "flops": tokens * (heads + kv_heads) * case["rotary"] * 3}
    pairs = sum(n * (t - n) + n * (n + 1) // 2 for n, t in zip(new, total))
    return {"bytes": 2 * case["tokens"] * heads * size * 2 + sum(total) * kv_heads * size * 2 * 2, "flops": 4 * pairs * heads * size}


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = TYPES[case["type"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(kind)

    if case["op"] == "linear":
        rows, k, n, group = case["rows"], case["k"], case["n"], case["group"]
        blocks = -(-k // group)
        s = {"x": normal(rows, k),
             "weights": torch.randint(0, 256, (n, blocks, group // 2), generator=gen, device="cuda", dtype=torch.uint8),
             "scales": ((torch.rand(n, blocks, generator=gen, device="cuda") + 0.5) * (0.2 / math.sqrt(k))).half()}
        if case["zero_points"]:  # two to a byte, around the middle of the range
            nibbles = torch.randint(5, 11, (n, blocks + blocks % 2), generator=gen, device="cuda", dtype=torch.uint8)
            s["zero_points"] = nibbles[:, 0::2] | (nibbles[:, 1::2] << 4)
        if case["bias"]:
            s["bias"] = torch.randn(n, generator=gen, device="cuda")
        return s

    new, total = _lengths(case)
    page, size, kv_heads = case["page"], case["size"], case["kv_heads"]
    used = [-(-t // page) for t in total]
    pages = sum(used) + 3
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(new), max(used) + 1), -1, device="cuda", dtype=torch.int32)
    at = torch.arange(max(used) + 1, device="cuda")
    filled = at[None, :] < torch.tensor(used, device="cuda")[:, None]
    table[filled] = order[: sum(used)]
    s = {"query": normal(case["tokens"], case["heads"] * size),
         "key_cache": normal(pages, page, kv_heads, size),
         "value_cache": normal(pages, page, kv_heads, size),
         "cu_query": torch.tensor([0] + list(np.cumsum(new)), device="cuda", dtype=torch.int32),
         "kv_lengths": torch.tensor(total, device="cuda", dtype=torch.int32),
         "page_table": table}
    if case["op"] == "append":
        if case["packed"]:
            s["query"] = normal(case["tokens"], (case["heads"] + 2 * kv_heads) * size)
        else:
            s["key"], s["value"] = normal(case["tokens"], kv_heads * size), normal(case["tokens"], kv_heads * size)
        positions, half = -(-max(total) // 1024) * 1024, case["rotary"] // 2
        angles = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
        s["cos"], s["sin"] = angles.cos().float(), angles.sin().float()
    return s


def _session(nodes, state, inputs, outputs, weights):
    """The planned session of `nodes` with `state`'s tensors bound to its inputs and outputs."""
    from oxionnx_b200.graph import Graph, Node
    from oxionnx_b200.session import Session

    def name(t):
        return str(t.dtype).replace("torch.", "")

    graph = Graph(nodes=[Node(*n) for n in nodes], input_names=inputs, output_names=list(outputs))
    session = (Session.builder().with_input_types({i: name(state[i]) for i in inputs})
               .with_input_shapes({i: tuple(state[i].shape) for i in inputs})
               .build_from_graph(graph, {w: state[w].cpu().numpy() for w in weights}))
    session.ensure_planned()
    for i in inputs:
        session.bind_input_device(i, state[i].data_ptr(), name(state[i]), state[i].numel())
    for o, tensor in outputs.items():
        session.bind_output_device(o, tensor.data_ptr(), tensor.numel(), name(tensor))
    return session


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    new, total = _lengths(case) if case["op"] != "linear" else ([], [])
    state["longest"] = (max(new, default=0), max(total, default=0))  # the program that made the lengths knows them
    if own:
        if case["op"] == "linear":
            state["y"] = torch.empty(case["rows"], case["n"], device="cuda", dtype=TYPES[case["type"]])
            weights = [w for w in ("weights", "scales", "zero_points", "bias") if w in state]
            names = ["x"] + [w if w in state else "" for w in ("weights", "scales", "zero_points")] + ["", "bias"] * ("bias" in state)
            nodes = [("MatMulNBits", "linear", names, ["y"], {"K": case["k"], "N": case["n"], "bits": 4, "block_size": case["group"]})]
            state["session"] = _session(nodes, state, ["x"], {"y": state["y"]}, weights)
            return state
        heads = {"num_heads": case["heads"], "kv_num_heads": case["kv_heads"]}
        tables = ["cu_query", "kv_lengths", "page_table"]
        if case["op"] == "append":
            state["rotated"] = torch.empty(case["tokens"], case["heads"] * case["size"], device="cuda", dtype=TYPES[case["type"]])
            new = ["query"] if case["packed"] else ["query", "key", "value"]
            names = ["query", *(("", "") if case["packed"] else ("key", "value")), "key_cache", "value_cache", *tables, "cos", "sin"]
            nodes = [("OxiPagedCacheAppend", "append", names, ["rotated", "key_cache_out", "value_cache_out"], {**heads, "interleaved": int(case["interleaved"])})]
            state["session"] = _session(nodes, state, [*new, "key_cache", "value_cache", *tables], {"rotated": state["rotated"]}, ["cos", "sin"])
            return state
        state["out"] = torch.empty_like(state["query"])
        names = ["query", "key_cache", "value_cache", *tables]
        nodes = [("OxiPagedAttention", "attend", names, ["out"], {**heads, "max_query_length": max(new)})]
        state["session"] = _session(nodes, state, names, {"out": state["out"]}, [])
    return state


def _linear(s):
    case = s["case"]
    n, k, group = case["n"], case["k"], case["group"]
    q = torch.stack((s["weights"] & 15, s["weights"] >> 4), -1).reshape(n, -1, group).float()
    zero = 8.0
    if "zero_points" in s:
        zero = torch.stack((s["zero_points"] & 15, s["zero_points"] >> 4), -1).reshape(n, -1)[:, : q.shape[1], None].float()
    w = ((q - zero) * s["scales"].float()[:, :, None]).reshape(n, -1)[:, :k]
    y = s["x"].float() @ w.t()
    if "bias" in s:
        y = y + s["bias"]
    return y.to(s["x"].dtype)


def _rows(s):
    """Sequence and position of each new token."""
    cu, total = s["cu_query"].long(), s["kv_lengths"].long()
    token = torch.arange(s["case"]["tokens"], device="cuda")
    b = torch.searchsorted(cu, token, right=True) - 1
    return b, total[b] - cu[b + 1] + token


def _rotate(x, cos, sin, interleaved):
    half = cos.shape[-1]
    part = x[..., : 2 * half].float()
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :half], part[..., half:])
    a, b = a * cos - b * sin, b * cos + a * sin
    part = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((part.to(x.dtype), x[..., 2 * half :]), -1)


def _append(s):
    case = s["case"]
    heads, kv_heads, size, page = case["heads"], case["kv_heads"], case["size"], case["page"]
    q, k, v = (s["query"], s["key"], s["value"]) if "key" in s else s["query"].split((heads * size, kv_heads * size, kv_heads * size), -1)
    b, position = _rows(s)
    cos, sin = s["cos"][position][:, None, :], s["sin"][position][:, None, :]
    slot = s["page_table"][b, position // page].long() * page + position % page
    s["key_cache"].view(-1, kv_heads, size)[slot] = _rotate(k.reshape(-1, kv_heads, size), cos, sin, case["interleaved"])
    s["value_cache"].view(-1, kv_heads, size)[slot] = v.reshape(-1, kv_heads, size)
    return _rotate(q.reshape(-1, heads, size), cos, sin, case["interleaved"]).flatten(1), s["key_cache"], s["value_cache"]


def _attend(s):
    case = s["case"]
    heads, kv_heads, size = case["heads"], case["kv_heads"], case["size"]
    group, (rows, length) = heads // kv_heads, s["longest"]
    count, kind = case["sequences"], s["query"].dtype
    cu, total = s["cu_query"].long(), s["kv_lengths"].long()
    b, position = _rows(s)
    row = torch.arange(case["tokens"], device="cuda") - cu[b]
    q = torch.zeros(count, rows, heads, size, device="cuda")  # every sequence padded to the longest
    q[b, row] = s["query"].view(-1, heads, size).float()
    q = q.view(count, rows, kv_heads, group, size).permute(0, 2, 3, 1, 4).reshape(count, kv_heads, group * rows, size)
    j = torch.arange(length, device="cuda")
    held = (j < total[:, None])[:, :, None, None]
    pages = s["page_table"].long().clamp(min=0)

    def rows_of(cache):
        x = cache[pages].reshape(count, -1, kv_heads, size)[:, :length].float()
        return torch.where(held, x, 0.0).transpose(1, 2)

    scores = (q @ rows_of(s["key_cache"]).transpose(2, 3)).view(count, kv_heads, group, rows, length) * (1.0 / math.sqrt(size))
    last = (total - (cu[1:] - cu[:-1]))[:, None] + torch.arange(rows, device="cuda")
    scores = scores.masked_fill_((j > last[:, :, None])[:, None, None], -math.inf)
    scores = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    weight = scores.sum(-1, keepdim=True)
    out = (scores.view(count, kv_heads, group * rows, length) @ rows_of(s["value_cache"])).view(count, kv_heads, group, rows, size) / weight
    return out.permute(0, 3, 1, 2, 4).reshape(count, rows, heads * size)[b, row].to(kind)


def run(state):
    op = state["case"]["op"]
    if own:
        state["session"].enqueue(torch.cuda.current_stream().cuda_stream)
        if op == "append":
            return state["rotated"], state["key_cache"], state["value_cache"]
        return state["y" if op == "linear" else "out"]
    return {"linear": _linear, "append": _append, "attend": _attend}[op](state)


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "linear":
        # y[m, j] = sum over groups of scale * (sum of x * code - zero * sum of x), column blocks at a time
        x = torch.nn.functional.pad(s["x"].double(), (0, -case["k"] % case["group"]))
        x = x.view(case["rows"], -1, case["group"]).transpose(0, 1)  # group, row, lane
        y = []
        for first in range(0, case["n"], 512):
            part = slice(first, min(first + 512, case["n"]))
            code = torch.empty(*s["weights"][part].shape, 2, device="cuda", dtype=torch.float64)
            code[..., 0], code[..., 1] = s["weights"][part] % 16, s["weights"][part] // 16
            code = code.flatten(-2)
            zero = torch.full(code.shape[:2], 8.0, device="cuda", dtype=torch.float64)
            if "zero_points" in s:
                z = s["zero_points"][part]
                zero[:, 0::2] = (z % 16)[:, : zero[:, 0::2].shape[1]].double()
                zero[:, 1::2] = (z // 16)[:, : zero[:, 1::2].shape[1]].double()
            scale = s["scales"][part].double()
            y.append((torch.bmm(x, (code * scale[:, :, None]).permute(1, 2, 0)) - x.sum(-1)[:, :, None] * (zero * scale).t()[:, None, :]).sum(0))
        y = torch.cat(y, 1)
        return y + s["bias"].double() if "bias" in s else y

    new, total = _lengths(case)
    heads, kv_heads, size, page = case["heads"], case["kv_heads"], case["size"], case["page"]
    if case["op"] == "append":
        width = case["rotary"]
        parts = [s["query"].double()] if case["packed"] else [s["query"].double(), s["key"].double(), s["value"].double()]
        lanes = torch.cat(parts, 1).view(case["tokens"], heads + 2 * kv_heads, size)
        keys, values = s["key_cache"].double(), s["value_cache"].double()
        first = 0
        for b in range(case["sequences"]):
            at = torch.arange(total[b] - new[b], total[b], device="cuda")
            turn = torch.complex(s["cos"][at].double(), s["sin"][at].double())[:, None, :]
            some = lanes[first : first + new[b], : heads + kv_heads, :width]
            half = some.reshape(*some.shape[:2], width // 2, 2) if case["interleaved"] else torch.stack((some[..., : width // 2], some[..., width // 2 :]), -1)
            half = torch.view_as_real(torch.view_as_complex(half.contiguous()) * turn)
            some.copy_(half.flatten(-2) if case["interleaved"] else torch.cat((half[..., 0], half[..., 1]), -1))
            held = s["page_table"][b, at // page].long()
            keys[held, at % page] = lanes[first : first + new[b], heads : heads + kv_heads]
            values[held, at % page] = lanes[first : first + new[b], heads + kv_heads :]
            first += new[b]
        return lanes[:, :heads].flatten(1), keys, values

    out = torch.empty(case["tokens"], heads, size, device="cuda", dtype=torch.float64)
    query = s["query"].double().view(-1, heads, size)
    first = 0
    for b in range(case["sequences"]):
        held = s["page_table"][b, : -(-total[b] // page)].long()
        for h in range(heads):
            k = s["key_cache"][held, :, h // (heads // kv_heads)].flatten(0, 1)[: total[b]].double()
            v = s["value_cache"][held, :, h // (heads // kv_heads)].flatten(0, 1)[: total[b]].double()
            logits = torch.einsum("id,jd->ij", query[first : first + new[b], h], k) / size**0.5
            logits += torch.full_like(logits, -math.inf).triu(total[b] - new[b] + 1)
            out[first : first + new[b], h] = torch.softmax(logits, -1) @ v
        first += new[b]
    return out.flatten(1)
