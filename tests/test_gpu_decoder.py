"""The operators of decoder graphs through planned sessions: MatMulNBits, OxiPagedCacheAppend, OxiPagedAttention against
their definitions in 64 bits (tests/decoder_oracle.py, which derives the tolerances), a run of them together, the ways in
(bound buffers, a caller's stream, a captured graph, host feeds), and what they refuse."""
import math

import numpy as np
import pytest

import decoder_oracle as D
from oxionnx_b200.graph import Graph, Node
from oxionnx_b200.session import CudaContext, Declined, OnnxError, Session, try_cuda_dispatch

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def name_of(t):
    return str(t.dtype).replace("torch.", "")


def session(nodes, inputs, outputs, weights=None, bind=True, **tuning):
    """A planned session with the device tensors of `inputs` and `outputs` bound."""
    graph = Graph(nodes=[Node(*n) for n in nodes], input_names=list(inputs), output_names=list(outputs))
    b = Session.builder().with_input_types({i: name_of(t) for i, t in inputs.items()}).with_input_shapes({i: tuple(t.shape) for i, t in inputs.items()})
    s = b.with_tuning(**tuning).build_from_graph(graph, weights or {})
    s.ensure_planned()
    s.buffers = (inputs, outputs)  # bound buffers outlive the runs that use them
    if bind:
        for i, t in inputs.items():
            s.bind_input_device(i, t.data_ptr(), name_of(t), t.numel())
        for o, t in outputs.items():
            s.bind_output_device(o, t.data_ptr(), t.numel(), name_of(t))
    return s


def run(s):
    s.enqueue(torch.cuda.current_stream().cuda_stream)
    s.wait()


def within(got, want, bound):
    got = got.double().cpu().reshape(want.shape)
    over = (got - want).abs() - bound
    assert not torch.isnan(over).any(), "NaN where a number was expected"
    worst = over.max().item() if over.numel() else 0.0
    assert worst <= 0, f"off by {worst:.3g} more than allowed at {int(over.argmax())} of {over.numel()}"


# ---- MatMulNBits ---------------------------------------------------------------------------------
def linear_node(k, n, group, w, y="y", x="x"):
    names = [x, "weights", "scales", "zero_points" if "zero_points" in w else "", "", "bias" if "bias" in w else ""]
    while names and not names[-1]:
        names.pop()
    return ("MatMulNBits", "linear", names, [y], {"K": k, "N": n, "bits": 4, "block_size": group})


def check_linear(rows, k, n, group, kind, zero_points=True, bias=False, seed=0, x=None):
    g = torch.Generator().manual_seed(seed)
    w = D.linear_weights(g, n, k, group, zero_points, bias)
    x = torch.randn(rows, k, generator=g).to(D.TYPES[kind]) if x is None else x
    y = torch.full((rows, n), math.nan, dtype=x.dtype, device="cuda")
    s = session([linear_node(k, n, group, w)], {"x": x.cuda()}, {"y": y}, w)
    run(s)
    many = rows > 16 and kind != "float32"  # these multiply 16-bit matrices, whose elements are rounded once
    within(y, D.linear(x, w, k), D.linear_bound(x, w, k, kind, rounded_weights=many))
    if many:
        within(y, D.linear(x, w, k, rounded=kind), D.linear_bound(x, w, k, kind, rounded_weights=False) * (1 + D.half_step(kind)))
    return s, x, y, w


@pytest.mark.parametrize("kind", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rows,k,n,group", [(1, 16, 1, 16), (1, 1, 1, 16), (1, 4096, 512, 128), (2, 1000, 65, 32), (3, 48, 17, 16), (7, 300, 129, 256), (8, 256, 64, 64),
                                            (9, 257, 33, 32), (16, 2048, 48, 128), (17, 130, 200, 64), (33, 777, 96, 16), (64, 512, 130, 32), (1, 8192, 40, 1024)])
def test_linear_over_few_rows(rows, k, n, group, kind):
    check_linear(rows, k, n, group, kind, zero_points=(rows + n) % 2 == 0, bias=n % 3 == 0, seed=rows + k)


@pytest.mark.parametrize("kind", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rows,k,n,group", [(65, 64, 64, 16), (100, 333, 77, 32), (128, 1024, 256, 128), (257, 520, 300, 64), (700, 96, 1111, 32)])
def test_linear_over_many_rows(rows, k, n, group, kind):
    check_linear(rows, k, n, group, kind, zero_points=rows % 2 == 1, bias=rows % 3 == 2, seed=rows)


@pytest.mark.parametrize("rows", [1, 6, 40, 130])
def test_linear_keeps_infinities_and_nan_in_their_rows(rows):
    g = torch.Generator().manual_seed(rows)
    k, n = 160, 72
    w = D.linear_weights(g, n, k, 32, False, False)
    w["weights"][:] = 0x99  # every weight is its scale: an infinity stays one
    x = torch.randn(rows, k, generator=g).half()
    x[0, 3] = math.inf
    if rows > 4:
        x[4, 150] = math.nan
    y = torch.zeros(rows, n, dtype=torch.float16, device="cuda")
    run(session([linear_node(k, n, 32, w)], {"x": x.cuda()}, {"y": y}, w))
    assert torch.isinf(y[0]).all()
    if rows > 4:
        assert torch.isnan(y[4]).all()
    for m in range(rows):
        if m not in (0, 4):
            assert torch.isfinite(y[m]).all()


def test_linear_runs_twice_to_the_same_bits_and_from_host_feeds():
    s, x, y, w = check_linear(5, 1000, 1111, 32, "bfloat16", bias=True)
    first = y.clone()
    run(s)
    assert torch.equal(first, y)
    graph = s.graph
    host = Session.builder().with_input_types({"x": "bfloat16"}).build_from_graph(graph, w)
    got = host.run({"x": x.float().numpy()})["y"]
    assert np.array_equal(got, first.float().cpu().numpy()), "host feeds are rounded to the declared type, fetches are its lanes"


def test_linear_of_three_dimensions_and_of_none():
    g = torch.Generator().manual_seed(2)
    w = D.linear_weights(g, 24, 64, 32, True, True)
    x = torch.randn(2, 3, 64, generator=g)
    y = torch.empty(2, 3, 24, device="cuda")
    run(session([linear_node(64, 24, 32, w)], {"x": x.cuda()}, {"y": y}, w))
    flat = x.reshape(6, 64)
    within(y, D.linear(flat, w, 64).reshape(2, 3, 24), D.linear_bound(flat, w, 64, "float32", False).reshape(2, 3, 24))


def test_linear_as_a_single_dispatch():
    g = torch.Generator().manual_seed(4)
    w = D.linear_weights(g, 40, 96, 32, True, False)
    x = torch.randn(3, 96, generator=g)
    node = Node(*linear_node(96, 40, 32, w))
    got = try_cuda_dispatch(node, w, {"x": x.numpy()}, CudaContext(0))[0]
    within(torch.from_numpy(got), D.linear(x, w, 96), D.linear_bound(x, w, 96, "float32", False))


def test_linear_between_float_operators():
    """f32 lanes in, f32 lanes out: a Relu in front and an Add behind read and write them as ever."""
    g = torch.Generator().manual_seed(5)
    w = D.linear_weights(g, 64, 64, 32, False, False)
    x = torch.randn(4, 64, generator=g)
    nodes = [("Relu", "r", ["x"], ["a"], {}), linear_node(64, 64, 32, w, "b", "a"), ("Add", "s", ["b", "x"], ["y"], {})]
    graph = Graph(nodes=[Node(*n) for n in nodes], input_names=["x"], output_names=["y"])
    got = torch.from_numpy(Session.builder().build_from_graph(graph, w).run({"x": x.numpy()})["y"])
    want = D.linear(x.clamp(min=0), w, 64) + x.double()
    within(got, want, D.linear_bound(x.clamp(min=0), w, 64, "float32", False) + 2.0**-23 * want.abs())


def test_sixteen_bit_values_are_f32_lanes_to_other_operators():
    g = torch.Generator().manual_seed(6)
    w = D.linear_weights(g, 64, 64, 32, False, False)
    x = torch.randn(4, 64, generator=g).half()
    y, z = torch.empty(4, 64, device="cuda"), torch.empty(4, 64, dtype=torch.float16, device="cuda")
    nodes = [linear_node(64, 64, 32, w, "a"), ("Add", "s", ["a", "x"], ["y"], {}), ("Reshape", "v", ["a", "shape"], ["z"], {})]
    run(session(nodes, {"x": x.cuda()}, {"y": y, "z": z}, {**w, "shape": np.array([64, 4], np.float32)}))
    want = D.linear(x, w, 64)
    within(z, want, D.linear_bound(x, w, 64, "float16", False))
    assert torch.equal(y.cpu(), z.cpu().float() + x.float())


# ---- OxiPagedCacheAppend -------------------------------------------------------------------------
TABLES = ["cu_query", "kv_lengths", "page_table"]


def check_append(p, half, interleaved, positions=None):
    cos, sin = D.angles(positions or max(max(p.total), 1), half) if half else (None, None)
    dev = {"query": (p.q if p.packed is None else p.packed).cuda()}
    if p.packed is None:
        dev |= {"key": p.k.cuda(), "value": p.v.cuda()}
    dev |= {"key_cache": p.kc.cuda(), "value_cache": p.vc.cuda(), "cu_query": p.cu.cuda(), "kv_lengths": p.len.cuda(), "page_table": p.table.cuda()}
    out = torch.full(p.q.shape, math.nan, dtype=D.TYPES[p.kind], device="cuda")
    names = ["query", *(["key", "value"] if p.packed is None else ["", ""]), "key_cache", "value_cache", *TABLES] + (["cos", "sin"] if half else [])
    node = ("OxiPagedCacheAppend", "append", names, ["rotated", "kc", "vc"], {"num_heads": p.heads, "kv_num_heads": p.kv_heads, "interleaved": int(interleaved)})
    s = session([node], dev, {"rotated": out}, {"cos": cos.numpy(), "sin": sin.numpy()} if half else {})
    for _ in range(2):  # putting the same tokens in twice changes nothing
        run(s)
        (rotated, rb), (kc, kb), vc = D.append(p, cos, sin, interleaved)
        within(out, rotated, rb)
        got = dev["key_cache"].cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(kc)), "a row that no new token has was written, or one was left out"
        within(torch.nan_to_num(got), torch.nan_to_num(kc), kb)
        assert torch.equal(torch.nan_to_num(dev["value_cache"].cpu()), torch.nan_to_num(vc))
        assert torch.equal(torch.isnan(dev["value_cache"].cpu()), torch.isnan(vc))
    return s, dev, out


@pytest.mark.parametrize("kind", ["float16", "bfloat16"])
@pytest.mark.parametrize("heads,kv_heads,size,half,interleaved,packed", [
    (4, 4, 64, 32, False, False), (8, 2, 128, 64, False, True), (6, 2, 80, 40, True, False), (3, 1, 40, 12, False, True), (5, 5, 8, 4, True, True),
    (2, 1, 256, 128, False, False), (4, 2, 96, 24, True, False), (7, 1, 64, 0, False, False), (2, 2, 24, 5, False, False), (2, 2, 24, 5, True, False), (32, 8, 128, 16, False, False)])
def test_append(heads, kv_heads, size, half, interleaved, packed, kind):
    check_append(D.Paged([1, 3, 17, 1], [1, 40, 17, 33], heads, kv_heads, size, 16, kind, seed=heads, behind=2, packed=packed), half, interleaved)


def test_append_rounds_f32_rows_to_the_caches_type():
    check_append(D.Paged([2, 5], [20, 5], 4, 2, 64, 16, "bfloat16", seed=1, q_kind="float32"), 32, False)
    check_append(D.Paged([2, 5], [20, 5], 4, 2, 64, 16, "float16", seed=1, q_kind="float32", packed=True), 16, True)


def test_append_skips_idle_streams():
    """Rows of negative position (a length below the number of new rows) go nowhere and rotate to 0."""
    check_append(D.Paged([1, 1, 4, 1], [0, 9, 2, 0], 4, 2, 64, 16, "float16", seed=3, behind=3), 32, False)


def test_append_of_many_streams_and_large_pages():
    new = [1 + i % 3 for i in range(70)]
    check_append(D.Paged(new, [n + 7 * i for i, n in enumerate(new)], 2, 1, 64, 128, "bfloat16", seed=4), 32, False)


def test_append_reports_what_is_wrong_and_skips_it():
    p = D.Paged([1, 1, 1], [5, 6, 7], 2, 2, 64, 16, "float16", seed=5)
    want, _, _ = D.append(p, *D.angles(8, 32), False)
    s, dev, out = check_append(p, 32, False, positions=8)
    table = dev["page_table"].clone()
    for page in (-1, p.pages, 2**31 - 1, -(2**31)):
        before = dev["value_cache"].clone()
        dev["page_table"][1, 0] = page
        with pytest.raises(OnnxError, match="page table"):
            run(s)
        assert torch.equal(torch.nan_to_num(before), torch.nan_to_num(dev["value_cache"]))
        dev["page_table"].copy_(table)
        run(s)
    dev["kv_lengths"][2] = 9  # position 8, and cos has 8 rows
    with pytest.raises(OnnxError, match="cos"):
        run(s)
    dev["kv_lengths"][2] = 10_000  # more than its row of the table holds
    with pytest.raises(OnnxError, match="cu_query"):
        run(s)
    dev["kv_lengths"][2] = 7
    for cu in ([0, 2, 1, 3], [0, 1, 2, 9], [1, 1, 2, 3], [0, -5, 2, 3]):
        dev["cu_query"].copy_(torch.tensor(cu, dtype=torch.int32))
        with pytest.raises(OnnxError, match="cu_query"):
            run(s)
    dev["cu_query"].copy_(p.cu)
    run(s)
    within(out, *want)


# ---- OxiPagedAttention ---------------------------------------------------------------------------
def attend_inputs(p):
    return {"query": p.q.cuda(), "key_cache": p.kc.cuda(), "value_cache": p.vc.cuda(), "cu_query": p.cu.cuda(), "kv_lengths": p.len.cuda(), "page_table": p.table.cuda()}


def check_attend(p, hint=True, scale=None):
    dev = attend_inputs(p)
    out = torch.full(p.q.shape, math.nan, dtype=D.TYPES[p.kind], device="cuda")
    attrs = {"num_heads": p.heads, "kv_num_heads": p.kv_heads}
    if hint:
        attrs["max_query_length"] = max(p.new)
    if scale is not None:
        attrs["scale"] = scale
    s = session([("OxiPagedAttention", "attend", ["query", "key_cache", "value_cache", *TABLES], ["out"], attrs)], dev, {"out": out})
    run(s)
    within(out, *D.attend(p, scale))
    first = out.clone()
    run(s)
    assert torch.equal(first, out), "two runs differ"
    return s, dev, out


HEADS = [(1, 1, 64), (4, 4, 64), (8, 2, 128), (32, 8, 128), (6, 2, 96), (5, 1, 80), (7, 7, 40), (16, 1, 128), (3, 1, 256), (2, 2, 8), (40, 1, 64), (10, 2, 160)]


@pytest.mark.parametrize("kind", ["float16", "bfloat16"])
@pytest.mark.parametrize("heads,kv_heads,size", HEADS)
def test_attention_of_single_tokens(heads, kv_heads, size, kind):
    check_attend(D.Paged([1] * 6, [1, 2, 63, 64, 65, 300], heads, kv_heads, size, 16, kind, seed=size))


@pytest.mark.parametrize("kind", ["float16", "bfloat16"])
@pytest.mark.parametrize("heads,kv_heads,size", HEADS)
def test_attention_of_prompts(heads, kv_heads, size, kind):
    check_attend(D.Paged([1, 128, 70, 200], [1, 128, 70, 200], heads, kv_heads, size, 16, kind, seed=size))


@pytest.mark.parametrize("page", [16, 32, 48, 64, 128, 256, 272])
@pytest.mark.parametrize("new,total", [([1, 1], [500, 33]), ([130, 9], [400, 300]), ([3, 64, 1], [90, 64, 257])])
def test_attention_over_pages(page, new, total):
    check_attend(D.Paged(new, total, 4, 2, 64, page, "bfloat16", seed=page))


@pytest.mark.parametrize("hint", [False, True])
@pytest.mark.parametrize("new,total", [([1, 300, 1, 2, 40], [700, 300, 5, 2, 1000]), ([1] * 40, list(range(1, 401, 10))), ([257], [257]), ([256], [1500]), ([1], [3000]), ([5] * 9, [77] * 9)])
def test_attention_of_mixed_batches(new, total, hint):
    check_attend(D.Paged(new, total, 8, 2, 128, 32, "float16", seed=sum(new)), hint=hint)


@pytest.mark.parametrize("new", [1, 2, 3, 4, 5, 8, 15, 16, 17, 33, 64, 65])
def test_attention_of_a_few_new_tokens(new):
    check_attend(D.Paged([new, new, 1], [new, new + 200, 129], 4, 1, 128, 16, "bfloat16", seed=new))


@pytest.mark.parametrize("size", [64, 128, 192])
def test_attention_leaves_idle_streams_and_rows_behind_at_zero(size):
    """No token to see: lengths of 0, lengths below the number of new rows, rows behind the last sequence."""
    for new, total in (([1, 1, 1], [0, 20, 0]), ([100, 5, 200], [30, 0, 130]), ([1, 0, 2], [4, 9, 2])):
        p = D.Paged(new, total, 4, 2, size, 16, "float16", seed=7, behind=37)
        s, dev, out = check_attend(p)
        idle = torch.ones(p.q.shape[0], dtype=torch.bool)
        for row, _, position in p.rows():
            idle[row] = position < 0
        assert torch.equal(out[idle.cuda()], torch.zeros_like(out[idle.cuda()]))


def test_attention_of_a_long_stream_and_of_scores_far_apart():
    check_attend(D.Paged([1], [20011], 4, 1, 128, 64, "bfloat16", seed=1))
    for kind in ("float16", "bfloat16"):  # scores of several hundred: one key takes everything
        check_attend(D.Paged([1, 150], [400, 150], 4, 2, 64, 16, kind, seed=2, spread=6.0))


@pytest.mark.parametrize("scale", [0.0, -0.2, 1.0])
def test_attention_scales(scale):
    check_attend(D.Paged([1, 140], [300, 140], 4, 2, 64, 16, "bfloat16", seed=9), scale=scale)


def test_attention_sees_infinities_of_its_own_keys_only():
    """A key of -infinity in every lane against a query without zeros or signs weighs nothing; NaN behind a row's position
    does not reach it; NaN before it does."""
    p = D.Paged([150, 1], [150, 90], 2, 1, 64, 16, "float16", seed=11)
    p.q.abs_().clamp_(min=0.1)
    slot = (int(p.table[0, 40 // 16]), 40 % 16)
    p.kc[slot] = -math.inf
    late = (int(p.table[0, 120 // 16]), 120 % 16)
    p.kc[late] = math.nan
    dev, out = attend_inputs(p), torch.zeros(p.q.shape, dtype=torch.float16, device="cuda")
    run(session([("OxiPagedAttention", "attend", list(dev), ["out"], {"num_heads": 2, "kv_num_heads": 1})], dev, {"out": out}))
    assert torch.isfinite(out[:120]).all() and torch.isfinite(out[150]).all()
    assert torch.isnan(out[120:150]).all()
    p.kc[late] = 0
    p.new, p.total = [120, 1], [120, 90]
    want, bound = D.attend(p)
    within(out[:120], want[:120], bound[:120])


def test_attention_reports_what_is_wrong():
    p = D.Paged([1, 100], [40, 130], 4, 2, 64, 16, "bfloat16", seed=12)
    s, dev, out = check_attend(p)
    want = out.clone()
    for row, col in ((0, 1), (1, 3)):
        for page in (-1, p.pages, 2**31 - 1, -(2**31)):
            held = dev["page_table"][row, col].clone()
            dev["page_table"][row, col] = page
            with pytest.raises(OnnxError, match="page table"):
                run(s)
            dev["page_table"][row, col] = held
    for cu in ([0, 101, 90], [0, 1, 400], [1, 1, 101], [0, -1, 101]):
        dev["cu_query"].copy_(torch.tensor(cu, dtype=torch.int32))
        with pytest.raises(OnnxError, match="cu_query|max_query_length"):
            run(s)
    dev["cu_query"].copy_(p.cu)
    dev["kv_lengths"][0] = 2**31 - 1
    with pytest.raises(OnnxError, match="cu_query"):
        run(s)
    dev["kv_lengths"].copy_(p.len)
    run(s)
    assert torch.equal(out, want)


def test_attention_reports_more_rows_than_it_was_promised():
    p = D.Paged([1, 1], [40, 30], 4, 2, 64, 16, "bfloat16", seed=13)
    s, dev, out = check_attend(p)
    dev["cu_query"].copy_(torch.tensor([0, 0, 2], dtype=torch.int32))
    with pytest.raises(OnnxError, match="max_query_length"):
        run(s)


def test_attention_rounds_an_f32_query():
    p = D.Paged([1, 90], [50, 90], 4, 2, 64, 16, "float16", seed=14, q_kind="float32")
    dev, out = attend_inputs(p), torch.empty(p.q.shape, dtype=torch.float16, device="cuda")
    run(session([("OxiPagedAttention", "attend", list(dev), ["out"], {"num_heads": 4, "kv_num_heads": 2})], dev, {"out": out}))
    within(out, *D.attend(p))


# ---- together ------------------------------------------------------------------------------------
def decoder_nodes(heads, kv_heads, size, group, hidden, most=0):
    qkv = (heads + 2 * kv_heads) * size
    shared = {"num_heads": heads, "kv_num_heads": kv_heads}
    return [("MatMulNBits", "qkv", ["x", "w1", "s1"], ["qkv"], {"K": hidden, "N": qkv, "bits": 4, "block_size": group}),
            ("OxiPagedCacheAppend", "append", ["qkv", "", "", "key_cache", "value_cache", *TABLES, "cos", "sin"], ["rotated", "kc", "vc"], shared),
            ("OxiPagedAttention", "attend", ["rotated", "kc", "vc", *TABLES], ["context"], {**shared, "max_query_length": most}),
            ("MatMulNBits", "o", ["context", "w2", "s2"], ["y"], {"K": heads * size, "N": hidden, "bits": 4, "block_size": group})]


class Layer:
    """The attention half of a decoder layer over a fixed batch of streams."""

    def __init__(self, kind, streams, rows, x_kind=None, heads=8, kv_heads=2, size=64, hidden=160, page=16, length=200):
        g = torch.Generator().manual_seed(21)
        self.kind, self.heads, self.kv_heads, self.size, self.hidden, self.page = kind, heads, kv_heads, size, hidden, page
        w1, w2 = D.linear_weights(g, (heads + 2 * kv_heads) * size, hidden, 32, False, False), D.linear_weights(g, hidden, heads * size, 32, False, False)
        self.w1, self.w2 = w1, w2
        self.cos, self.sin = D.angles(length, size // 2)
        self.weights = {"w1": w1["weights"], "s1": w1["scales"], "w2": w2["weights"], "s2": w2["scales"], "cos": self.cos.numpy(), "sin": self.sin.numpy()}
        self.columns = -(-length // page)
        pages = streams * self.columns + 1
        dt = D.TYPES[kind]
        self.table = torch.randperm(pages, generator=g)[: streams * self.columns].reshape(streams, -1).to(torch.int32)
        self.dev = {"x": torch.zeros(rows, hidden, dtype=D.TYPES[x_kind or kind], device="cuda"),
                    "key_cache": torch.full((pages, page, kv_heads, size), math.nan, dtype=dt, device="cuda"),
                    "value_cache": torch.full((pages, page, kv_heads, size), math.nan, dtype=dt, device="cuda"),
                    "cu_query": torch.zeros(streams + 1, dtype=torch.int32, device="cuda"),
                    "kv_lengths": torch.zeros(streams, dtype=torch.int32, device="cuda"), "page_table": self.table.cuda()}
        self.y = torch.full((rows, hidden), math.nan, dtype=dt, device="cuda")
        self.session = session(decoder_nodes(heads, kv_heads, size, 32, hidden), self.dev, {"y": self.y}, self.weights)
        self.keys, self.values = [[] for _ in range(streams)], [[] for _ in range(streams)]

    def set(self, x, new, total):
        self.dev["x"].zero_()
        self.dev["x"][: x.shape[0]] = x.cuda()
        self.dev["cu_query"].copy_(torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32))
        self.dev["kv_lengths"].copy_(torch.tensor(total, dtype=torch.int32))

    def plain(self, x, new):
        """The same steps, each result rounded to the type, keys and values kept in lists."""
        dt = D.TYPES[self.kind]
        rounded = self.kind if x.shape[0] > 16 and x.dtype != torch.float32 else None
        x = x.double()
        qkv = (x @ D.linear_matrix(self.w1, self.hidden, rounded).t()).to(self.dev["x"].dtype)
        q, k, v = qkv.split((self.heads * self.size, self.kv_heads * self.size, self.kv_heads * self.size), 1)
        context, row = torch.zeros(x.shape[0], self.heads, self.size, dtype=torch.float64), 0
        for b, n in enumerate(new):
            for _ in range(n):
                position = len(self.keys[b])
                turn = lambda t, heads: D.rotate(t.reshape(heads, self.size), self.cos, self.sin, position, False)[0].to(dt).double()  # noqa: E731
                self.keys[b].append(turn(k[row], self.kv_heads))
                self.values[b].append(v[row].reshape(self.kv_heads, self.size).to(dt).double())
                qq, kk, vv = turn(q[row], self.heads), torch.stack(self.keys[b]), torch.stack(self.values[b])
                for head in range(self.heads):
                    s = kk[:, head // (self.heads // self.kv_heads)] @ qq[head] / math.sqrt(self.size)
                    context[row, head] = torch.softmax(s, 0) @ vv[:, head // (self.heads // self.kv_heads)]
                row += 1
        rounded = self.kind if x.shape[0] > 16 else None
        return context.flatten(1).to(dt).double() @ D.linear_matrix(self.w2, self.heads * self.size, rounded).t()


@pytest.mark.parametrize("kind,x_kind", [("bfloat16", None), ("float16", None), ("bfloat16", "float32")])
def test_prompts_and_then_tokens_through_a_layer(kind, x_kind):
    """Prompts of three streams in one call, then token after token through a second plan on the same cache.  The roundings
    of the steps may fall differently where the f32 sums in front of them do, one step each; four of them in a row, two of
    them scaled by a product, stay within 12 half steps of the size of what is summed."""
    g = torch.Generator().manual_seed(31)
    prompts = [70, 9, 31]
    layer = Layer(kind, 3, sum(prompts), x_kind)
    step = Layer(kind, 3, 3, x_kind)
    x = torch.randn(sum(prompts), layer.hidden, generator=g).to(layer.dev["x"].dtype)
    layer.set(x, prompts, prompts)
    run(layer.session)
    want = layer.plain(x, prompts)
    bound = 12 * D.half_step(kind) * math.sqrt(layer.heads * layer.size) * 0.3
    assert (layer.y.double().cpu() - want).abs().max() < bound
    assert want.abs().max() > 20 * D.half_step(kind)
    # the decoding plan on the prompts' cache
    step.keys, step.values = layer.keys, layer.values
    for name in ("key_cache", "value_cache"):
        step.session.bind_input_device(name, layer.dev[name].data_ptr(), kind, layer.dev[name].numel())
    lengths = list(prompts)
    for _ in range(4):
        x = torch.randn(3, layer.hidden, generator=g).to(layer.dev["x"].dtype)
        lengths = [n + 1 for n in lengths]
        step.set(x, [1, 1, 1], lengths)
        run(step.session)
        assert (step.y.double().cpu() - step.plain(x, [1, 1, 1])).abs().max() < bound


def test_a_captured_layer_replays_with_what_its_buffers_hold():
    g = torch.Generator().manual_seed(41)
    layer = Layer("bfloat16", 4, 4)
    bound = 12 * D.half_step("bfloat16") * math.sqrt(layer.heads * layer.size) * 0.3
    x = torch.randn(4, layer.hidden, generator=g).bfloat16()
    layer.set(x, [1] * 4, [1] * 4)
    run(layer.session)  # outside a capture first: it sets the kernels' one-time attributes
    assert (layer.y.double().cpu() - layer.plain(x, [1] * 4)).abs().max() < bound
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        layer.session.enqueue(torch.cuda.current_stream().cuda_stream)
    for length in range(2, 40):
        x = torch.randn(4, layer.hidden, generator=g).bfloat16()
        layer.set(x, [1] * 4, [length] * 4)
        graph.replay()
        torch.cuda.synchronize()
        assert (layer.y.double().cpu() - layer.plain(x, [1] * 4)).abs().max() < bound
    layer.session.wait()


def test_runs_of_one_session_on_two_streams_follow_one_another():
    p = D.Paged([1] * 8, [900 + i for i in range(8)], 8, 2, 128, 16, "bfloat16", seed=51)
    s, dev, out = check_attend(p)
    want = out.clone()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(40):
        s.enqueue(streams[i % 2].cuda_stream)
    s.wait()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_two_sessions_side_by_side():
    p = D.Paged([1] * 8, [900 + i for i in range(8)], 8, 2, 128, 16, "bfloat16", seed=52)
    q = D.Paged([200, 30], [200, 400], 4, 4, 64, 32, "float16", seed=53)
    (s, _, a), (t, _, b) = check_attend(p), check_attend(q)
    wa, wb = a.clone(), b.clone()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        s.enqueue(streams[0].cuda_stream)
        t.enqueue(streams[1].cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(a, wa) and torch.equal(b, wb)


def test_host_feeds_give_what_bound_buffers_give_and_leave_the_feeds_alone():
    p = D.Paged([1, 90], [50, 90], 4, 2, 64, 16, "float16", seed=54)
    p.kc, p.vc = torch.nan_to_num(p.kc), torch.nan_to_num(p.vc)
    s, dev, out = check_attend(p)
    feeds = {n: (t.float() if t.is_floating_point() else t).cpu().numpy() for n, t in dev.items()}
    host = Session.builder().with_input_types({n: name_of(t) for n, t in dev.items()}).build_from_graph(s.graph, {})
    assert np.array_equal(host.run(feeds)["out"], out.float().cpu().numpy())
    assert np.array_equal(host.run_pipelined([feeds, feeds, feeds])[2]["out"], out.float().cpu().numpy())
    bound = s.run_with_binding()  # fetched as f32 lanes, and written to the bound buffer too
    assert np.array_equal(bound["out"], out.float().cpu().numpy())


def test_an_appended_cache_can_be_fetched():
    p = D.Paged([2, 1], [20, 3], 2, 2, 64, 16, "float16", seed=55)
    p.kc, p.vc = torch.nan_to_num(p.kc), torch.nan_to_num(p.vc)
    names = ["query", "key", "value", "key_cache", "value_cache", *TABLES]
    node = Node("OxiPagedCacheAppend", "append", names, ["rotated", "kc", "vc"], {"num_heads": 2, "kv_num_heads": 2})
    feeds = dict(zip(names, (t.numpy() for t in (p.q, p.k, p.v, p.kc, p.vc, p.cu, p.len, p.table))))
    types = {n: "int32" if n in TABLES else "float16" for n in names}
    s = Session.builder().with_input_types(types).build_from_graph(Graph([node], names, ["rotated", "kc", "vc"]), {})
    got = s.run(feeds)
    (rotated, _), (kc, _), vc = D.append(p, None, None, False)
    assert np.array_equal(got["rotated"], rotated.numpy()) and np.array_equal(got["kc"], kc.numpy()) and np.array_equal(got["vc"], vc.float().numpy())
    assert np.array_equal(s.run(feeds)["kc"], got["kc"])


def test_outputs_that_cannot_be_written_in_place_are_copied():
    p = D.Paged([1, 90], [50, 90], 4, 2, 64, 16, "float16", seed=56)
    s, dev, out = check_attend(p)
    n = out.numel()
    odd = torch.zeros(n + 3, dtype=torch.float16, device="cuda")
    s.bind_output_device("out", odd[3:].data_ptr(), n, "float16")  # 6 bytes off 16
    run(s)
    assert torch.equal(odd[3:].view_as(out), out) and torch.equal(odd[:3], torch.zeros_like(odd[:3]))
    q = dev["query"].clone()
    s.bind_output_device("out", dev["query"].data_ptr(), n, "float16")  # over the query itself
    run(s)
    assert torch.equal(dev["query"], out)
    dev["query"].copy_(q)
    with pytest.raises(OnnxError, match="bound"):
        s.output_device_ptr("out")
    s.clear_bindings()
    with pytest.raises(OnnxError, match="not bound"):
        s.enqueue(0)


def test_enqueue_on_the_default_stream_keeps_the_current_device():
    s, x, y, w = check_linear(1, 256, 64, 32, "bfloat16")
    want = y.clone()
    y.zero_()
    s.enqueue(0)
    torch.cuda.synchronize()
    assert torch.equal(y, want) and torch.cuda.current_device() == 0


def test_recorded_sessions_give_the_same(monkeypatch):
    p = D.Paged([1, 90], [50, 90], 4, 2, 64, 16, "float16", seed=57)
    dev, out = attend_inputs(p), torch.zeros(p.q.shape, dtype=torch.float16, device="cuda")
    s = session([("OxiPagedAttention", "attend", list(dev), ["out"], {"num_heads": 4, "kv_num_heads": 2})], dev, {"out": out}, cuda_graph=True)
    for _ in range(4):
        out.zero_()
        s.run_with_binding(fetch=False)
        within(out, *D.attend(p))
    assert s.cuda_cache_counters()["graph_replays"] >= 1
    other = torch.zeros_like(out)
    s.bind_output_device("out", other.data_ptr(), other.numel(), "float16")
    s.run_with_binding(fetch=False)
    assert torch.equal(other, out)


# ---- refusals ------------------------------------------------------------------------------------
@pytest.mark.parametrize("change,match", [
    ({"bits": 8}, "4-bit"), ({"block_size": 24}, "block_size"), ({"block_size": 8}, "block_size"), ({"K": 0}, "K 0"), ({"N": 32}, "codes"), ({"K": 63}, "last extent"),
    ({"new_attribute": 1}, "attribute")])
def test_linear_refuses(change, match):
    g = torch.Generator().manual_seed(1)
    w = D.linear_weights(g, 64, 64, 32, True, False)
    op, name, ins, outs, attrs = linear_node(64, 64, 32, w)
    graph = Graph([Node(op, name, ins, outs, {**attrs, **change})], ["x"], ["y"])
    with pytest.raises(Declined, match=match):
        Session.builder().with_input_shapes({"x": (2, 64)}).build_from_graph(graph, w).ensure_planned()


@pytest.mark.parametrize("name,value,match", [("scales", np.ones(3, np.float32), "scales"), ("zero_points", np.zeros((64, 2), np.float32), "zero points"),
                                              ("weights", np.full((64, 2, 16), 0.5, np.float32), "bytes"), ("bias", np.zeros(5, np.float32), "bias")])
def test_linear_refuses_weights(name, value, match):
    g = torch.Generator().manual_seed(1)
    w = D.linear_weights(g, 64, 64, 32, True, True)
    w[name] = value
    with pytest.raises(Declined, match=match):
        Session.builder().with_input_shapes({"x": (2, 64)}).build_from_graph(Graph([Node(*linear_node(64, 64, 32, w))], ["x"], ["y"]), w).ensure_planned()


@pytest.mark.parametrize("op", ["OxiPagedCacheAppend", "OxiPagedAttention"])
@pytest.mark.parametrize("change,match", [
    ({"num_heads": 3}, "num_heads"), ({"kv_num_heads": 4}, "num_heads"), ({"unknown": 1}, "attribute"), ({"type:key_cache": "float32"}, "caches"),
    ({"type:value_cache": "bfloat16"}, "caches"), ({"type:cu_query": "float32"}, "i32"), ({"type:query": "bfloat16"}, "bf16"), ({"shape:query": (3, 100)}, "tokens"),
    ({"shape:key_cache": (5, 24, 2, 64)}, "caches"), ({"shape:cu_query": (2,)}, "bounds"), ({"shape:page_table": (2, 0)}, "page_table"),
    ({"cache": (5, 24, 2, 64)}, "pages of 24"), ({"cache": (5, 16, 2, 60)}, "heads of 60"), ({"cache": (5, 16, 2, 264)}, "heads of 264")])
def test_paged_operators_refuse(op, change, match):
    change = dict(change)
    cache = change.pop("cache", (5, 16, 2, 64))
    size = cache[3]
    shapes = {"query": (3, 4 * size), "key": (3, 2 * size), "value": (3, 2 * size), "key_cache": cache, "value_cache": cache, "cu_query": (3,), "kv_lengths": (2,),
              "page_table": (2, 3)}
    types = {n: "int32" if n in TABLES else "float16" for n in shapes}
    attrs = {"num_heads": 4, "kv_num_heads": 2}
    for what, value in change.items():
        if what.startswith("type:"):
            types[what[5:]] = value
        elif what.startswith("shape:"):
            shapes[what[6:]] = value
        else:
            attrs[what] = value
    names = list(shapes) if op == "OxiPagedCacheAppend" else ["query", *list(shapes)[3:]]
    node = Node(op, "n", names, ["a", "b", "c"] if op == "OxiPagedCacheAppend" else ["a"], attrs)
    b = Session.builder().with_input_shapes({n: shapes[n] for n in names}).with_input_types({n: types[n] for n in names})
    with pytest.raises(Declined, match=match):
        b.build_from_graph(Graph([node], names, ["a"]), {}).ensure_planned()


def test_append_refuses_a_cache_that_something_else_reads():
    shapes = {"query": (3, 256), "key": (3, 128), "value": (3, 128), "key_cache": (5, 16, 2, 64), "value_cache": (5, 16, 2, 64), "cu_query": (3,), "kv_lengths": (2,), "page_table": (2, 3)}
    types = {n: "int32" if n in TABLES else "float16" for n in shapes}
    attrs = {"num_heads": 4, "kv_num_heads": 2}
    append = Node("OxiPagedCacheAppend", "append", list(shapes), ["a", "b", "c"], attrs)
    attend = Node("OxiPagedAttention", "attend", ["a", "key_cache", "c", *TABLES], ["y"], attrs)  # the cache from before the update
    for nodes, outs in (([append, attend], ["y"]), ([append], ["a", "key_cache"])):
        with pytest.raises(Declined, match="updated where it lies"):
            Session.builder().with_input_shapes(shapes).with_input_types(types).build_from_graph(Graph(nodes, list(shapes), outs), {}).ensure_planned()


def test_bindings_refuse_other_types():
    s, x, y, w = check_linear(2, 64, 32, 32, "float16")
    with pytest.raises(OnnxError, match="planned as f16"):
        s.bind_input_device("x", x.cuda().data_ptr(), np.float32, x.numel())
    with pytest.raises(OnnxError, match="planned as f16"):
        s.bind_output_device("y", y.data_ptr(), y.numel(), "bfloat16")
    with pytest.raises(OnnxError, match="aligned"):
        s.bind_output_device("y", y.data_ptr() + 1, y.numel(), "float16")
    with pytest.raises(OnnxError, match="holds"):
        s.bind_output_device("y", y.data_ptr(), y.numel() - 1, "float16")


@pytest.mark.parametrize("half,interleaved,packed", [(32, False, True), (16, True, False), (0, False, False), (5, False, True)])
def test_append_of_a_long_batch(half, interleaved, packed):
    """Enough tokens for the kernel that serves several of them a block; idle ones among them, rows behind the last."""
    new = [1200, 1, 700, 333, 210]
    check_append(D.Paged(new, [1500, 0, 700, 300, 4000], 2, 1, 64, 32, "bfloat16", seed=6, behind=21, packed=packed), half, interleaved)


# ---- sizes and orders that take other ways -------------------------------------------------------
def test_attention_of_thousands_of_streams():
    new = [1] * 4096
    check_attend(D.Paged(new, [1 + i % 37 for i in range(4096)], 2, 1, 64, 16, "bfloat16", seed=60))


def test_attention_of_hundreds_of_prompts():
    """More sequences than the prompt kernel's block has threads, of which some are streamed and some multiplied."""
    new = [1 + (i * 7) % 40 for i in range(500)]
    check_attend(D.Paged(new, [n + i % 90 for i, n in enumerate(new)], 4, 1, 64, 16, "float16", seed=61))


@pytest.mark.parametrize("heads,size", [(192, 64), (130, 40), (128, 128)])
def test_attention_with_very_many_heads_to_a_key_head(heads, size):
    check_attend(D.Paged([3, 1], [40, 100], heads, 1, size, 16, "bfloat16", seed=62))


def test_offsets_behind_four_gigabytes():
    """The same small sequences at the far end of caches of 2^32 lanes and more each."""
    p = D.Paged([1, 90], [50, 120], 8, 4, 128, 64, "bfloat16", seed=63)
    dev = attend_inputs(p)
    pages = 2**32 // (64 * 4 * 128) + 40
    for name in ("key_cache", "value_cache"):
        big = torch.empty(pages, 64, 4, 128, dtype=torch.bfloat16, device="cuda")
        big[pages - p.pages :] = dev[name]
        dev[name] = big
    dev["page_table"] = torch.where(dev["page_table"] >= 0, dev["page_table"] + (pages - p.pages), dev["page_table"]).to(torch.int32)
    out = torch.full(p.q.shape, math.nan, dtype=torch.bfloat16, device="cuda")
    run(session([("OxiPagedAttention", "attend", list(dev), ["out"], {"num_heads": 8, "kv_num_heads": 4})], dev, {"out": out}))
    within(out, *D.attend(p))
    rows = {"query": p.q.cuda(), "key": p.k.cuda(), "value": p.v.cuda(), **{n: dev[n] for n in ("key_cache", "value_cache", *TABLES)}}
    rotated = torch.empty(p.q.shape, dtype=torch.bfloat16, device="cuda")
    run(session([("OxiPagedCacheAppend", "append", list(rows), ["r", "kc", "vc"], {"num_heads": 8, "kv_num_heads": 4})], rows, {"r": rotated}))
    (want, _), (kc, _), vc = D.append(p, None, None, False)
    assert torch.equal(rotated.double().cpu(), want)
    tail = dev["value_cache"][pages - p.pages :].cpu()
    assert torch.equal(torch.nan_to_num(tail), torch.nan_to_num(vc))
    tail = dev["key_cache"][pages - p.pages :].double().cpu()
    assert torch.equal(torch.nan_to_num(tail), torch.nan_to_num(kc))


def test_linear_of_the_largest_numbers():
    """f32 rows at the end of their range: the parts of a number round to no infinity."""
    g = torch.Generator().manual_seed(64)
    w = D.linear_weights(g, 33, 64, 32, False, False)
    w["weights"][:] = 0x88  # code 8: weights of 0
    w["weights"][:, 0, 0] = 0x89  # and one of the scale
    x = torch.full((2, 64), torch.finfo(torch.float32).max)
    x[1] = 0.0
    x[1, 0] = -torch.finfo(torch.float32).max
    y = torch.empty(2, 33, device="cuda")
    run(session([linear_node(64, 33, 32, w)], {"x": x.cuda()}, {"y": y}, w))
    within(y, D.linear(x, w, 64), 4 * 2.0**-23 * D.linear(x, w, 64).abs())


def test_host_feeds_never_go_into_bound_buffers():
    p = D.Paged([1, 90], [50, 90], 4, 2, 64, 16, "float16", seed=65)
    p.kc, p.vc = torch.nan_to_num(p.kc), torch.nan_to_num(p.vc)
    s, dev, out = check_attend(p)
    want, kept = out.clone(), {n: t.clone() for n, t in dev.items()}
    feeds = {n: (t.float() if t.is_floating_point() else t).cpu().numpy() for n, t in dev.items()}
    feeds["query"] = feeds["query"] * 0.5
    other = s.run(feeds)["out"]
    assert not np.array_equal(other, want.float().cpu().numpy())
    assert np.array_equal(s.run_pipelined([feeds, feeds])[1]["out"], other)
    assert all(torch.equal(kept[n], dev[n]) for n in dev)
    out.zero_()
    run(s)  # the bindings still hold
    assert torch.equal(out, want)


def test_models_with_typed_inputs_through_the_loader():
    p = D.Paged([1, 20], [50, 20], 4, 2, 64, 16, "bfloat16", seed=66)
    p.kc, p.vc = torch.nan_to_num(p.kc), torch.nan_to_num(p.vc)
    s, dev, out = check_attend(p)
    feeds = {n: (t.float() if t.is_floating_point() else t).cpu().numpy() for n, t in dev.items()}
    b = Session.builder().with_input_types({n: name_of(t) for n, t in dev.items()}).with_input_shapes({n: tuple(t.shape) for n, t in dev.items()})
    loaded = b.with_optimization_level(1).build_from_graph(s.graph, {})
    assert np.array_equal(loaded.run(feeds)["out"], out.float().cpu().numpy())


@pytest.mark.parametrize("kind", ["float16", "bfloat16"])
@pytest.mark.parametrize("rows,k,n,group,zero_points,bias", [(1, 4096, 2600, 128, True, True), (3, 1030, 9500, 16, True, False), (8, 2080, 4801, 32, False, True), (9, 1500, 6600, 64, True, True),
                                                             (16, 4100, 2400, 32, True, False), (13, 1024, 9500, 16, False, True), (2, 70001, 150, 256, True, False), (1, 8192, 1200, 1024, False, False), (16, 10000, 1000, 128, True, True)])
def test_linear_of_large_matrices(rows, k, n, group, zero_points, bias, kind):
    """Whole and cut blocks and groups, rows that fill shared memory and more than that, tiles that do not come out even."""
    s, x, y, w = check_linear(rows, k, n, group, kind, zero_points=zero_points, bias=bias, seed=rows + n)
    first = y.clone()
    for _ in range(3):
        run(s)
    assert torch.equal(first, y)


def test_linear_of_a_large_matrix_with_scales_beyond_f16():
    g = torch.Generator().manual_seed(71)
    for group in (16, 32, 128):
        w = D.linear_weights(g, 2401, 4111, group, True, True)
        w["scales"] = (w["scales"].astype(np.float32) * np.float32(1.00001)).astype(np.float32)
        x = torch.randn(5, 4111, generator=g).bfloat16()
        y = torch.empty(5, 2401, dtype=torch.bfloat16, device="cuda")
        run(session([linear_node(4111, 2401, group, w)], {"x": x.cuda()}, {"y": y}, w))
        within(y, D.linear(x, w, 4111), D.linear_bound(x, w, 4111, "bfloat16", rounded_weights=False))


def test_host_runs_follow_enqueued_ones():
    """run and the pipelined form right behind runs on another stream: the session's buffers are not theirs before."""
    p = D.Paged([1500, 1], [1500, 3000], 8, 2, 128, 16, "bfloat16", seed=72)
    p.kc, p.vc = torch.nan_to_num(p.kc), torch.nan_to_num(p.vc)
    s, dev, out = check_attend(p)
    want = out.clone()
    feeds = {n: (t.float() if t.is_floating_point() else t).cpu().numpy() for n, t in dev.items()}
    other = {**feeds, "query": feeds["query"] * 0.5}
    half = s.run(other)["out"]
    side = torch.cuda.Stream()
    for _ in range(3):
        out.zero_()
        side.wait_stream(torch.cuda.current_stream())
        for _ in range(8):
            s.enqueue(side.cuda_stream)
        assert np.array_equal(s.run(other)["out"], half)
        side.synchronize()
        assert torch.equal(out, want)
        out.zero_()
        side.wait_stream(torch.cuda.current_stream())
        for _ in range(8):
            s.enqueue(side.cuda_stream)
        assert all(np.array_equal(r["out"], half) for r in s.run_pipelined([other, other, other]))
        side.synchronize()
        assert torch.equal(out, want)


def test_linears_of_two_sessions_at_once():
    """The streaming kernel has no state of its own: two sessions on two streams, one of them replayed from a graph."""
    a, xa, ya, _ = check_linear(2, 4096, 2600, 32, "bfloat16", seed=73)
    b, xb, yb, _ = check_linear(7, 2500, 6000, 128, "float16", seed=74)
    wa, wb = ya.clone(), yb.clone()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=one):
        a.enqueue(torch.cuda.current_stream().cuda_stream)
    ya.zero_(), yb.zero_()
    torch.cuda.synchronize()
    for _ in range(20):
        with torch.cuda.stream(one):
            graph.replay()
        b.enqueue(two.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(ya, wa) and torch.equal(yb, wb)
