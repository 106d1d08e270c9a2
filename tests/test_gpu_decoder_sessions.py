"""The decoder operators inside sessions: what stands next to them, what order their runs keep, what is left when one fails, and
which graphs are refused."""
import ctypes
import math
import os
import shutil
import subprocess

import numpy as np
import pytest

import decoder_oracle as D
import test_gpu_decoder as G
from oxionnx_b200 import _ffi
from oxionnx_b200.graph import Graph, Node
from oxionnx_b200.session import Declined, OnnxError, Session

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="session")
def session_state(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    lib = str(tmp_path_factory.mktemp("session_state") / "session_state.so")
    src = os.path.join(os.path.dirname(os.path.abspath(__file__)), "host_checks", "session_state.cpp")
    subprocess.run(["g++", "-std=c++17", "-O1", "-fPIC", "-shared", "-I/usr/local/cuda/include", "-o", lib, src], check=True)
    w = ctypes.CDLL(lib)
    w.error_word.restype = ctypes.POINTER(ctypes.c_int)
    w.error_word.argtypes = w.add_failing_step.argtypes = w.drop_last_step.argtypes = [ctypes.c_void_p]
    w.arrival_counts.restype = ctypes.c_uint32
    w.arrival_counts.argtypes = [ctypes.c_void_p, ctypes.POINTER(ctypes.c_void_p), ctypes.POINTER(ctypes.c_uint64), ctypes.c_uint32]
    return w


def device_words(ptr, count):
    """`count` int32 of device memory as a tensor over them."""
    holder = type("", (), {"__cuda_array_interface__": {"shape": (count,), "typestr": "<i4", "data": (ptr, False), "version": 3, "strides": None}})()
    return torch.as_tensor(holder, device="cuda")


def host_feeds(dev):
    return {n: (t.float() if t.is_floating_point() else t).cpu().numpy() for n, t in dev.items()}


# ---- beside kernels that hold tensor memory ------------------------------------------------------
@pytest.mark.parametrize("sequences", [8, 900])
def test_prompts_in_front_of_a_small_product(sequences):
    """A prompt kernel of 64-lane heads leaves room on its SM for a block of the small product kernel behind it, which takes its
    tensor memory before it waits: the prompt's own must have been taken by then.  With hundreds of sequences the prompt kernel
    is still counting them when the other starts.  Products of TF32 round both factors, 2^-11 of each at most."""
    new = [70 if i % 170 == 3 else 1 for i in range(sequences)]
    p = D.Paged(new, [n + i % 50 for i, n in enumerate(new)], 1, 1, 64, 16, "float16", seed=80)
    w = torch.randn(64, 32, generator=torch.Generator().manual_seed(80))
    dev = G.attend_inputs(p)
    z = torch.empty(p.q.shape[0], 32, device="cuda")
    nodes = [("OxiPagedAttention", "attend", list(dev), ["out"], {"num_heads": 1, "kv_num_heads": 1}), ("MatMul", "product", ["out", "w"], ["z"], {})]
    s = G.session(nodes, dev, {"z": z}, {"w": w.numpy()})
    assert any(step["kernel"].startswith("umma") for step in s.steps()), s.steps()
    want, bound = D.attend(p)
    bound = bound @ w.double().abs() + (2 * 2.0**-11 + 66 * 2.0**-23) * (1 + 2.0**-10) * ((want.abs() + bound) @ w.double().abs())
    for _ in range(20):
        z.fill_(math.nan)
        G.run(s)
        G.within(z, want @ w.double(), bound)


# ---- views of a cache ----------------------------------------------------------------------------
SHAPES = {"query": (3, 256), "key": (3, 128), "value": (3, 128), "key_cache": (5, 16, 2, 64), "value_cache": (5, 16, 2, 64), "cu_query": (3,), "kv_lengths": (2,), "page_table": (2, 3)}
HEADS = {"num_heads": 4, "kv_num_heads": 2}


def append_node(kc, vc, out="", name="append"):
    return Node("OxiPagedCacheAppend", name, ["query", "key", "value", kc, vc, *G.TABLES], ["a" + out, "b" + out, "c" + out], HEADS)


def view(src, dst, op="Identity"):
    return Node(op, f"{src}-{dst}", [src, "cache_shape"] if op == "Reshape" else [src], [dst], {})


@pytest.mark.parametrize("nodes,outs,match", [
    # another reader of the input behind the view, a graph output out of it, the input itself as an output
    ([view("key_cache", "k"), append_node("k", "value_cache"), Node("OxiPagedAttention", "t", ["a", "key_cache", "c", *G.TABLES], ["y"], HEADS)], ["y"], "updated where it lies"),
    ([view("key_cache", "k"), append_node("k", "value_cache"), view("key_cache", "y")], ["a", "y"], "updated where it lies"),
    ([view("key_cache", "k", "Reshape"), append_node("k", "value_cache"), view("key_cache", "y")], ["a", "y"], "updated where it lies"),
    ([view("value_cache", "v"), append_node("key_cache", "v")], ["a", "value_cache"], "updated where it lies"),
    ([view("key_cache", "k"), view("k", "l"), append_node("l", "value_cache")], ["a", "k"], "updated where it lies"),
    # two appends on two views, one of them of the cache from before the other
    ([view("key_cache", "k"), append_node("k", "value_cache"), view("key_cache", "l"), append_node("l", "c", "2", "again")], ["a", "a2"], "updated where it lies"),
    # one input as both caches
    ([view("key_cache", "k"), view("key_cache", "l"), append_node("k", "l")], ["a"], "one buffer for keys and values"),
    ([view("key_cache", "k"), append_node("k", "key_cache")], ["a"], "one buffer for keys and values"),
])
def test_append_refuses_views_of_a_cache_that_something_else_reads(nodes, outs, match):
    used = {i for n in nodes for i in n.inputs} | set(outs)
    inputs = [n for n in SHAPES if n in used]
    types = {n: "int32" if n in G.TABLES else "float16" for n in inputs}
    weights = {"cache_shape": torch.tensor(SHAPES["key_cache"]).float().numpy()}
    with pytest.raises(Declined, match=match):
        Session.builder().with_input_shapes({n: SHAPES[n] for n in inputs}).with_input_types(types).build_from_graph(Graph(nodes, inputs, outs), weights).ensure_planned()


def test_append_through_views_that_nothing_else_reads():
    """A chain of views in front and two appends in a row, the second on the first one's outputs."""
    p = D.Paged([2, 1], [20, 3], 4, 2, 64, 16, "float16", seed=81)
    dev = {"query": p.q.cuda(), "key": p.k.cuda(), "value": p.v.cuda(), "flat": p.kc.reshape(-1).cuda(), "value_cache": p.vc.cuda(), "cu_query": p.cu.cuda(), "kv_lengths": p.len.cuda(),
           "page_table": p.table.cuda()}
    out = torch.full(p.q.shape, math.nan, dtype=torch.float16, device="cuda")
    heads = {"num_heads": 4, "kv_num_heads": 2}
    nodes = [("Reshape", "r", ["flat", "cache_shape"], ["k"], {}), ("Identity", "i", ["k"], ["l"], {}),
             ("OxiPagedCacheAppend", "one", ["query", "key", "value", "l", "value_cache", *G.TABLES], ["a", "b", "c"], heads),
             ("OxiPagedCacheAppend", "two", ["query", "key", "value", "b", "c", *G.TABLES], ["a2", "b2", "c2"], heads)]
    s = G.session(nodes, dev, {"a2": out}, {"cache_shape": torch.tensor(p.kc.shape).float().numpy()})
    G.run(s)
    (rotated, bound), (kc, _), vc = D.append(p, None, None, False)
    G.within(out, rotated, bound)
    got = dev["flat"].view(kc.shape).double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(kc)) and torch.equal(torch.nan_to_num(got), torch.nan_to_num(kc))
    assert torch.equal(torch.nan_to_num(dev["value_cache"].cpu()), torch.nan_to_num(vc))


# ---- after a kernel has given up -----------------------------------------------------------------
@pytest.mark.parametrize("way", ["collect", "run", "wait", "resident"])
def test_a_run_that_gave_up_leaves_no_counts_of_parts(session_state, way):
    """The error word set as a bounded wait that ran out sets it, counts of parts left as a block that gave up leaves them:
    whichever call reports it clears them, so that the next run does not join parts too early."""
    p = D.Paged([1, 300], [3000, 1500], 8, 2, 128, 16, "bfloat16", seed=82)
    p.kc, p.vc = torch.nan_to_num(p.kc), torch.nan_to_num(p.vc)
    s, dev, out = G.check_attend(p)
    want = out.float().cpu().numpy()
    feeds = host_feeds(dev)
    ptr, size = (ctypes.c_void_p * 4)(), (ctypes.c_uint64 * 4)()
    assert session_state.arrival_counts(s.ctx.handle, ptr, size, 4) == 1
    words = device_words(ptr[0], size[0] // 4)
    s.run(feeds)
    if way == "collect":
        s.submit(feeds)
    elif way == "wait":
        s.enqueue(0)
    torch.cuda.synchronize()
    words.fill_(1)
    torch.cuda.synchronize()
    session_state.error_word(s.ctx.handle)[0] = 43
    with pytest.raises(OnnxError, match="43"):
        {"collect": s.collect, "run": s.download, "wait": s.wait, "resident": lambda: s.run_resident(0)}[way]()
    torch.cuda.synchronize()
    assert int(words.count_nonzero()) == 0, "counts of parts are left behind"
    assert np.array_equal(s.run(feeds)["out"], want)


# ---- the order of one session's runs ---------------------------------------------------------------
def refused_calls(s):
    """Calls that the library refuses after it has begun them."""
    lib, h = _ffi.lib(), s.ctx.handle
    fetches = (_ffi.Result * 1)()

    def submit_nothing():
        return lib.oxb200_run_submit(h, None, 0)

    def run_nothing():
        return lib.oxb200_run(h, None, 0, fetches, 1)

    def fetch_nothing():
        return lib.oxb200_fetch_value(h, b"query", ctypes.byref(_ffi.Result(lanes=(ctypes.c_float * 1)(), cap=1)))

    def bound_without_a_feed():
        return lib.oxb200_run_bound(h, None, 0, fetches, 1)

    return {"run": run_nothing, "submit": submit_nothing, "fetch": fetch_nothing, "bound": bound_without_a_feed}


@pytest.mark.parametrize("call", ["run", "submit", "fetch", "bound", "upload"])
def test_a_refused_call_between_two_enqueued_runs_leaves_their_order(call):
    """A run behind 100 ms of sleep on one stream, a call that is refused, a run on another stream: the second run ends after
    the first."""
    p = D.Paged([1, 90], [50, 90], 4, 2, 64, 16, "float16", seed=86)
    p.kc, p.vc = torch.nan_to_num(p.kc), torch.nan_to_num(p.vc)
    s, dev, out = G.check_attend(p)
    want = out.clone()
    feeds = host_feeds(dev)
    calls = refused_calls(s)
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    first, second = torch.cuda.Event(), torch.cuda.Event()
    for _ in range(2):
        out.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(one):
            torch.cuda._sleep(200_000_000)
        s.enqueue(one.cuda_stream)
        first.record(one)
        if call == "upload":  # its copies have begun when the last feed turns out to be missing
            lib = _ffi.lib()
            ops, keep = (_ffi.Operand * (len(feeds) - 1))(), _ffi.Keep()
            names = list(feeds)[:-1]
            for op, n in zip(ops, names):
                code = _ffi.dtype_code(s._input_types[n])
                _ffi.pack_operand(op, n, _ffi.lanes_of(feeds[n], code), keep, dtype=code)
            assert lib.oxb200_upload_feeds(s.ctx.handle, ops, len(names)) == _ffi.FAILED
        elif call == "bound":
            s.clear_bindings()
            assert calls[call]() == _ffi.FAILED
            for n, t in dev.items():
                s.bind_input_device(n, t.data_ptr(), G.name_of(t), t.numel())
            s.bind_output_device("out", out.data_ptr(), out.numel(), "float16")
        else:
            assert calls[call]() == _ffi.FAILED
        s.enqueue(two.cuda_stream)
        second.record(two)
        second.synchronize()
        assert first.query(), "the second run did not wait for the first"
        s.wait()
        assert torch.equal(out, want)


def test_a_run_that_failed_half_way_is_waited_for(session_state):
    """A launch that fails behind others: what is in the stream of that run still comes before the next one."""
    p = D.Paged([1, 90], [50, 90], 4, 2, 64, 16, "float16", seed=87)
    s, dev, out = G.check_attend(p)
    want = out.clone()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    first, second = torch.cuda.Event(), torch.cuda.Event()
    out.zero_()
    torch.cuda.synchronize()
    with torch.cuda.stream(one):
        torch.cuda._sleep(200_000_000)
    session_state.add_failing_step(s.ctx.handle)
    with pytest.raises(OnnxError, match="a step that fails"):
        s.enqueue(one.cuda_stream)
    session_state.drop_last_step(s.ctx.handle)
    first.record(one)
    s.enqueue(two.cuda_stream)
    second.record(two)
    second.synchronize()
    assert first.query(), "the second run did not wait for what the failed one had launched"
    s.wait()
    assert torch.equal(out, want)


def test_host_runs_then_enqueued_ones():
    """run and the pipelined form end before they return; a run enqueued behind them reads its own inputs."""
    p = D.Paged([1, 90], [50, 90], 4, 2, 64, 16, "float16", seed=88)
    p.kc, p.vc = torch.nan_to_num(p.kc), torch.nan_to_num(p.vc)
    s, dev, out = G.check_attend(p)
    want = out.clone()
    feeds = host_feeds(dev)
    feeds["query"] = feeds["query"] * 0.5
    half = s.run(feeds)["out"]
    stream = torch.cuda.Stream()
    for _ in range(5):
        assert np.array_equal(s.run(feeds)["out"], half)
        s.enqueue(stream.cuda_stream)
        assert all(np.array_equal(r["out"], half) for r in s.run_pipelined([feeds] * 3))
        s.enqueue(stream.cuda_stream)
        s.wait()
        assert torch.equal(out, want)


# ---- f32 lanes of outputs that a run left in the caller's buffer -----------------------------------
def test_lanes_that_the_last_run_did_not_make_are_not_handed_out():
    p = D.Paged([1, 90], [50, 90], 4, 2, 64, 16, "float16", seed=84)
    s, dev, out = G.check_attend(p)  # enqueued with `out` bound in its own type: f32 lanes were never made
    for call in (s.download, lambda: s.output_device_ptr("out"), lambda: s.fetch_value("out")):
        with pytest.raises(OnnxError, match="own type"):
            call()
    s.clear_bindings()
    for call in (s.download, lambda: s.output_device_ptr("out"), lambda: s.fetch_value("out")):
        with pytest.raises(OnnxError, match="own type"):
            call()
    for n, t in dev.items():
        s.bind_input_device(n, t.data_ptr(), G.name_of(t), t.numel())
    want = out.float().cpu().numpy()
    assert np.array_equal(s.run_with_binding()["out"], want)  # makes them
    assert np.array_equal(s.download()["out"], want) and np.array_equal(s.fetch_value("out"), want) and s.output_device_ptr("out")[1] == want.size
    # the pipelined form makes its own, and a bound run without fetches leaves them out again
    s.bind_output_device("out", out.data_ptr(), out.numel(), "float16")
    p2 = dev["query"].clone()
    dev["query"].mul_(0.5)
    s.run_with_binding(fetch=False)
    dev["query"].copy_(p2)
    s.clear_bindings()
    with pytest.raises(OnnxError, match="own type"):
        s.download()


def test_one_output_in_its_own_type_beside_one_in_f32():
    """Only what the run left out is refused."""
    g = torch.Generator().manual_seed(85)
    w = D.linear_weights(g, 64, 64, 32, False, False)
    x = torch.randn(4, 64, generator=g).half().cuda()
    y, z = torch.empty(4, 64, dtype=torch.float16, device="cuda"), torch.empty(4, 64, device="cuda")
    s = G.session([G.linear_node(64, 64, 32, w, "y"), ("Add", "s", ["y", "x"], ["z"], {})], {"x": x}, {"y": y, "z": z}, w)
    s.bind_output_device("z", z.data_ptr(), z.numel())
    G.run(s)
    s.clear_bindings()
    assert np.array_equal(s.fetch_value("z"), z.cpu().numpy())
    with pytest.raises(OnnxError, match="own type"):
        s.output_device_ptr("y")
    s.bind_input_device("x", x.data_ptr(), "float16", x.numel())
    s.enqueue(0)
    s.wait()
    got = s.download()
    assert np.array_equal(got["y"], y.float().cpu().numpy()) and np.array_equal(got["z"], z.cpu().numpy())


# ---- what the error word says --------------------------------------------------------------------
def test_every_call_that_waits_says_what_is_wrong():
    """Bounds that fall also give a sequence two rows where one was promised: the word holds either."""
    p = D.Paged([1, 1], [40, 30], 4, 2, 64, 16, "float16", seed=83)
    p.kc, p.vc = torch.nan_to_num(p.kc), torch.nan_to_num(p.vc)
    s, dev, out = G.check_attend(p)
    good = host_feeds(dev)
    for change, match in (({"page_table": np.full_like(good["page_table"], 10_000)}, "page table"), ({"cu_query": np.array([0, 2, 1], np.int32)}, "cu_query|max_query_length"),
                          ({"cu_query": np.array([0, 0, 2], np.int32)}, "max_query_length")):
        bad = {**good, **change}
        with pytest.raises(OnnxError, match=match):
            s.run(bad)
        s.upload(bad)
        with pytest.raises(OnnxError, match=match):
            s.run_resident(1)
        s.submit(bad)
        with pytest.raises(OnnxError, match=match):
            s.collect()
        assert np.array_equal(s.run(good)["out"], out.float().cpu().numpy())


def test_a_linear_and_a_small_product_on_two_streams():
    """Both run in clusters whose blocks take tensor memory and meet; side by side on the same SMs they end, and give what each
    gives alone."""
    g = torch.Generator().manual_seed(89)
    w = D.linear_weights(g, 1024, 4096, 32, True, False)
    x, y = torch.randn(64, 4096, generator=g).bfloat16().cuda(), torch.empty(64, 1024, dtype=torch.bfloat16, device="cuda")
    a = G.session([G.linear_node(4096, 1024, 32, w)], {"x": x}, {"y": y}, w)
    u, z = torch.randn(256, 2048, generator=g).cuda(), torch.empty(256, 256, device="cuda")
    b = G.session([("MatMul", "product", ["u", "w"], ["z"], {})], {"u": u}, {"z": z}, {"w": torch.randn(2048, 256, generator=g).numpy()})
    G.run(a), G.run(b)
    first, second = y.clone(), z.clone()
    y.zero_(), z.zero_()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(300):
        a.enqueue(streams[0].cuda_stream)
        b.enqueue(streams[1].cuda_stream)
    a.wait(), b.wait()
    assert torch.equal(y, first) and torch.equal(z, second)


# ---- beside operators on f32 lanes -----------------------------------------------------------------
@pytest.mark.parametrize("kind", ["float16", "bfloat16"])
def test_a_typed_input_of_a_product_with_16_bit_weights(kind):
    """The product takes 16-bit operands: its copy of the input's f32 lanes stands beside the input in its own type."""
    g = torch.Generator().manual_seed(90)
    x, w = torch.randn(24, 64, generator=g).to(D.TYPES[kind]), torch.randn(64, 32, generator=g).half()
    graph = Graph([Node("MatMul", "m", ["x", "w"], ["y"], {}), Node("Add", "a", ["y", "b"], ["z"], {})], ["x"], ["z"])
    got = Session.builder().with_input_types({"x": kind}).build_from_graph(graph, {"w": w.numpy(), "b": np.ones(32, np.float32)}).run({"x": x.float().numpy()})["z"]
    want = x.double() @ w.double() + 1
    # bf16 rows meet f16 weights as whichever type the product takes, rounded once
    size = x.double().abs() @ w.double().abs()
    G.within(torch.from_numpy(got), want, (2.0**-11 if kind == "bfloat16" else 0.0) * size + 66 * 2.0**-23 * (size + 1))


@pytest.mark.parametrize("views", [[], ["Identity"], ["Relu", "Reshape"]])
def test_rows_that_a_product_reads_too_are_whole_to_a_linear(views):
    """A product's output that another product reads leaves as TF32, the operands of that; a 4-bit linear that reads it too takes
    all of its bits, the same as without the other product."""
    g = torch.Generator().manual_seed(91)
    w = D.linear_weights(g, 48, 64, 32, True, False)
    x, m, o = torch.randn(40, 96, generator=g), torch.randn(96, 64, generator=g), torch.randn(64, 16, generator=g)
    weights = {**w, "m": m.numpy(), "o": o.numpy(), "shape": np.array([40, 64], np.float32)}
    nodes, last = [Node("MatMul", "m", ["x", "m"], ["a"], {})], "a"
    for i, op in enumerate(views):
        nodes.append(Node(op, f"view{i}", [last, "shape"] if op == "Reshape" else [last], [f"v{i}"], {}))
        last = f"v{i}"
    nodes.append(Node(*G.linear_node(64, 48, 32, w, "y", last)))
    want = Session.builder().build_from_graph(Graph(nodes, ["x"], ["y"]), weights).run({"x": x.numpy()})["y"]
    got = Session.builder().build_from_graph(Graph([*nodes, Node("MatMul", "o", ["a", "o"], ["p"], {})], ["x"], ["y", "p"]), weights).run({"x": x.numpy()})
    assert np.array_equal(got["y"], want)
    a = x.double() @ m.double()
    size = x.double().abs() @ m.double().abs() @ o.double().abs()
    G.within(torch.from_numpy(got["p"]), a @ o.double(), (4 * 2.0**-11 + 164 * 2.0**-23) * (1 + 2.0**-9) * size)


def test_a_pipelined_run_uploads_behind_an_enqueued_one():
    """An input that the product's kernel reads at a fixed address is copied there by the enqueued run, behind 100 ms of sleep, and
    uploaded there by the pipelined one: the upload is the later of the two, also when a refused call came in between."""
    g = torch.Generator().manual_seed(92)
    w, x = torch.randint(-127, 128, (256, 128), generator=g), torch.randint(0, 255, (512, 256), generator=g, dtype=torch.uint8)
    u, z = x.cuda(), torch.empty(512, 128, device="cuda")
    graph = Graph([Node("MatMulInteger", "product", ["u", "w"], ["p"], {}), Node("Cast", "c", ["p"], ["z"], {"to": 1})], ["u"], ["z"])
    s = Session.builder().with_input_types({"u": np.uint8}).with_input_shapes({"u": (512, 256)}).build_from_graph(graph, {"w": w.float().numpy()})
    s.ensure_planned()
    s.bind_input_device("u", u.data_ptr(), np.uint8, u.numel())
    s.bind_output_device("z", z.data_ptr(), z.numel())
    G.run(s)
    first = z.clone()
    assert torch.equal(first.cpu().long(), x.long() @ w)
    feeds = {"u": (x // 2).numpy()}
    half = s.run(feeds)["z"]
    assert np.array_equal(half, ((x // 2).long() @ w).float().numpy())
    assert np.array_equal(s.run_pipelined([feeds])[0]["z"], half)
    one = torch.cuda.Stream()
    for refused in (False, True):
        z.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(one):
            torch.cuda._sleep(200_000_000)
        s.enqueue(one.cuda_stream)
        if refused:
            assert _ffi.lib().oxb200_run(s.ctx.handle, None, 0, (_ffi.Result * 1)(), 1) == _ffi.FAILED
        s.submit(feeds)
        assert np.array_equal(s.collect()["z"], half)
        one.synchronize()
        assert torch.equal(z, first)
