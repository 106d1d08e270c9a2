"""Rules that the device code keeps and that no run may be made to break, read from the sources."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "oxionnx_b200", "csrc")


def functions(name):
    """(name, body without comments) of every kernel and inlined device procedure of a source file."""
    with open(os.path.join(CSRC, name)) as fh:
        text = re.sub(r"//[^\n]*", "", fh.read())
    text = re.sub(r"__launch_bounds__\([^{;]*?\)\s+(?=\w+\()", "", text)
    for m in re.finditer(r"(?:__global__|__device__ __forceinline__)\s+void\s+(\w+)\([^{;]*\{", text):
        depth, at = 1, m.end()
        while depth:
            depth += {"{": 1, "}": -1}.get(text[at], 0)
            at += 1
        yield m.group(1), text[m.end() : at]


SOURCES = sorted(f for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh")))


def test_kernels_let_their_successor_in_behind_their_tensor_memory():
    """A dependent grid starts once every block of this one has said so, and may take tensor memory before it waits.  Said in
    front of the block's own allocation, that allocation can wait for columns which the successor holds until this grid ends."""
    seen = 0
    for source in SOURCES:
        for name, body in functions(source):
            alloc = [m.start() for m in re.finditer(r"tcgen05\.alloc", body)]
            lets_in = [m.start() for m in re.finditer(r"griddepcontrol\.launch_dependents|pdl_enter\(\)", body)]
            if alloc and lets_in:
                seen += 1
                assert min(lets_in) > max(alloc), f"{source}: {name}"
    assert seen >= 5


def test_blocks_that_others_read_from_leave_together():
    """Shared memory that the peers of a cluster read goes away with its block: the last thing that all of the cluster does,
    outside of any branch that depends on a block's own work or on its having given up, is a barrier of the cluster."""
    for source, name in (("umma_chain.cu", "umma_chain_kernel"), ("linear4.cu", "linear4_rows"), ("umma_linear4.cu", "umma_linear4_kernel")):
        body = dict(functions(source))[name]
        reads = [m.start() for m in re.finditer(r"ld_dsmem_v4\(|map_shared_rank\(", body)]
        barriers = [m.start() for m in re.finditer(r"cluster_sync_all\(\)|cluster\.sync\(\)", body)]
        assert reads and barriers and barriers[-1] > reads[-1], source
        depth = body[: barriers[-1]].count("{") - body[: barriers[-1]].count("}")
        assert depth <= 1, f"{source}: the last barrier of the cluster stands inside of {depth} blocks"
    assert "if (clustered) cluster_sync_all();" in dict(functions("umma_chain.cu"))["umma_chain_kernel"]


def test_blocks_of_the_linear_hold_no_tensor_memory_while_they_wait_for_their_cluster():
    """Two kernels of clusters on two streams, each with a block that waits for the other's columns, would wait for good if blocks
    kept theirs while they wait for their peers.  The other kernels of clusters take so much shared memory beside their columns that
    those of one SM never run out; this one takes all columns and little more than half of the shared memory."""
    body = dict(functions("umma_linear4.cu"))["umma_linear4_kernel"]
    assert body.count("tcgen05.dealloc") == 1 and body.index("tcgen05.dealloc") < body.index("cluster.sync()")


def test_codes_of_the_error_word_say_one_thing():
    """The codes that have a text of their own are no kernel's code of a wait that ran out."""
    with open(os.path.join(CSRC, "decoder.hpp")) as fh:
        named = {int(c) for c in re.findall(r"kErr\w+ = (\d+)", fh.read())}
    assert len(named) == 4
    waits = set()
    for source in SOURCES:
        for _, body in functions(source):
            waits |= {int(c) for c in re.findall(r"(?:give_up\(|fail\(abortp, p\.err_flag, |atomicExch\([^;]*?err[^;]*?, )(\d+)\)", body)}
            waits |= {int(c) for c in re.findall(r"wait\(bar_\w+(?:\[[^;]*?\])?, [^;]*?, (\d+)\)", body)}
    assert len(waits) > 15 and not waits & named, sorted(waits & named)
