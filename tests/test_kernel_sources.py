"""Orders inside kernels that a run cannot show (a missing wait mostly goes unpunished): read from the sources."""
import re

import pytest

from conftest import ROOT

SOURCES = sorted((ROOT / "pytriton_llama_b200" / "csrc").glob("*.cu*"))


def _kernels(path):
    """(name, body) of every __global__ function of a source, comments left out."""
    text = re.sub(r"//[^\n]*", "", path.read_text())
    for m in re.finditer(r"__global__", text):
        open_at = text.index("{", m.end())
        depth, at = 1, open_at + 1
        while depth:
            depth += {"{": 1, "}": -1}.get(text[at], 0)
            at += 1
        names = [n for n in re.findall(r"(\w+)\s*\(", text[m.end():open_at]) if n != "__launch_bounds__"]
        yield names[0], text[open_at:at]


KERNELS = [(path.name, name, body) for path in SOURCES for name, body in _kernels(path)]
PEER_ACCESS = re.compile(r"\b(?:st_peer_\w+|ld_peer_\w+|mbar_arrive_cluster|tma_load_2d_pair)\s*\(")


@pytest.mark.parametrize("source,name,body", [k for k in KERNELS if PEER_ACCESS.search(k[2])], ids=lambda v: v if len(v) < 60 else "")
def test_peers_run_before_their_shared_memory_is_touched(source, name, body):
    """The shared memory of another block of a cluster may be used only once that block is known to run: a cluster barrier comes first."""
    waits = [m.start() for m in re.finditer(r"\bcluster_(?:wait|meet)\s*\(", body)]
    assert waits and waits[0] < PEER_ACCESS.search(body).start(), f"{source}: {name}"


@pytest.mark.parametrize("name,inputs", [("token_side_cluster_kernel", ["tokens", "table", "residual"]), ("sample_cluster_kernel", ["logits"]),
                                         ("decode_units_kernel", ["items", "tok_req", "positions"])])
def test_what_a_kernel_of_the_step_may_have_written_is_read_after_the_wait(name, inputs):
    """Reads above the wait on the predecessor are for what no kernel of the step writes; the step's tokens are not (a device kernel
    puts the sampled ones in), nor is what is read by them."""
    body = next(b for _, n, b in KERNELS if n == name)
    for array in inputs:
        read = re.search(rf"\b{array}\s*(?:\[|\+)", body)
        assert read and body.index("pdl_wait()") < read.start(), (name, array)


def test_the_kernels_with_clusters_are_found():
    found = {name for _, name, body in KERNELS if PEER_ACCESS.search(body)}
    assert {"decode_attention_kernel", "gemm_tc_kernel", "sample_cluster_kernel", "token_side_cluster_kernel"} <= found


def _blocks_around(body, at):
    """Where the blocks that hold a place of a kernel's body open, outermost first."""
    opened = []
    for i, c in enumerate(body[:at]):
        if c == "{":
            opened.append(i)
        elif c == "}":
            opened.pop()
    return opened


@pytest.mark.parametrize("source,name,body", [k for k in KERNELS if "pdl_launch_dependents()" in k[2]], ids=lambda v: v if len(v) < 60 else "")
def test_dependents_start_behind_the_wait_on_the_predecessor(source, name, body):
    """A kernel that let its successor start before it has waited itself would have three kernels run side by side, and the successor's
    reads ahead of its wait are right beside its predecessor only: on every path a wait of the same or an enclosing block comes first."""
    for launch in re.finditer(r"pdl_launch_dependents\(\)", body):
        around = _blocks_around(body, launch.start())
        waits = [_blocks_around(body, w.start()) for w in re.finditer(r"(?<=[;{}])\s*pdl_wait\(\);", body[:launch.start()])]
        assert any(w == around[:len(w)] for w in waits), f"{source}: {name}"


@pytest.mark.parametrize("name,reads", [("rope_kv8_write_kernel", ["p.block_of(", "p.angle(", "p.slots"]), ("read_kv8_kernel", ["block_table"]),
                                        ("kv8_expand_kernel", ["p.tiles", "p.block_table"])])
def test_integers_of_an_8_bit_cache_are_read_behind_a_wait(name, reads):
    """Slots, tables and tiles may come from the kernel directly before the call; only a caller that says otherwise (``early``) has them read
    ahead of the wait."""
    body = next(b for _, n, b in KERNELS if n == name)
    first_wait = re.search(r"(?:if \(!p\.early\) )?pdl_wait\(\);", body).start()
    for array in reads:
        assert array in body and first_wait < body.index(array), (name, array)
    if "p.early" in body:        # and what the kernel before this one computed is read behind a wait that every caller has
        assert re.search(r"(?<=[;{}])\s*pdl_wait\(\);\s*pdl_launch_dependents\(\);", body)


@pytest.mark.parametrize("name", ["prefill_attention_tc_kernel", "rope_kv8_write_kernel"])
def test_blocks_without_work_wait_too(name):
    """A kernel whose blocks all left without a wait would be through before its predecessor, and the kernel after it, which waits for this
    one only, would run beside what it counts on: a return ahead of the wait that every block with work has stands behind one of its own."""
    body = next(b for _, n, b in KERNELS if n == name)
    main = re.search(r"(?<=[;{}])\s*pdl_wait\(\);\s*pdl_launch_dependents\(\);\s*(?:__syncthreads|const)", body).start()
    inside = lambda at: re.search(r"\[&\]\([^)]*\)\s*$", body[:_blocks_around(body, at)[-1]])        # of a function of the kernel's own
    left = [m.start() for m in re.finditer(r"\breturn;", body[:main]) if "blockIdx" in body[:m.start()] and not inside(m.start())]
    assert left
    for at in left:
        around = _blocks_around(body, at)
        assert any(_blocks_around(body, w.start()) == around for w in re.finditer(r"(?<=[;{}])\s*pdl_wait\(\);", body[:at])), body[at - 200:at]
