"""Source audit of the integer product's kernels for what no test may bring about on a GPU: waits that run out."""
import os
import re

SRC = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "csrc", "gemm_int8.cu")).read()


def _body(name):
    """The kernel's statements, without comments."""
    m = re.search(r"__global__[^{;]*\b" + name + r"\s*\([^{]*\{", SRC)
    depth, i = 1, m.end()
    while depth:
        depth += {"{": 1, "}": -1}.get(SRC[i], 0)
        i += 1
    return re.sub(r"//[^\n]*", "", SRC[m.end():i])


def _roles(body):
    """Statements of the copying, the issuing and the storing warps (the branches on the warp index)."""
    a = body.index("if (warp == 0) {")
    b = body.index("} else if (warp == 1) {", a)
    c = re.compile(r"\n  \} else \{|\n  if \(warp >= 2\) \{").search(body, b).start()
    return body[a:b], body[b:c], body[c:]


def test_bounded_waits_start_behind_the_predecessor():
    """A kernel may be resident long before its inputs are written. A warp that polled a barrier before griddepcontrol.wait
    would time the predecessors' work and give up on a copy that was never late."""
    for name in ("gemm_int8_kernel", "gemm_int8_pair_kernel"):
        for role in _roles(_body(name)):
            assert "pdl_wait()" in role and role.index("pdl_wait()") < role.index("mbar_wait("), (name, role[:200])


def test_a_lost_part_is_never_summed():
    """With K split over a cluster, a part whose wait ran out has no sums to give. It says so to every part, and no part
    stores: a row that lacks a piece of K would look like a result."""
    for name in ("gemm_int8_kernel", "gemm_int8_pair_kernel"):
        body = _body(name)
        assert re.search(r"if \(have\) send_partials\(.*?\);\s*else report_lost\(lost, p\.split, to_rank\);", body, re.S), name
        assert re.search(r"cluster_sync_all\(\);\s*if \(warp >= 2 && !\*lost\) finish_partials", body), name
        assert re.search(r"\*lost = 0;.*fence_mbar_init\(\)", body, re.S) and body.index("*lost = 0") < body.index("cluster_sync_all()")


def test_failed_blocks_outlive_their_copies():
    """A block that gave up waits for what is in flight: it looks at the flag once all its warps (the pair: both CTAs) have
    passed the last point at which they may set it."""
    for name, last in (("gemm_int8_kernel", "__syncthreads()"), ("gemm_int8_pair_kernel", "cluster_sync_all()")):
        body = _body(name)
        look = body.index("if (*abort_flag)")
        assert body.rindex("fail(VG_ERR") < body.rindex(last) < look < body.index("dealloc"), name
        assert "__nanosleep" in body[look:]
    assert "smem_u32(const_cast<const int*>(abort_flag)), crank ^ 1)" in _body("gemm_int8_pair_kernel")


def test_dependents_start_behind_the_tensor_memory_allocation():
    """A dependent kernel may allocate all of an SM's tensor memory and then wait for this grid to end. Were this grid's own
    allocation still to come, neither would move on."""
    for name, alloc in (("gemm_int8_kernel", "tmem_alloc("), ("gemm_int8_pair_kernel", "tcgen05.alloc")):
        body = _body(name)
        assert body.index(alloc) < body.index("__syncthreads()") < body.index("pdl_trigger()"), name
