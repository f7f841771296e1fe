"""Rules of the kernels on drafted tokens that no run shows, read from the sources: what breaks them shows up as a wrong value or a fault once in a long while, if at all."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "zllm_b200", "csrc")


def _source(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def test_verification_stores_into_ctas_that_run():
    """Shared memory of another CTA may be touched once that CTA has started, which a barrier of the cluster alone tells: every thread arrives at one as the kernel
    begins and waits for it, outside of any condition, before the first exchange and before it can leave."""
    text = _source("zq_verify.cu")
    kernel = text[text.index("verify_draft_kernel(const VerifyArgs a) {"):]
    kernel = kernel[:kernel.index("static int launch_verify")]
    arrive, wait = kernel.index("cluster.barrier_arrive();"), kernel.index("cluster.barrier_wait();")
    assert kernel.count("barrier_arrive") == kernel.count("barrier_wait") == 1
    first = min(kernel.index(word) for word in ("exchange_rows(", "exchange_sums(", "map_shared_rank", "cluster.sync()") if word in kernel)
    assert arrive < wait < first
    assert kernel[:arrive].count("{") - kernel[:arrive].count("}") == 1 and kernel[:wait].count("{") - kernel[:wait].count("}") == 1  # in the body itself
    assert "return" not in kernel[:wait]


def test_sums_in_tensor_memory_are_stored_before_they_are_loaded_again():
    """tcgen05.st and a later tcgen05.ld of the same columns: only tcgen05.wait::st between them orders the two.  Each row of V with an infinity adds to the same sums."""
    text = _source("zq_attn_wide.cu")
    loop = text[text.index("for (int r = 0; r < kWideTile; ++r) {"):]
    depth, end = 0, 0
    for end, c in enumerate(loop):
        depth += (c == "{") - (c == "}")
        if c == "}" and depth == 0:
            break
    body = loop[:end]
    assert body.index("tm_ld32(t_o") < body.index("tm_st32(t_o") < body.index("tm_st_wait();")


def test_tensor_memory_is_given_back_behind_its_last_products():
    """`wait` returns at once where any wait of the CTA has run out: the one in front of the deallocation must not."""
    text = _source("zq_attn_wide.cu")
    end = text[text.index("tc_commit(bars + kEnd)"):text.index("tcgen05.dealloc")]
    assert "mbar_wait_bounded(&bar.end, 0)" in end and not re.search(r"\bwait\(kEnd", end)
    assert end.index("mbar_wait_bounded(&bar.end, 0)") < end.index("__syncthreads();")
