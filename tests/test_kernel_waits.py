"""What the sources of the kernels with bounded waits have to keep to, and no run of them shows."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sana_b200", "csrc")


def code(name):
    src = open(os.path.join(CSRC, name)).read()
    src = re.sub(r"//[^\n]*|/\*.*?\*/", "", src, flags=re.S)
    return re.sub(r"\\[nt]", " ", src)  # the line breaks inside assembly strings


def test_a_barrier_object_is_initialised_once():
    """mbarrier.init on a live barrier object is undefined: the decaying attention goes through its barriers in one loop,
    which knows the arrivals of each."""
    assert len(re.findall(r"\bmbar_init\s*\(", code("la_decay_tc.cu"))) == 1


def test_no_role_waits_without_a_limit():
    """A role that has given up leaves for the last __syncthreads(); a named barrier that its siblings enter after that
    would never fill.  The one there is (among the warps of the state) is entered by each of them once a chunk, whatever
    its bounded waits have said, and decides for all of them whether to leave."""
    src = code("la_decay_tc.cu")
    assert len(re.findall(r"__syncthreads\s*\(", src)) == 2  # after the set-up, and before tensor memory is freed
    assert re.findall(r"\b(?:bar|barrier)\.[a-z.]*", src) == ["bar.red.and.pred"]
    state = src[src.index("if (warp < 4)"):src.index("} else if (warp < 8)")]
    loop = state[state.index("for (int c = 0; c < chunks; ++c)"):]
    before, after = loop.split("lt_all(ok)")
    assert not re.search(r"\b(break|return|continue)\b", before)
    # behind it: out of the loop at once when it says so (heads that do not meet there leave alone), else only to the next chunk
    assert re.match(r";\s*if \(!ok\) break;", after) and len(re.findall(r"\bbreak\b", after)) == 2 and "return" not in after
    assert re.search(r"else if \(!ok\) \{\s*break;", after)


def test_a_kernel_that_gives_up_lets_its_copies_and_products_end():
    """Whichever role's wait ran out: before the last rendezvous all warps look at the flag and leave time for the copies
    into shared memory and the products into tensor memory that are still under way."""
    pause = re.compile(r"if \(\*abort_flag\) \{\s*const long long t0 = clock64\(\);\s*while \(clock64\(\) - t0 < 2000000LL\) \{\}\s*\}")
    for name, kernels in (("la_decay_tc.cu", 1), ("gemm_fp8.cu", 2)):
        src = code(name)
        ends = [m.start() for m in re.finditer(r"tcgen05\.dealloc", src)]
        assert len(ends) == kernels
        for e in ends:
            last_sync = src.rindex("__syncthreads()", 0, e)
            assert any(0 < last_sync - m.end() < 200 for m in pause.finditer(src)), (name, e)
