"""What the device-planned cache does when something fails, checked in its
source: a bounded wait that runs out in its kernels, or a captured call whose
workspace cannot be cleared, cannot be caused without a fault, so what keeps
warps from waiting for one another for ever, and memory from staying, is read
here."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "whisper.rs_b200", "csrc")


def source(name):
    text = open(os.path.join(CSRC, name)).read()
    return re.sub(r"//[^\n]*", "", text)


def test_softmax_warps_meet_with_a_limit():
    """The wide kernel's softmax warps leave one by one where a wait runs out:
    none may wait for the others at a barrier without a limit."""
    text = source("paged_attend_wide.cu")
    assert not re.search(r"\bbar(rier)?(\.cta)?\.(sync|red)", text)
    body = text[text.index("void pw_softmax("):text.index("paged_attend_wide_kernel(")]
    assert "__syncthreads" not in body
    calls = re.findall(r"[^\n]*\bpw_sync\([^\n]*", body)
    assert len(calls) == 6 and all(re.match(r"\s*if \(!pw_sync\(.*\) return;", c) for c in calls)


def test_lanes_leave_together():
    """Where a wait's result decides what a whole warp does next, its lanes go
    the same way: it may run out for some of them only. They vote, or those
    end the warp's share in what all of them read next."""
    text = source("paged_attend.cu")
    kernel = text[text.index("paged_attend_stream_kernel("):text.index("int pa_sms()")]
    assert kernel.count("mbar_wait(") == 2
    assert re.search(r"if \(!__all_sync\(0xffffffffu, mbar_wait\([^;]*\)\)\)\s*break;", kernel)
    assert re.search(r"if \(!mbar_wait\([^;]*\)\)\s*s\.queue\[warp\]\[i % kPaQueue\]\.nr = 0;\s*__syncwarp\(\);"
                     r"\s*\}\s*const PaItem it = s\.queue\[warp\]\[i % kPaQueue\];\s*if \(it\.nr == 0\) break;", kernel)
    assert len(re.findall(r"\bif \(!mbar_wait\(", text)) == 1
    wide = source("paged_attend_wide.cu")
    softmax = wide[wide.index("void pw_softmax("):wide.index("paged_attend_wide_kernel(")]
    load = wide[wide.index("void pw_load("):wide.index("void pw_products(")]
    for body in (softmax, load):
        assert "mbar_wait(" in body and not re.search(r"\bif \(!mbar_wait\(", body)


def test_a_captured_workspace_is_freed_on_every_way_out():
    """After its allocation joins a graph, a call ends by freeing it."""
    text = source("paged_attend.cu")
    rest = text[text.index("cudaMallocAsync(&own"):]
    failed = rest[rest.index("cudaMemsetAsync(own"):]
    assert failed.index("cudaFreeAsync(own, st)") < failed.index("return")
    done = rest[rest.index("rc = launch_attend("):]
    assert done.index("cudaFreeAsync(own, st)") < done.index("return")
