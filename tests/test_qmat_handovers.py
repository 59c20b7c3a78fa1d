"""How the products' kernels hand back what asynchronous copies or the tensor core write next.  Read from the sources."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vq_b200", "csrc")


def source(name):
    return re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())


def test_places_of_the_ring_are_released():
    """A place's values are read by ordinary loads and overwritten by a copy that another warp asks for: the arrival between the two releases."""
    text = source("product_few.cu")
    assert "mbar_arrive(&empty[st])" in text and "relaxed" not in text


def test_a_relaxed_arrival_stands_between_the_fences_of_tensor_memory():
    """Only accumulators are handed back that way: loads have been waited for, the fence is before the arrival, and the other one behind the wait for it."""
    text = source("product_tc.cu")
    uses = [m.start() for m in re.finditer(r"arrive_at\(in_cta\(&bars->tempty", text)]
    assert len(uses) == 1 and text.count("arrive_at(") == 2  # (its definition)
    before = text[:uses[0]]
    assert before.rindex("__syncwarp();") > before.rindex("tcgen05.fence::before_thread_sync;")
    behind = text[re.search(r"mbar_wait\(&bars->tempty\[b\]", text).end():]
    assert behind.index("tcgen05.fence::after_thread_sync;") < behind.index("umma_i8(")
    for read in re.finditer(r"has_been_read\(\);", text):  # the last of a warp's loads has been waited for, or there was none
        lead = text[:read.start()]
        assert lead.rindex("tmem_wait();") > lead.rindex("tmem_ld32_issue(") or lead.rstrip().endswith("if (32 * turn >= columns)")
