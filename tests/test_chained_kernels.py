"""Rules of kernels that are set up while the kernel before them ends, read off their sources: breaking one can leave a GPU
waiting for good, so none is tried out."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "streamdiffusionv2_b200", "csrc")
SOURCES = ["q8_cache.cu", "attn_q8_few.cu", "attn_q8_spans.cu"]


def _kernels(name):
    """(kernel name, body without comments) of every __global__ function of a source."""
    text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())
    for part in text.split("__global__")[1:]:
        body = part[:part.index("\n}\n")]
        yield re.search(r"(\w+)\s*\(const __grid_constant__", body).group(1), body


def test_every_chained_kernel_is_looked_at():
    launched = [f for f in sorted(os.listdir(CSRC)) if f.endswith(".cu") and "launch_chained(" in open(os.path.join(CSRC, f)).read()]
    assert sorted(launched) == sorted(SOURCES)


@pytest.mark.parametrize("name", SOURCES)
def test_tensor_memory_is_held_before_the_next_kernel_may_come_in(name):
    """The next kernel may allocate tensor memory in its set-up and then wait for this one: by then every block of this one
    must have its own, so the release stands behind a block barrier that follows the allocation.  Before the wait
    nothing is released."""
    for kernel, body in _kernels(name):
        begin = re.search(r"(begin_after|wait_for)_previous_kernel\(\)", body)
        assert begin, kernel
        release = begin.start() if begin.group(1) == "begin_after" else body.index("let_next_kernel_in()")
        assert release >= begin.start() and body.count("let_next_kernel_in()") <= 1, kernel
        if "tmem_alloc(" in body:
            assert "__syncthreads()" in body[body.index("tmem_alloc("):release], kernel


@pytest.mark.parametrize("name", SOURCES + ["q8.cuh", "attn_items.cuh"])
def test_no_load_promises_that_nobody_writes_its_operands_meanwhile(name):
    """ld.global.nc and __ldg hold for data that stays as it is for the kernel's whole run, which here begins while the
    kernel in front may still be writing it; table_entry is the append's lookup that uses them."""
    text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())
    assert not re.search(r"__ldg|\.nc\b|table_entry\(", text), name
