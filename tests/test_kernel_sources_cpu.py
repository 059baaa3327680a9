"""Rules of synchronisation that no run can show to be broken: they are read off the kernels' sources."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pto_isa_mirror_b200", "csrc")


def source(name):
    """A source without its comments."""
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


@pytest.mark.parametrize("name,reads", [
    ("nvfp4_quantize.cuh", r"ptx::ld_shared_cluster_f32x4\("),
    ("gemm_nvfp4.cuh", r"ptx::ld_shared_cluster_f32x4\("),
    ("gemm_nvfp4.cuh", r"nv_add_parts<[^>]*, OUT>"),  # calls of the function with the reads
    ("gemm_wgrad_mx.cuh", r"ptx::ld_shared_cluster_f32x4\("),
    ("gemm_wgrad_mx.cuh", r"wg_add_parts<\d"),
])
def test_reads_of_another_ctas_shared_memory_are_ordered_before_it_may_leave(name, reads):
    # the arrival behind such reads tells that CTA that it may go: a relaxed one orders nothing
    text = source(name)
    found = [m.end() for m in re.finditer(reads, text)]
    assert found
    for at in found:
        end = text.find("__global__", at)
        arrival = re.compile(r"ptx::cluster_arrive\w*\(\)").search(text, at, end if end > 0 else len(text))
        if "add_parts" not in reads:  # which arrives itself
            assert arrival, text[at - 200:at]
        assert arrival is None or arrival.group() == "ptx::cluster_arrive()", text[at - 200:at]
