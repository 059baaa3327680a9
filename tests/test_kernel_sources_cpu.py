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


@pytest.mark.parametrize("name", ["gemm_nvfp4.cuh", "gemm_wgrad_mx.cuh"])
def test_a_warp_that_elects_a_lane_agrees_on_its_waits(name):
    # lanes for which a wait has run out must not leave a loop in which the others still elect a lane among all 32
    text = source(name)
    assert "elect_one()" in text
    bare = list(re.finditer(r"bounded_wait(_quiet)?\((.*?), p\.wait_limit\);", text, re.S))
    assert len(bare) == len(re.findall(r"bounded_wait(?:_quiet)?\(", text))
    for m in bare:
        if re.search(r"ST_\w+_(EPILOGUE|WORKER)$", m.group(2)):  # these roles elect nobody; they agree behind the wait
            assert "ok = __all_sync(0xFFFFFFFFu, ok);" in text[m.end():m.end() + 700], m.group()
        else:
            assert "raw_empty_bar" in m.group(2) and "lane == 0)" in text[m.start() - 900:m.start()], m.group()  # a loop of one lane
    for form in ("bounded_wait_warp", "bounded_wait_quiet_warp"):  # which answer by votes alone
        body = source("gemm_tile_loop.cuh").split(f"bool {form}(")[1].split("}")[0].split("return ")[1]
        assert all(term.strip().startswith("__all_sync(0xFFFFFFFFu, ") for term in body.split("||"))


@pytest.mark.parametrize("name,wait", [("gemm_nvfp4.cuh", "bounded_wait_warp"), ("gemm_wgrad_mx.cuh", "bounded_wait_quiet_warp")])
def test_no_signal_reaches_a_cta_of_the_pair_after_it_has_left(name, wait):
    text = source(name)
    # from the even CTA: a stage of the ring is handed back only to be filled again, or the loading warp waits once more for
    # every stage behind its last load
    if name == "gemm_nvfp4.cuh":
        assert re.search(r"if \(left > STAGES\) {\s*ptx::umma_commit_pair\(&empty_bar\[stage\], 0x3\);", text)
        assert text.count("umma_commit_pair(&empty_bar") == 1 and text.count("--left;") == 1
    else:
        assert re.search(r"for \(int i = 0; ok && i < kWgStages; \+\+i\) {\s*ok = " + wait + r"\(&empty_bar\[stage\], phase \^ 1u", text)
    # to it: its product warp waits once more for every accumulator to be handed back
    issue = text.index("umma_commit_pair(")
    waits = [m.start() for m in re.finditer(wait + r"\(&?acc_empty_bar", text)]
    assert len(waits) == 2 and waits[0] < issue < waits[1]


@pytest.mark.parametrize("name", ["row_elements.cuh", "nvfp4_quantize.cuh", "gemm_nvfp4.cuh", "gemm_wgrad_mx.cuh", "mx_quantize.cuh"])
def test_launches_that_may_start_early_use_no_read_only_loads(name):
    # such a launch runs while the one before it still writes what it is going to read
    text = source(name)
    if name == "mx_quantize.cuh":  # its other kernels wait for the launch before them as a whole
        kernels = [t for t in re.split(r"template <", text) if "grid_dependency_wait()" in t]
        assert len(kernels) == 1
        text = kernels[0]
    assert not re.search(r"\.nc\b|__ldg\(|__restrict__", text)


def test_no_signal_reaches_a_cta_of_the_tile_loops_pair_after_it_has_left():
    # both sides wait once more, behind their last load and their last product, for what the other still signals
    text = source("gemm_tile_loop_2cta.cuh")
    for last, bar, rounds in (("tma_load_2d_pair(", "empty_bar[stage], phase", "STAGES"),
                              ("umma_commit_pair(&acc_full_bar", "acc_empty_bar[acc], acc_phase", "kNumAcc")):
        behind = text[text.rindex(last):]
        assert re.search(r"for \(int i = 0; ok && i < " + rounds + r"; \+\+i\) {\s*ok = bounded_wait\(&" + re.escape(bar) + r" \^ 1u", behind)
