"""The loss kernels' source against the numbers that its barrier model (test_loss_protocol_cpu.py) and its
register split rest on: stages, score buffers, arrivals per barrier, and who arrives."""
import inspect
import os
import re

import test_loss_protocol_cpu as model

SOURCE = open(os.path.join(os.path.dirname(__file__), "..", "rust_ppocrv6_b200", "csrc", "loss_kernels.cu")).read()


def number(name):
    return int(re.search(rf"\b{name} = (\d+)", SOURCE)[1])


def by_type(name):
    """(f32, bf16) values of one of Ring's constants."""
    return tuple(int(i) for i in re.search(rf"{name} = F32 \? (\d+)u : (\d+)u", SOURCE).groups())


def arrivals(barrier):
    return re.search(rf"mbar_init\(bar\({barrier}[^)]*\), ([^)]+)\)", SOURCE)[1]


def test_the_models_stages_and_buffers_are_the_kernels():
    m = re.search(r"stages, bufs = \((\d), (\d)\) if f32 else \((\d), (\d)\)", inspect.getsource(model.simulate))
    assert (int(m[1]), int(m[3])) == by_type("kStages") and (int(m[2]), int(m[4])) == by_type("kBufs")


def test_every_barrier_counts_those_who_arrive():
    assert number("kMainThreads") == 32 * (4 + 16 + 8)  # control, four softmax and two adding warpgroups
    assert arrivals("kLBarFull") == "1"                 # the producer, with the copies' bytes
    assert arrivals("kLBarEmpty") == str(1 + 8)         # the product's commit, a pair of warpgroups
    assert arrivals("kLBarAFull") == f"F32 ? {16 * 32} : 1"
    for one in ("kLBarAEmpty", "kLBarSFull", "kLBarSFree", "kLBarOFull", "kLBarDone"):  # commits
        assert arrivals(one) == "1", one
    assert arrivals("kLBarPFull") == "4"                # the warps of a half
    assert arrivals("kLBarOEmpty") == "8"               # the adding warps
    assert arrivals("kLBarRing") == "4"                 # the first half's warps
    assert arrivals("kLBarTop") == "2"                  # a quadrant's two halves
    assert arrivals("kLBarMsFull") == str(16 * 32) and arrivals("kLBarMsEmpty") == "128"


def test_the_register_split_is_covered_at_launch_and_checked_for_every_variant():
    ctrl, soft, add, launch = (number(i) for i in ("kCtrlRegs", "kSoftRegs", "kAddRegs", "kLaunchRegs"))
    assert 128 * ctrl + 512 * soft + 256 * add <= number("kMainThreads") * launch <= 65_536 and soft == launch
    setup = SOURCE[SOURCE.index("cudaError_t loss_kernel_setup"):]
    setup = setup[:setup.index("\n}")]
    listed = {tuple(i.split(", ")) for i in re.findall(r"loss_main_kernel<([^>]+)>", setup)}
    start = SOURCE.index("cudaError_t launch_loss_main")
    used = {tuple(i.split(", ")) for i in re.findall(r"loss_main_kernel<([^>]+)>", SOURCE[start:SOURCE.index("\n}", start)])}
    assert used == listed and len(used) == 10 and "split_fits(a.numRegs)" in setup
