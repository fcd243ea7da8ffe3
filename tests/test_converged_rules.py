"""Instructions that a warp executes as one (cluster barriers, reads and writes of tensor memory, matrix instructions) come where its lanes
are together.  Behind a loop or a branch whose course differs between lanes, PTX leaves it open whether they are: a warp-wide barrier or
vote stands between.  Checked on the sources of the kernels with 4-bit weights, in the order of their lines: no run shows a warp that is
apart only sometimes."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rocmforge_b200", "csrc")
FILES = ("quantized.cu", "quantized_tc.cu")
AS_ONE = re.compile(r"barrier\.cluster\.\w+\.\w+\.aligned|\btcgen05_(?:ld|st)(?:16|32)\(|\btcgen05_wait_(?:ld|st)\(|\bmma_(?:s8|bf16)\(|\bquarter\(")
# what lets lanes part: a branch or a loop over something of the lane's own, a call that holds such a loop, a bounded wait
APART = re.compile(r"\bif \(.*\b(?:lane|t|there|tok|live|threadIdx\.x)\b|\bfor \(.*\b(?:lane|threadIdx\.x)\b|\bwrite_round\(\w|\bwait_for\(|\blet_land\(|\bthere && ")
TOGETHER = re.compile(r"__syncwarp\(\)|__syncthreads\(\)|__all_sync\(")


def found_apart(text):
    """The lines in which a warp acts as one while, as far as the order of the lines tells, its lanes may be apart; and the functions of that
    kind (called in loops) at whose end they may be."""
    apart = acts = False
    name, out = None, []
    for line in [*re.sub(r"//[^\n]*", "", text).split("\n"), "__device__ end("]:
        if re.search(r"__global__|__device__", line):
            if apart and acts and name is not None:
                out.append(f"the end of {name}")
            apart = acts = False
            name = None if "__global__" in line else re.findall(r"(\w+)\(", line)[-1]
            continue
        if AS_ONE.search(line):
            acts = True
            if apart:
                out.append(line.strip())
        if APART.search(line):
            apart = True
        if TOGETHER.search(line):
            apart = False
    return out


@pytest.mark.parametrize("name", FILES)
def test_a_warp_is_together_where_it_acts_as_one(name):
    text = open(os.path.join(CSRC, name)).read()
    assert found_apart(text) == []
    # in loops over the weights a lane's own arrival or copy is a predicate of the instruction, not a branch
    assert not re.search(r"if \(lane == 0\) at_arrive|if \(t < GROUPS\)", text)


def test_the_check_sees_lanes_apart():
    barrier = 'asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");\n'
    loop = "for (int i = threadIdx.x; i < n; i += 32)\n    x[i] = 0;\n"
    assert found_apart(loop + barrier) == [barrier.strip()]
    assert found_apart(loop + "__syncwarp();\n" + barrier) == []
    assert len(found_apart("if (lane == 0) at_arrive(bar);\ntcgen05_st32(to, out);\n")) == 1
    assert found_apart("at_arrive_if(bar, lane == 0);\ntcgen05_st32(to, out);\n") == []
    assert len(found_apart("write_round(round - 1);\nto_a[0] = a;\n" + barrier)) == 1
    assert found_apart("__device__ void f(int t) {\ntcgen05_wait_ld();\nif (there && x) y();\n}\n") == ["the end of f"]
