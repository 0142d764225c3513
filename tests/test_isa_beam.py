"""CPU check of the choice's first launch in its compiled gfx950 assembly: a wave's
list, which its lanes wrote each for itself, is read by other lanes behind a point that
orders the wave's accesses to LDS."""
import re

import pytest

from test_isa_arrival import kernel_asm
from test_isa_paged import asm_of  # noqa: F401  (a fixture)

COUNTED = re.compile(r"^\s*ds_add_rtn_u32\s")   # the list's place among the block's
LIST_READ = re.compile(r"^\s*ds_read\w*_b64\s")
ORDERED = re.compile(r"^\s*; wave barrier")


def joint_list_problems(asm: str):
    """Faults of the step that puts a wave's list with those of the block."""
    lines = asm.split("\n")
    counted = [i for i, l in enumerate(lines) if COUNTED.match(l)]
    if len(counted) != 1:
        return [f"{len(counted)} counts of lists"]
    reads = [i for i in range(counted[0], len(lines)) if LIST_READ.match(lines[i])]
    if not reads:
        return ["no list is read"]
    if not any(ORDERED.match(l) for l in lines[counted[0]:reads[0]]):
        return ["the list is read with nothing that orders it behind the writes of other lanes"]
    return []


def test_detector():
    good = "\tds_add_rtn_u32 v3, v3, v4\n\t; wave barrier\n\tds_read_b64 v[2:3], v26\n"
    assert joint_list_problems(good) == []
    for bad in (good.replace("\t; wave barrier\n", ""), good.replace("\tds_read_b64 v[2:3], v26\n", ""),
                "\t; wave barrier\n" + good.replace("\t; wave barrier\n", ""), good + good, ""):
        assert joint_list_problems(bad)


@pytest.mark.parametrize("groups", [4, 8])
def test_a_waves_list_is_ordered(asm_of, groups):  # noqa: F811
    problems = joint_list_problems(kernel_asm(asm_of("neon_beam"), f"k_beam_partILi{groups}E"))
    assert problems == []
