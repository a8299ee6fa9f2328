"""Memory order of the launch for few tokens, on the kernel's text (CPU)."""

import re
from pathlib import Path

TEXT = re.sub(r"//[^\n]*", "", (Path(__file__).resolve().parents[1] / "dist_moe_b200" / "csrc" / "few_tokens.cu").read_text())


def test_lanes_that_read_other_blocks_parts_come_after_the_one_that_acquired_them():
    """One lane counts the block's arrival and acquires what the blocks before it released; a shuffle hands its result on, but orders
    no memory.  Between it and the other lanes' reads of the parts the warp has to meet."""
    arrive = TEXT.index("atom_add_acq_rel(arrived")
    handed_on = TEXT.index("__shfl_sync", arrive)
    read = TEXT.index("__ldcg", handed_on)
    assert "__syncwarp()" in TEXT[handed_on:read]


def test_what_a_warp_stored_comes_before_its_arrival():
    stored, arrive = TEXT.index("__stcg"), TEXT.index("atom_add_acq_rel(arrived")
    assert stored < arrive and "__syncwarp()" in TEXT[stored:arrive]


def test_every_lane_that_copies_rows_of_h_has_acquired_them_itself():
    """The warp that copies rows waits for the other blocks with all of its lanes: no lane-0 branch stands around that wait."""
    wait = TEXT.index("ld_acquire_gpu(p.meeting)")
    around = TEXT[TEXT.rindex("few_load_rows<false>", 0, wait):wait]
    assert "lane == 0" not in around
