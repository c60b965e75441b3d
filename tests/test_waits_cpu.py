"""Waits on mbarriers by whole warps, in the sources.

Lanes of a warp that part at a wait (some give up, others see the barrier complete) would meet again at an instruction that needs all of them, and
might never.  Only a launch that hangs could show that, so it is read: what a warp's lanes all execute ends in a vote."""

from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "qwen3_runtime_b200" / "csrc"
VOTED = "__all_sync(0xffffffffu, mbar_"


def waits(name):
    """Lines of a source that wait on a barrier and may give up."""
    return [line.strip() for line in (CSRC / name).read_text().splitlines()
            if any(call in line.split("//")[0] for call in ("mbar_wait(", "mbar_try_wait(", "mbar_wait_warp("))]


def test_the_warp_s_wait_votes_on_both_ways_out():
    source = (CSRC / "async_tiles.cuh").read_text()
    body = source[source.index("bool mbar_wait_warp_on("):source.index("// the same for a barrier on which other blocks")]
    assert body.count("return") == 3 and VOTED + "wait(" in body and VOTED + "try_wait(" in body


@pytest.mark.parametrize("name", ["prompts_tiles.cuh", "attention_prefill_tc.cu"])
def test_every_wait_is_a_warp_s(name):
    found = waits(name)
    assert found and all(VOTED in line or "mbar_wait_warp(" in line for line in found), [
        line for line in found if VOTED not in line and "mbar_wait_warp(" not in line]


def test_the_products_epilogues_wait_as_warps():
    """(The other waits of this source are single threads'.)"""
    found = [line for line in waits("gemm_tcgen05.cu") if "(acc_full" in line]
    assert len(found) == 3 and all("mbar_wait_warp(" in line for line in found), found
