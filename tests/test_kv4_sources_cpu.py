"""Rules of the 4-bit kernels' sources that no run can be trusted to break."""
import os
import re

import pytest

from conftest import ROOT

CSRC = os.path.join(ROOT, "msa-for-sail_b200", "csrc")


def code(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*|/\*.*?\*/", "", f.read(), flags=re.S)


def test_warps_wait_as_one_and_outlast_what_is_in_flight():
    text = code("fmha_kv4_tc.cu")
    assert "mbar_wait_warp(" in text and not re.search(r"\bmbar_wait\(", text)
    end = text.rsplit("if (*abort_flag) {", 1)[1]
    assert end.index("outlast_async_work();") < end.index("tmem_dealloc(")


def test_register_moves_are_checked_before_the_launch():
    """A setmaxnreg increase beyond what the launch allocated never completes."""
    text = code("fmha_kv4_tc.cu")
    launch = text.split("int launch(const MsaFmhaParams& p")[1]
    assert launch.index("fa.numRegs * NTHREADS < REGS_NEEDED") < launch.index("<<<")
    n = {k: int(v) for k, v in re.findall(r"(REGS_\w+) = (\d+)", text)}
    assert 128 * (n["REGS_SOFTMAX"] + n["REGS_MMA"] + 4 * n["REGS_CONVERT"]) <= 65536
    assert all(v % 8 == 0 and 24 <= v <= 256 for v in n.values())


@pytest.mark.parametrize("name", ["fmha_kv4.cu", "fmha_kv4_tc.cu"])
def test_kernels_read_coherently(name):
    assert not re.search(r"__restrict__|__ldg\b|\.nc\b", code(name))


@pytest.mark.parametrize("name", ["fmha_kv4.cu", "fmha_kv4_tc.cu"])
def test_every_stage_is_a_group_of_copies(name):
    """A warp waits for all but the newest groups of its copies: a list of fewer pages than stages has a group for each stage all the same,
    or its last pages would be read while they are on their way."""
    text = code(name)
    before = text.split("cp_async_wait<")[0]
    prologue = re.search(r"for \(int j = 0; j < (?:C::STAGES|RING); \+\+j\) \{(.*?)\n\s*\}", before, flags=re.S).group(1)
    assert re.search(r"^\s*cp_async_commit\(\);", prologue, flags=re.M)
    loop = text.split("cp_async_wait<", 1)[1]
    assert len(re.findall(r"^\s*cp_async_commit\(\);", loop, flags=re.M)) == 1 and "else cp_async_commit" not in loop
    fetch = re.search(r"auto fetch = (.*?)\n    \};|auto fetch = (.*?)\n  \};", text, flags=re.S).group(0)
    assert "cp_async_commit" not in fetch
