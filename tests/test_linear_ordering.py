"""CPU tests of the linear kernels' hand-overs between blocks, read from their
source: a missing release does not show on today's hardware, so no run can."""
import os
import re

from quant_2bit_b200.build import CSRC


def _source(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def test_relaxed_arrivals_in_other_blocks_announce_no_data():
    """A relaxed arrival in another block orders nothing that its thread has
    written or seen before it.  What it may announce is that accumulators have
    been read (their loads have returned); operands in shared memory, zeroed or
    loaded, need a release, or loads that complete on that barrier themselves."""
    barriers = re.findall(r"bar_arrive_relaxed_in\(smem_u32\(&ctl\.(\w+)", _source("bcjr_mm.cuh"))
    assert set(barriers) <= {"tempty"}, barriers


def test_every_wait_has_its_limit_from_its_own_start():
    """Waits are bounded in one place, by the time since the wait began and the
    work waited for.  One bounded by the time since the kernel began would give
    up in a healthy launch that runs longer."""
    source = _source("bcjr_mm.cuh")
    uses = [line.strip() for line in source.splitlines() if "kWaitLimitClocks" in line]
    assert uses[0].startswith("constexpr long long kWaitLimitClocks")
    for line in uses[1:]:
        assert "clock64() - t0 > kWaitLimitClocks + 4096ll * stages" in line or "bar_wait" in line, line
    body = source[source.index("bool bar_wait"):]
    assert body.index("t0 = clock64()") < body.index("while (true)")
    assert "clock64" not in source[source.index("mm_kernel("):]
