"""What of the attention kernels' state the built code keeps in memory: nothing for
16-bit rows but two registers of the 128-row tiles over codes, and in f32 what the
tiles of 128 rows of 128 have too much for two workgroups to a compute unit."""

import re

import pytest

from test_cpu_serving_code import functions  # noqa: F401 (a fixture)

NAMES = {"Codes(Decode|Solo|SharedSmall)Kernel": 44, "CodesWideKernel": 12, "17CodesSharedKernel": 24, "12SharedKernel": 18,
         "17SharedSmallKernel": 6}


def bytes_a_lane(text):
    """The furthest that a scratch access reaches."""
    ends = [0]
    for line in text.splitlines():
        m = re.match(r"\s+scratch_(?:load|store)_(\w+) (.*?)\s*(?://.*)?$", line)
        if m:
            size = {"dword": 4, "dwordx2": 8, "dwordx3": 12, "dwordx4": 16}[m.group(1)]
            off = re.search(r"offset:(\d+)", m.group(2))
            ends.append(size + (int(off.group(1)) if off else 0))
    return max(ends)


@pytest.mark.parametrize("kernels", NAMES)
def test_state_stays_in_registers(functions, kernels):  # noqa: F811
    mine = {n: t for n, t in functions.items() if re.search(kernels, n)}
    got = {n: bytes_a_lane(t) for n, t in mine.items()}
    assert len(mine) == NAMES[kernels], sorted(mine)
    for name, n in got.items():
        most = 0
        if re.search("CodesWide.*ELi128E|CodesShared.*ELi128ELb1E|12SharedKernel.*ELi128ELi1E", name):
            most = 256 if "3F32" in name else 8 if "CodesShared" in name else 0
        assert n <= most, (name, n)
