"""What the built code of the kernels over 8-bit caches and shared positions has to
keep, read from the library: no matrix instruction's result over its own A or B
operands, counted waits where loads go to LDS, m0 for those loads alone."""

import re

import pytest

from test_cpu_serving_code import functions, overlaps  # noqa: F401 (a fixture)

KERNELS = {"CodesDecodeKernel": 12, "CodesSoloKernel": 20, "CodesWideKernel": 12, "12SharedKernel": 18,
           "CodesSharedKernel": 24, "SharedSmallKernel": 18}


@pytest.mark.parametrize("kernel", KERNELS)
def test_no_product_over_its_operands(functions, kernel):  # noqa: F811
    mine = {n: t for n, t in functions.items() if kernel in n}
    assert len(mine) == KERNELS[kernel], sorted(mine)
    for name, text in mine.items():
        seen, bad = overlaps(text)
        assert seen >= 8 and not bad, (name, bad)


def test_loads_to_lds_of_the_shared_kernels(functions):  # noqa: F811
    """Groups of one wave wait for K with as many loads outstanding as V has, and for V
    with as many as the next K."""
    mine = {n: t for n, t in functions.items() if "12SharedKernel" in n}
    solo = 0
    for name, text in mine.items():
        lines = [x.split("//")[0].strip() for x in text.splitlines()]
        uses = [x for x in lines if re.search(r"\bm0\b", x)]
        loads = [x for x in lines if re.match(r"buffer_load_dwordx4 .* lds$", x)]
        assert loads and len(uses) == len(loads) and all(re.match(r"s_mov_b32 m0, s\d+$", x) for x in uses), (name, uses[:5])
        if re.search(r"ELi\d+ELi4EEE", name):
            solo += 1
            waits = re.findall(r"s_waitcnt vmcnt\((\d+)\)\s", text)
            assert len(loads) % 4 == 0 and waits.count(str(len(loads) // 4)) >= 2, (name, len(loads))
    assert solo == 6


def test_few_registers_go_to_memory(functions):  # noqa: F811
    """The kernels of 16-bit rows keep their state in registers."""
    for name, text in functions.items():
        if re.search(r"Codes(Decode|Solo)Kernel", name) and "3F32" not in name:
            assert "scratch_" not in text, name
