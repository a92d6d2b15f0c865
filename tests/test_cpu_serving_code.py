"""What the serving kernels' built code has to keep, read from the library: no
matrix instruction's result over its own A or B operands (wrong sums on gfx950),
and as many LDS loads in flight as the counted waits of the one-wave groups say."""

import os
import re
import shutil
import subprocess

import pytest

import rpgbarengine_amd as eng

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
KERNELS = ["PromptKernel", "DecodeKernel"]


@pytest.fixture(scope="module")
def functions(tmp_path_factory):
    if not os.path.exists(OBJDUMP):
        pytest.skip("no llvm-objdump")
    d = tmp_path_factory.mktemp("code")
    lib = shutil.copy(eng.LIB_PATH, str(d))
    subprocess.run([OBJDUMP, "--offloading", lib], check=True, capture_output=True)
    found = {}
    for f in sorted(os.listdir(d)):
        if "gfx950" not in f:
            continue
        with open(os.path.join(d, f), "rb") as h:
            if b"5paged" not in h.read():
                continue
        text = subprocess.run([OBJDUMP, "-d", os.path.join(d, f)], check=True, capture_output=True, text=True).stdout
        for part in re.split(r"\n(?=[0-9a-f]+ <)", text):
            m = re.match(r"[0-9a-f]+ <(\S+)>:", part)
            if m and "5paged" in m.group(1):
                found[m.group(1)] = part
    return found


def registers(word):
    m = re.fullmatch(r"([va])\[(\d+):(\d+)\]", word) or re.fullmatch(r"([va])(\d+)()", word)
    if m is None:
        return set()
    lo = int(m.group(2))
    return {(m.group(1), i) for i in range(lo, int(m.group(3) or lo) + 1)}


def overlaps(text):
    seen, bad = 0, []
    for line in text.splitlines():
        m = re.match(r"\s+v_mfma\S+ (\S+), (\S+), (\S+), \S+", line)
        if m:
            seen += 1
            d, a, b = (registers(x) for x in m.groups())
            if d & (a | b):
                bad.append(line.strip())
    return seen, bad


@pytest.mark.parametrize("kernel", KERNELS)
def test_no_product_over_its_operands(functions, kernel):
    mine = {n: t for n, t in functions.items() if kernel in n and "Join" not in n}
    assert len(mine) >= 6
    for name, text in mine.items():
        seen, bad = overlaps(text)
        assert seen >= 8 and not bad, (name, bad)


def test_the_check_sees_an_overlap():
    ok = "\tv_mfma_f32_32x32x16_bf16 v[0:15], v[16:19], v[20:23], v[0:15]\n"
    bad = "\tv_mfma_f32_32x32x16_bf16 v[16:31], v[16:19], v[20:23], 0\n"
    assert overlaps(ok) == (1, [])
    assert overlaps(ok + bad)[0] == 2 and len(overlaps(ok + bad)[1]) == 1


def test_counted_waits_of_one_wave_groups(functions):
    """A wave waits for K with as many loads outstanding as V has, and for V with
    as many as the next K: every tile's loads number what the waits count (others
    in between would only make them wait longer)."""
    solo = {n: t for n, t in functions.items() if re.search(r"PromptKernelI\S+ELi\d+ELi[48]ELb0E", n)}
    assert len(solo) == 10
    shared = [t for n, t in functions.items() if re.search(r"PromptKernelI\S+ELi\d+ELi4ELb1E", n)]
    assert len(shared) == 1  # K and V in one place: nothing else in flight, waits for all
    loop = re.findall(r"buffer_load_dwordx4 [^\n]* lds|s_waitcnt vmcnt\(0\)", shared[0])
    assert len(loop) > 20 and not re.search(r"lds(?:(?!s_waitcnt vmcnt\(0\)).)*ds_read_b128", shared[0], re.S)
    for name, text in solo.items():
        dma = len(re.findall(r"buffer_load_dwordx4 [^\n]* lds", text))
        # K and V before the loop and in it
        waits = re.findall(r"s_waitcnt vmcnt\((\d+)\)\s", text)
        assert dma % 4 == 0 and waits.count(str(dma // 4)) >= 2, (name, dma, waits)
        assert "scratch_" not in text, name
