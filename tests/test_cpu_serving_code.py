"""What the serving kernels' built code has to keep, read from the library: no
matrix instruction's result over its own A or B operands (wrong sums on gfx950),
and as many LDS loads in flight as the counted waits of the one-wave groups say.
And what their inline assembly has to name: the registers that it overwrites."""

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


def statements(text):
    """(assembly, clobbers) of every asm statement of a source file."""
    text = re.sub(r"//[^\n]*", "", text)
    for m in re.finditer(r"\basm volatile\s*\(", text):
        at, depth = m.end(), 1
        while depth:
            depth += {"(": 1, ")": -1}.get(text[at], 0)
            at += 1
        body = text[m.end():at - 1]
        code = re.match(r'\s*((?:"(?:[^"\\]|\\.)*"\s*)+)', body)
        fields = re.split(r":", re.sub(r'"(?:[^"\\]|\\.)*"', lambda q: q.group(0).replace(":", ";"), body[code.end():]))
        yield "".join(re.findall(r'"((?:[^"\\]|\\.)*)"', code.group(1))), fields[3] if len(fields) > 3 else ""


def unnamed(text):
    """The fixed registers that asm statements write and do not name as clobbered."""
    bad = []
    for code, clobbers in statements(text):
        for line in code.split(r"\n\t"):
            m = re.match(r"\s*[sv]_\w+\s+(m0|vcc\w*|exec\w*|[sv]\d+|[sv]\[\d+:\d+\])\s*,", line)
            if m and f'"{m.group(1)}"' not in clobbers:
                bad.append((m.group(1), code))
    return bad


def test_assembly_names_the_registers_it_overwrites():
    src = os.path.join(os.path.dirname(eng.LIB_PATH), "csrc")
    seen = 0
    for f in sorted(os.listdir(src)):
        with open(os.path.join(src, f), encoding="utf-8") as h:
            text = h.read()
        seen += len(list(statements(text)))
        assert not unnamed(text), (f, unnamed(text))
    assert seen >= 20


def test_the_check_sees_an_unnamed_register():
    line = 'asm volatile("s_mov_b32 m0, %0\\n\\tbuffer_load_dwordx4 %1, %2, %3 offen lds" : : "s"(f(a)), "v"(b), "s"(c), "s"(d)'
    assert [r for r, _ in unnamed(line + ");")] == ["m0"]
    assert unnamed(line + ' : "m0");') == [] and unnamed(line + ' : "m0", "memory");') == []


def test_m0_serves_the_loads_to_lds_alone(functions):
    """Nothing else in the prompt kernels sets or reads it."""
    for name, text in functions.items():
        if "PromptKernel" not in name:
            continue
        lines = [x.split("//")[0].strip() for x in text.splitlines()]
        uses = [x for x in lines if re.search(r"\bm0\b", x)]
        loads = [x for x in lines if re.match(r"buffer_load_dwordx4 .* lds$", x)]
        assert loads and len(uses) == len(loads) and all(re.match(r"s_mov_b32 m0, s\d+$", x) for x in uses), (name, uses[:5])
