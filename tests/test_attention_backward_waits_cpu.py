"""Wait states of the attention gradients' own MFMAs, read from the machine code built here.

S and dP of the larger units are MFMAs in inline assembly, whose results the compiler takes for ready at
once.  Along the program text (in which every loop body stands once) this holds for every MFMA that writes
vector registers:
  * 12 wait states before anything but an MFMA's accumulation touches the result (what the compiler itself
    leaves after an MFMA of 8 passes; an instruction is one, s_nop n is n + 1);
  * 2 between a vector operation that writes an operand and the MFMA;
  * no write to an MFMA's separate c operand before another MFMA has been issued, or 8 wait states.
"""
import re
import subprocess

import pytest

from neptune_codegen import attention_backward as AB, hip

REG = re.compile(r"\b([va])(?:\[(\d+):(\d+)\]|(\d+))(?![\w\]])")
RESULT, OPERAND, READ = 12, 2, 8


def registers(text):
    out = set()
    for kind, first, last, one in REG.findall(text):
        lo, hi = (int(first), int(last)) if first else (int(one), int(one))
        out |= {(kind, i) for i in range(lo, hi + 1)}
    return out


def instructions(listing):
    for line in listing.splitlines():
        if line.startswith("\t"):
            text = line.split("//")[0].strip()
            op, _, rest = text.partition(" ")
            yield op, text, [a.strip() for a in re.split(r",(?![^\[]*\])", rest)]
        elif line.strip().endswith(">:"):
            yield "start", "", []


def violations(listing):
    bad, recent = [], []                             # recent: wait states since, what, registers, text
    for op, text, args in instructions(listing):
        if op == "start":
            recent = []
            continue
        states = int(args[0], 0) + 1 if op == "s_nop" else 1
        mfma = op.startswith("v_mfma")
        if mfma:
            result, sources, c = registers(args[0]), registers(args[1]) | registers(args[2]), registers(args[3])
            touched = set()
        else:
            touched = set() if op.startswith("s_") else registers(text)
        for age, what, regs, of in recent:
            if (what == "result" and age < RESULT and regs & (sources if mfma else touched)
                    or what == "written" and mfma and age < OPERAND and regs & (sources | c)
                    or what == "read" and not mfma and age < READ and regs & touched):
                bad.append(f"{age} after {of}: {text}")
        issued = mfma and any(what != "written" for _, what, _, _ in recent)
        recent = [(age + (READ if issued and what == "read" else states), what, regs, of)
                  for age, what, regs, of in recent if age < 20]
        if mfma:
            if any(kind == "v" for kind, _ in result):
                recent.append((0, "result", result, text))
            if c and c != result:
                recent.append((0, "read", c, text))
        elif op.startswith("v_") and not op.startswith("v_cmp"):
            recent.append((0, "written", registers(args[0]), text))
    return bad


def listing(program, tmp_path):
    path = tmp_path / "unit.co"
    program.precompile()
    path.write_bytes(hip._cache_file(program.source, program.options).read_bytes())
    return subprocess.run(["/opt/rocm/llvm/bin/llvm-objdump", "-d", str(path)], check=True, capture_output=True,
                          text=True).stdout


UNITS = [(stage, dim, blocks, parts) for dim in (64, 128, 256) for stage, blocks, parts in AB.unit_kinds(dim)
         if stage != "rows"]


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("stage,dim,blocks,parts", UNITS)
def test_results_are_waited_for(stage, dim, blocks, parts, dtype, tmp_path):
    for causal in (True, False):
        text = listing(AB._program(stage, dim, causal, dtype, blocks, parts), tmp_path)
        assert text.count("v_mfma_f32_32x32x16") >= 8
        assert violations(text) == []


MFMA = "\tv_mfma_f32_32x32x16_bf16 v[0:15], v[32:35], v[36:39], {c}\n"


@pytest.mark.parametrize("text,found", [
    (MFMA.format(c="v[0:15]") + "\tv_exp_f32_e32 v40, v3\n", 1),
    (MFMA.format(c="v[0:15]") + "\ts_nop 10\n\tv_exp_f32_e32 v40, v3\n", 1),
    (MFMA.format(c="v[0:15]") + "\ts_nop 11\n\tv_exp_f32_e32 v40, v3\n", 0),
    (MFMA.format(c="v[0:15]") + MFMA.format(c="v[0:15]"), 0),
    ("\tv_mov_b32_e32 v33, v50\n" + MFMA.format(c="v[0:15]"), 1),
    ("\tv_mov_b32_e32 v33, v50\n\ts_nop 1\n" + MFMA.format(c="v[0:15]"), 0),
    (MFMA.format(c="v[16:31]") + "\tds_read_b128 v[16:19], v60\n", 1),
    (MFMA.format(c="v[16:31]") + MFMA.format(c="v[0:15]") + "\tds_read_b128 v[16:19], v60\n", 0),
])
def test_the_reader_finds_what_it_looks_for(text, found):
    assert len(violations(text)) == found
