"""Wait states of the attention gradients' own MFMAs along every path of the machine code built here: over
branches, joins and the loops' back edges, where test_attention_backward_waits_cpu.py follows the text.  Its
rules hold on each path; a branch counts as one wait state, taken or not.
"""
import re

import pytest

from neptune_codegen import attention_backward as AB
from test_attention_backward_waits_cpu import OPERAND, READ, RESULT, UNITS, listing, registers

FORGET = max(RESULT, OPERAND, READ)


def program(listing):
    """Per instruction (op, text, arguments, wait states), and the instructions that may follow it."""
    code, at, jumps = [], {}, {}
    start = None
    for line in listing.splitlines():
        name = re.match(r"([0-9a-f]+) <(.+)>:", line)
        if name:
            start = int(name.group(1), 16)
            code.append(("start", "", [], 0))
        elif line.startswith("\t"):
            text, _, place = line.partition("//")
            text = text.strip()
            op, _, rest = text.partition(" ")
            args = [a.strip() for a in re.split(r",(?![^\[]*\])", rest)]
            at[int(re.match(r"\s*([0-9A-F]+)", place).group(1), 16)] = len(code)
            target = re.search(r"<[^>+]+(?:\+0x([0-9a-f]+))?>", place)
            if op.startswith(("s_cbranch", "s_branch")):
                jumps[len(code)] = start + int(target.group(1) or "0", 16)
            elif op.startswith(("s_setpc", "s_swappc", "s_call", "s_getpc")):
                raise AssertionError(f"a path that is not in the text: {text}")
            code.append((op, text, args, int(args[0], 0) + 1 if op == "s_nop" else 1))
    after = [[] for _ in code]
    for i, (op, *_) in enumerate(code):
        if i in jumps:
            after[i].append(at[jumps[i]])
        if i + 1 < len(code) and op not in ("s_branch", "s_endpgm") and code[i + 1][0] != "start":
            after[i].append(i + 1)
    return code, after


def violations(listing):
    code, after = program(listing)
    effects = []                                     # touched, MFMA sources, c, what it leaves behind
    for op, text, args, states in code:
        if op.startswith("v_mfma"):
            result, sources, c = registers(args[0]), registers(args[1]) | registers(args[2]), registers(args[3])
            left = [("result", result)] if any(kind == "v" for kind, _ in result) else []
            effects.append((set(), sources, c, left + ([("read", c)] if c and c != result else [])))
        else:
            left = ([("written", registers(args[0]))] if op.startswith("v_") and not op.startswith("v_cmp") else [])
            effects.append((set() if op.startswith("s_") else registers(text), set(), set(), left))
    # per instruction: {(instruction, kind of event): the fewest wait states since} on some path to it
    before, todo, bad = [{} for _ in code], list(range(len(code))), {}
    while todo:
        i = todo.pop()
        op, text, args, states = code[i]
        mfma, (touched, sources, c, left) = op.startswith("v_mfma"), effects[i]
        for (j, n), age in before[i].items():
            what, regs = effects[j][3][n]
            if (what == "result" and age < RESULT and regs & (sources if mfma else touched)
                    or what == "written" and mfma and age < OPERAND and regs & (sources | c)
                    or what == "read" and not mfma and age < READ and regs & touched):
                bad[i, j] = f"{age} after {code[j][1]}: {text}"
        # an MFMA that has been issued has read its c once the next one is issued
        out = {}
        for (j, n), age in before[i].items():
            age += READ if mfma and effects[j][3][n][0] == "read" else states
            if age < FORGET:
                out[j, n] = age
        out.update({(i, n): 0 for n in range(len(left))})
        for k in after[i]:
            new = {e: age for e, age in out.items() if age < before[k].get(e, FORGET)}
            if new:
                before[k].update(new)
                todo.append(k)
    return list(bad.values())


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("stage,dim,blocks,parts", UNITS)
def test_results_are_waited_for_on_every_path(stage, dim, blocks, parts, dtype, tmp_path):
    for causal in (True, False):
        text = listing(AB._program(stage, dim, causal, dtype, blocks, parts), tmp_path)
        code, after = program(text)
        assert sum(op.startswith("v_mfma_f32_32x32x16") for op, *_ in code) >= 8
        assert any(k <= i for i, ks in enumerate(after) for k in ks), "no loop was found"
        assert violations(text) == []


def lines(*texts):
    """A listing of instructions 4 bytes apart; "-> n" is a jump to the n-th."""
    out = ["0000000000001000 <kernel>:"]
    for i, text in enumerate(texts):
        text, _, to = text.partition("->")
        out.append(f"\t{text.strip()}  // {0x1000 + 4 * i:012X}: 00000000"
                   + (f" <kernel+{4 * int(to):#x}>" if to else ""))
    return "\n".join(out)


MFMA = "v_mfma_f32_32x32x16_bf16 v[0:15], v[32:35], v[36:39], v[0:15]"


@pytest.mark.parametrize("texts,found", [
    ((MFMA, "v_exp_f32_e32 v40, v3"), 1),
    ((MFMA, "s_nop 11", "v_exp_f32_e32 v40, v3"), 0),
    # over a back edge: the loop's last MFMA and its first instruction
    (("v_exp_f32_e32 v40, v3", MFMA, "s_cbranch_scc1 65533 -> 0", "s_endpgm"), 1),
    (("v_exp_f32_e32 v40, v3", MFMA, "s_nop 10", "s_cbranch_scc1 65532 -> 0", "s_endpgm"), 0),
    # around a wait that stands in a branch
    ((MFMA, "s_cbranch_execz 1 -> 3", "s_nop 11", "v_exp_f32_e32 v40, v3"), 1),
    ((MFMA, "s_branch 1 -> 3", "v_exp_f32_e32 v40, v3", "s_nop 11", "v_exp_f32_e32 v41, v4"), 0),
    (("v_mov_b32_e32 v33, v50", "s_branch 0 -> 2", MFMA), 1),
    (("ds_read_b128 v[16:19], v60", MFMA[:-7] + "v[16:31]", "s_cbranch_scc1 65533 -> 0"), 1),
    (("ds_read_b128 v[16:19], v60", MFMA[:-7] + "v[16:31]", MFMA, "s_cbranch_scc1 65532 -> 0"), 0),
])
def test_the_reader_finds_what_it_looks_for(texts, found):
    assert len(violations(lines(*texts))) == found
