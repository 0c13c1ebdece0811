"""Lanes of a wavefront that hand each other LDS words in the embedding's order meet in between, read from the
kernel's source: the compiler may otherwise move an access across another lane's that it takes for another address."""
import pathlib
import re

import neptune_codegen

TEXT = (pathlib.Path(neptune_codegen.__file__).parent.parent / "csrc/kernels/nep_embedding.h").read_text()
MEET = "lanes_meet();"


def body(text, start):
    """The block in braces behind `start`, without comments, as its statements' lines."""
    at = text.index("{", text.index(start) + len(start) - 1)
    depth = 0
    for end in range(at, len(text)):
        depth += {"{": 1, "}": -1}.get(text[end], 0)
        if depth == 0:
            break
    lines = (re.sub(r"//.*", "", line).strip() for line in text[at + 1:end].splitlines())
    return [line for line in lines if line]


ORDER = "\n".join(body(TEXT, "void embedding_order("))


def test_lanes_meet_in_front_of_the_lists_reads_and_behind_them():
    for name in ("tally", "empty"):
        lines = body(ORDER, f"auto {name} = [&]() {{")
        reads = [i for i, line in enumerate(lines) if "list[wave][l" in line]
        meets = [i for i, line in enumerate(lines) if line == MEET]
        assert reads and meets and meets[0] < min(reads) and max(reads) < meets[-1], name


def test_a_counter_is_written_before_another_batch_reads_it():
    lines = body(ORDER, "auto empty = [&]() {")
    assert lines.index(MEET, lines.index("if (before == 0) *counter = place + __builtin_popcountll(same);")) \
        < len(lines) - 1                             # (inside the loop over the batches)


def test_counters_are_zero_before_they_count():
    lines = ORDER.splitlines()
    zero = next(i for i, line in enumerate(lines) if "counters[wave][k] = 0" in line)
    assert lines[zero + 1] == MEET


def test_meeting_orders_the_memory_and_the_lanes():
    assert body(TEXT, "void lanes_meet() {") == [
        '__builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");', "__builtin_amdgcn_wave_barrier();"]
