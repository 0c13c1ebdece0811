"""LDS accesses of the residual norm's gradients, read from the machine code built here: none may reach past
its unit's allocation (a constant offset is the least that an access adds to its address)."""
import re
import subprocess

import pytest
import torch

from neptune_codegen import hip, residual_norm as RN
from neptune_codegen.emitters import residual_norm_kernel_name

WIDTH = re.compile(r"_[bu](\d+)")
LLVM = "/opt/rocm/llvm/bin/"


def reach(listing):
    """The furthest byte that a DS instruction's own offsets reach."""
    most = 0
    for line in listing.splitlines():
        text = line.split("//")[0].strip()
        op = text.split(" ")[0]
        if not re.match(r"ds_(read|write)", op):
            continue
        width = int(WIDTH.search(op).group(1)) // 8
        unit = width * 64 if "st64" in op else width     # two-address forms count elements
        offsets = [int(n, 0) for n in re.findall(r"offset:(\w+)", text)]
        pairs = [int(n, 0) * unit for n in re.findall(r"offset[01]:(\w+)", text)]
        most = max([most, width] + [o + width for o in offsets + pairs])
    return most


def run(tool, *args):
    return subprocess.run([LLVM + tool, *args], check=True, capture_output=True, text=True).stdout


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("n", [24, 520, 8192, 12288, 16384])
@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("after", [True, False])
def test_lds_accesses_fit_the_allocation(dtype, n, aligned, after):
    x = torch.empty((64, n), device="meta", dtype=getattr(torch, dtype))
    for gate in ("none", "rows", "group"):
        var = RN._variant(x, aligned, 64, n, after, gate, True)
        program, name = RN._program("backward", var), residual_norm_kernel_name("backward", var)
        program.precompile()
        path = str(hip._cache_file(program.source, program.options))
        code = re.search(rf"<{name}>:(.*?)(?:\n\n|\Z)", run("llvm-objdump", "-d", path), re.S).group(1)
        notes = run("llvm-readelf", "--notes", path).split("- .agpr_count")
        (kernel,) = [part for part in notes if re.search(rf"\.name: +{name}\n", part)]
        allocated = int(re.search(r"group_segment_fixed_size: (\d+)", kernel).group(1))
        assert reach(code) <= allocated, f"{name}: {reach(code)} of {allocated} bytes"


@pytest.mark.parametrize("text,found", [
    ("\tds_write_b128 v2, v[2:5] offset:33168", 33184),
    ("\tds_write_b32 v41, v40", 4),
    ("\tds_read2_b32 v[0:1], v2 offset0:3 offset1:255", 1024),
    ("\tds_write2st64_b64 v2, v[0:1], v[2:3] offset1:2", 1032),
    ("\tv_mov_b32_e32 v33, v50", 0),
])
def test_the_reader_finds_what_it_looks_for(text, found):
    assert reach(text) == found
