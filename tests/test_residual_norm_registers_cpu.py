"""Which forms of the residual norm's gradient hold a row's state in registers, read from the units built here."""
import re
import subprocess

import pytest
import torch

from neptune_codegen import hip, residual_norm as RN
from neptune_codegen.emitters import residual_norm_kernel_name


def spilled(var):
    program, name = RN._program("backward", var), residual_norm_kernel_name("backward", var)
    program.precompile()
    notes = subprocess.run(["/opt/rocm/llvm/bin/llvm-readelf", "--notes",
                            str(hip._cache_file(program.source, program.options))],
                           check=True, capture_output=True, text=True).stdout
    (kernel,) = [part for part in notes.split("- .agpr_count") if re.search(rf"\.name: +{name}\n", part)]
    return int(re.search(r"\.vgpr_spill_count: +(\d+)", kernel).group(1))


# (columns, slots a lane, whether a form spills)
@pytest.mark.parametrize("dtype,n,slots,spills", [
    ("bfloat16", 4096, 1, lambda *_: False), ("float32", 4096, 1, lambda *_: False),
    ("bfloat16", 8192, 1, lambda aligned, after, gate: after and (gate == "group" or gate == "rows" and not aligned)),
    ("bfloat16", 12288, 3, lambda aligned, after, gate: after and gate == "group" and not aligned),
    ("float16", 12288, 3, lambda aligned, after, gate: after and gate == "group" and not aligned)])
@pytest.mark.parametrize("aligned", [True, False])
def test_forms_that_fit_their_registers(dtype, n, slots, spills, aligned):
    x = torch.empty((64, n), device="meta", dtype=getattr(torch, dtype))
    for after in (True, False):
        for gate in ("none", "rows", "group"):
            var = RN._variant(x, aligned, 64, n, after, gate, True)
            assert var.nv == slots
            assert spills(aligned, after, gate) or spilled(var) == 0, (after, gate)
