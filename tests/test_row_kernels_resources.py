"""Registers of the 8-bit row kernels as the compiler reports them (no GPU needed).

The norm's backward launches as many blocks as are resident at once: four of 128 threads
an SM with vector loads, three with single ones.  A kernel whose registers leave room for
fewer makes the last of them wait for the others to end, and one that spills moves the
spilled values through the memory that bounds it."""
import os
import re
import subprocess

import pytest

from momentummamba_b200 import build

REGISTERS = 65536   # of an SM


@pytest.fixture(scope="module")
def backward_forms():
    """{(dn type, dx type, vector loads, chunks, threads): (registers, spilled bytes)}"""
    cmd = [build._nvcc(), *build.NVCC_FLAGS, "-I", os.path.join(build.ROOT, "include"), "-Xptxas", "-v", "-cubin",
           os.path.join(build.CSRC, "rows8.cu"), "-o", os.devnull]
    out = subprocess.run(cmd, capture_output=True, text=True, check=True).stderr
    forms = {}
    for name, rest in re.findall(r"Compiling entry function '(\w*r8_bwd_kernel\w*)'(.*?Used \d+ registers)", out, re.S):
        t = re.search(r"T8(F32|BF16|F16)ENS_\d+T8(F32|BF16|F16)ELb([01])ELi(\d+)ELi\d+ELi(\d+)E"
                      r"|T8(F32|BF16|F16)ES1_Lb([01])ELi(\d+)ELi\d+ELi(\d+)E", name)
        assert t, name
        a, b, vec, nc, nt = t.groups()[:5] if t.group(1) else (t.group(6), *t.groups()[5:])
        regs = int(re.search(r"Used (\d+) registers", rest).group(1))
        spill = int(re.search(r"(\d+) bytes spill stores", rest).group(1))
        key = (a, b, vec == "1", int(nc), int(nt))
        forms[key] = max(forms.get(key, (0, 0)), (regs, spill))
    assert len(forms) >= 40
    return forms


def test_blocks_of_the_backward_fit_side_by_side(backward_forms):
    for (a, b, vec, nc, threads), (regs, spill) in backward_forms.items():
        if threads == 128:
            assert regs * threads * (4 if vec else 3) <= REGISTERS, (a, b, vec, nc, regs)


def test_rows_of_up_to_8192_columns_spill_nothing(backward_forms):
    """Wider rows take four chunks in blocks of up to 512 threads, where some forms do."""
    for form, (regs, spill) in backward_forms.items():
        if form[3:] != (4, 512):
            assert spill == 0, (form, spill)
