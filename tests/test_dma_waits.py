"""A load in inline asm that reads a scalar less than five states after a vector
instruction wrote it reads another one, and the compiler, which waits before its own
loads, does not look into asm.  It restores spilled scalars by vector instructions
wherever it likes, so every such DMA waits by itself."""
import os
import re

from conftest import ROOT

CSRC = os.path.join(ROOT, "circulantattention.jl_amd", "csrc")


def test_buffer_loads_in_asm_wait_for_their_scalars():
    found = 0
    for name in sorted(os.listdir(CSRC)):
        text = open(os.path.join(CSRC, name)).read()
        for stmt in re.findall(r"asm\s+volatile\s*\((.*?)\);", text, flags=re.S):
            if "buffer_load" in stmt:
                own = re.match(r'\s*"s_nop (\d+)\\n', stmt)
                assert stmt.lstrip().startswith("CIRCATT_SCALARS_READY") or own and int(own[1]) + 1 >= 5, (name, stmt)
                found += 1
    assert found >= 3
    wait = re.search(r'#define CIRCATT_SCALARS_READY "s_nop (\d+)\\n\\t"', open(os.path.join(CSRC, "buffer_dma.h")).read())
    assert int(wait[1]) + 1 >= 5
