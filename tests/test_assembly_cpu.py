"""The kernels' assembly, compiled here from their sources: registers are saved with all lanes on.

Where a branch takes some lanes, its end is a label and the restoring of the lanes (``s_or_b64 exec, exec, ..``).  The compiler
may put a register that it has to save to memory between the two: then only the branch's lanes are saved, and the others read
back what lay there.  Two builds had it, both with more to hold than registers (284 bytes a lane in memory in one): a row's number
and place were saved, and results were written to other rows.  No source asks for such a save, so that only the result can be
looked at.
"""

from __future__ import annotations

import os
import re
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

from flux_amd import build

SOURCES = sorted((s for s in build.SOURCES if s.endswith(".hip")), key=lambda s: -os.path.getsize(os.path.join(build.CSRC, s)))


def saves_with_lanes_off(assembly: str) -> list[str]:
    """Lines that save or reload a register behind a label and before the lanes are restored in its block."""
    found, held = [], None
    for line in assembly.splitlines():
        text = line.strip()
        if re.match(r"\.LBB\w+:", text):
            held = []
        elif not text or text[0] in ".;":
            if text.startswith("; %bb"):
                held = None
        elif held is not None:
            if re.match(r"s_or_b64 exec, exec|s_or_saveexec_b64", text):
                found += held
                held = None
            elif text.startswith(("s_cbranch", "s_branch")) or re.match(r"s_\w+ .*exec", text):
                held = None
            elif re.search(r"; .*(Spill|Reload)", text):
                held.append(text)
    return found


def test_the_search_finds_a_planted_save():
    before = "\n".join((".LBB14_146:", "\ts_or_b64 exec, exec, s[28:29]", "\tscratch_store_dword off, v1, off ; 4-byte Folded Spill",
                        ".LBB14_147:", "\tv_mov_b32_e32 v2, v3"))
    after = "\n\ts_or_b64 exec, exec, s[10:11]\n\tscratch_load_dword v5, off, off offset:8 ; 4-byte Folded Reload\n"
    assert saves_with_lanes_off(before + after) == []
    planted = "\tscratch_store_dword off, v192, off offset:268 ; 4-byte Folded Spill"
    assert saves_with_lanes_off(before + "\n" + planted + after) == [planted.strip()]
    moved = "\tv_accvgpr_write_b32 a3, v7 ;  Reload Reuse"
    assert saves_with_lanes_off(before + "\n" + moved + after) == [moved.strip()]


@pytest.fixture(scope="module")
def assemblies(tmp_path_factory):
    out = tmp_path_factory.mktemp("assembly")

    def compile_one(source: str) -> str:
        target = str(out / (source + ".s"))
        command = [build.hipcc(), *build._flags(), "-S", "--cuda-device-only", os.path.join(build.CSRC, source), "-o", target]
        result = subprocess.run(command, capture_output=True, text=True)
        assert result.returncode == 0, result.stderr
        with open(target) as file:
            return file.read()

    with ThreadPoolExecutor(max_workers=min(4, os.cpu_count() or 1)) as pool:
        return dict(zip(SOURCES, pool.map(compile_one, SOURCES)))


@pytest.mark.parametrize("source", SOURCES)
def test_registers_are_saved_with_all_lanes_on(assemblies, source):
    assert assemblies[source].count("s_endpgm") > 0
    assert saves_with_lanes_off(assemblies[source]) == []
