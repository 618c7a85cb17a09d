"""CPU check on the gfx950 assembly of paged.hip (no GPU needed): m0, the LDS base
of its direct global->LDS loads, is set from inline asm that the compiler does not
see, so nothing else in the unit may define or read it. Kernels spill no VGPRs."""

import importlib.util
import os
import re

_REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_spec = importlib.util.spec_from_file_location(
    "fa_build", os.path.join(_REPO, "flash-attention-cuda_amd", "build.py"))
fa_build = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(fa_build)


def test_paged_kernels_touch_m0_only_in_their_loads_and_do_not_spill(tmp_path):
    text = fa_build.device_assembly("paged", str(tmp_path))
    assert "global_load_lds_dwordx4" in text
    problems = fa_build.m0_problems(text)
    assert not problems, "; ".join(problems[:5])
    spills = [int(n) for n in re.findall(r"\.vgpr_spill_count:\s+(\d+)", text)]
    assert spills and not any(spills)
