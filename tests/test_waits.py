"""The waits that the instruction set leaves to the program, in the built code (accera_amd/csrc/check_waits.py); on the host alone."""
import importlib.util
import os
import shutil
import subprocess
import sys

import pytest

from accera_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_spec = importlib.util.spec_from_file_location("check_waits", os.path.join(ROOT, "accera_amd", "csrc", "check_waits.py"))
check_waits = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(check_waits)

FILL = ["s_mov_b32 m0, s0", "s_nop 0", "global_load_lds_dwordx4 v9, s[4:5]"]


@pytest.mark.parametrize("code,what", [
    (["v_readlane_b32 s5, v251, 30", *FILL], "memory read"),
    (["v_readfirstlane_b32 s4, v1", "v_add_u32_e32 v2, v3, v4", *FILL], "memory read"),
    (["v_readlane_b32 s5, v251, 30", "s_nop 1", "v_add_u32_e32 v2, v3, v4", *FILL], None),
    (["v_readlane_b32 s5, v251, 30", "s_mov_b32 m0, s0", "s_mov_b64 s[6:7], s[4:5]", "global_load_lds_dwordx4 v9, s[6:7]"], None),
    (["v_readlane_b32 s6, v251, 30", "s_mov_b32 m0, s0", "s_mov_b64 s[6:7], s[4:5]", "global_load_lds_dwordx4 v9, s[6:7]"], None),
    (["v_readlane_b32 s5, v251, 30", "global_store_dword v[2:3], v4, off"], None),
    (["v_cmp_lt_f32_e32 vcc, v1, v2", "v_cndmask_b32_e32 v3, v4, v5, vcc"], "vector read"),
    (["v_cmp_lt_f32_e32 vcc, v1, v2", "s_nop 1", "v_cndmask_b32_e32 v3, v4, v5, vcc"], None),
    (["v_readlane_b32 s4, v250, 53", "v_mul_lo_u32 v225, v7, s4"], "vector read"),
    (["v_readfirstlane_b32 s4, v250", "s_nop 2", "v_readlane_b32 s5, v1, s4"], "number of a lane"),
    (["v_add_f64 v[2:3], v[4:5], v[6:7]", "v_readlane_b32 s1, v3, 16"], "read of a lane"),
    (["v_max_f64 v[2:3], v[4:5], v[6:7]", "s_nop 0", "v_mov_b32_dpp v1, v2 row_ror:8 row_mask:0xf bank_mask:0xf bound_ctrl:1"], "DPP read"),
    (["v_max_f64 v[2:3], v[4:5], v[6:7]", "s_nop 1", "v_mov_b32_dpp v1, v2 row_ror:8 row_mask:0xf bank_mask:0xf bound_ctrl:1"], None),
    (["v_exp_f32_e32 v1, v2", "v_add_f32_e32 v3, v1, v4"], "transcendental"),
    (["v_exp_f32_e32 v1, v2", "v_rcp_f32_e32 v3, v1"], None),
])
def test_the_check_sees_what_comes_too_soon(code, what):
    found = list(check_waits.violations(["0000000000001000 <kernel>:", *("\t" + line + "    // 000000001000: 00000000" for line in code)]))
    assert all(kernel == "kernel" for kernel, _, _, _ in found)
    assert [what in w for _, w, _, _ in found] == ([] if what is None else [True])


@pytest.mark.skipif(not shutil.which(check_waits.OBJDUMP), reason="no disassembler")
def test_no_instruction_of_the_built_kernels_comes_too_soon():
    """All kernels of the library: most of what inline assembly fetches stands behind addresses that the compiler may have brought back just before."""
    probes = os.path.join(os.path.dirname(_lib.LIB_PATH), "libaccera_mi355x_probes.so")
    assert sum(1 for _ in check_waits.code_objects(_lib.LIB_PATH)) >= 15
    run = subprocess.run([sys.executable, check_waits.__file__, _lib.LIB_PATH, probes], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr[:2000]
