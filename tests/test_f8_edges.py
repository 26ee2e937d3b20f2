"""C ABI, build and documents of the feed-forward operators in 8-bit floating point, on the host alone: no call here gets as far as a launch."""
import os
import struct
import subprocess
import sys

import pytest

from accera_amd import _lib
from test_f8_abi import GOOD, ROOT, _fields


def _packed(entry, **change):
    args = dict(GOOD[entry], **change)
    fields = _fields(entry + "_call")
    return struct.pack("".join("d" if d else "Q" if p else "q" for _, d, p in fields), *(args[n] for n, _, _ in fields))


@pytest.mark.parametrize("entry,sizes", [("acc950_expert_plan", ("tokens", "top_k", "experts")), ("acc950_f8_expert_ffn", ("tokens", "hidden", "inner", "experts", "top_k"))])
def test_a_workspace_that_is_too_small_is_refused(entry, sizes):
    L = _lib.lib()
    need = getattr(L, entry + "_workspace")(*(GOOD[entry][n] for n in sizes))
    assert need > 0
    for smaller in (need - 1, 1, 0, -1):
        assert getattr(L, entry + "_within")(_packed(entry), smaller) == _lib.INVALID_ARGUMENT
        assert b"workspace is smaller" in L.acc950_last_error()
    assert getattr(L, entry + "_within")(None, need) == _lib.INVALID_ARGUMENT
    # a size that the call does not take, whatever the workspace; nothing to do
    assert getattr(L, entry + "_within")(_packed(entry, experts=2000), 1 << 60) == _lib.INVALID_ARGUMENT and b"1024 experts" in L.acc950_last_error()
    if entry == "acc950_f8_expert_ffn":
        assert L.acc950_f8_expert_ffn_within(_packed(entry, tokens=0), 0) == _lib.OK


@pytest.mark.parametrize("python,binding", [(sys.executable, True), (sys.executable + " -S -E", False)])
def test_the_c_library_is_built_without_torch(python, binding):
    """The binding to torch tensors needs torch's headers; a Python that has no torch builds everything else."""
    out = subprocess.run(["make", "-n", "-B", "-C", os.path.join(ROOT, "accera_amd", "csrc"), f"PYTHON={python}"], capture_output=True, text=True, timeout=100)
    assert out.returncode == 0, out.stderr[-500:]
    assert "-o ../lib/libaccera_mi355x.so" in out.stdout and "-o ../lib/libaccera_mi355x_probes.so" in out.stdout
    assert ("-o ../lib/_torch_f8.so" in out.stdout) == binding and ("is left out" in out.stdout) != binding
