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


def test_offsets_past_32_bits_go_to_the_kernels_that_hold_them():
    """What the kernels with 32-bit offsets from a tile's first row cannot reach, told by the scratch memory that the other path takes."""
    def layer(hidden):
        return _lib.lib().acc950_f8_expert_ffn_workspace(1, hidden, 128, 1, 1)

    def codes_only(hidden):  # every step's results but the gate and up product's in fp32
        up = lambda n: -(-n // 256) * 256  # noqa: E731
        return 6 * 256 + up(hidden) + up(hidden // 128 * 4) + up(4 * hidden) + up(hidden // 64 * 2 * 4)
    small, large = (1 << 24) - 128, 1 << 25
    assert layer(small) == codes_only(small) and layer(large) == codes_only(large) + 2 * 128 * 4

    def product(**change):
        return getattr(_lib.lib(), "acc950_f8_gemm_workspace")(_packed("acc950_f8_gemm", **{**dict(out_type=_lib.F32, M=256, N=512, K=1 << 20, a_row_stride=1 << 20, b_col_stride=1 << 20,
                                                                                                  as_block_stride=256, bs_col_stride=1 << 13, c_row_stride=512), **change}))
    assert product() > 0  # (slices of K)
    # rows that overlap (a matrix of all windows of a long row): the last one ends far behind its start
    far = (1 << 24) - 16
    assert product(a_row_stride=16) > 0 and product(K=1 << 25, b_col_stride=far, a_row_stride=16, bs_col_stride=1 << 18) == 0
    assert product(K=1 << 25, b_col_stride=16, a_row_stride=far, bs_col_stride=1 << 18) == 0
    # strides whose product with a tile's rows passes 64 bits
    assert product(a_row_stride=1 << 56) == 0 and product(b_col_stride=1 << 56) == 0 and product(as_row_stride=1 << 54) == 0
