"""The dense prefill kernels keep their values in registers: what the compiler prints of them."""
import re
import subprocess

import pytest


@pytest.mark.slow
def test_the_dense_prefill_kernels_do_not_spill(tmp_path):
    from npu_b200 import build

    try:
        nvcc = build._nvcc()
    except RuntimeError:
        pytest.skip("needs nvcc")
    r = subprocess.run([nvcc, *build.ARCH, *build.NVCC_FLAGS, *build.FAST_MATH, "-Xptxas", "-v", "-c",
                        str(build.CSRC / "prefill.cu"), "-o", str(tmp_path / "prefill.o")],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    entries = re.findall(r"Compiling entry function '(\S+)'.*?(\d+) bytes spill stores, (\d+) bytes spill loads",
                         r.stderr, re.S)
    # fa_prefill_kernel<D, tiles, head pairs, packed>: the flags are b0 / b1 in the mangled names.
    dense = [(name, int(stores), int(loads)) for name, stores, loads in entries
             if re.search(r"fa_prefill_kernelILi\d+ELi\d+ELb\dELb0E", name)]
    assert len(dense) == 6
    assert all(stores == loads == 0 for _, stores, loads in dense), dense
