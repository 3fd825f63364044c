"""The built libraries share the process's C++ runtime. With a copy of their own (a compiler that links libstdc++
statically) a refusal that printed a size ended the process: the copy's locale is not the one torch has set up."""
import shutil
import subprocess

import pytest


@pytest.mark.parametrize("name", ["LIB", "BINDING"])
def test_no_copy_of_the_cpp_runtime(name):
    from npu_b200 import build

    if not shutil.which("nm"):
        pytest.skip("needs nm")
    path = getattr(build, name)
    if not path.exists():
        build.build()
    r = subprocess.run(["nm", "-D", "--defined-only", str(path)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    symbols = [line.split()[-1] for line in r.stdout.splitlines()]
    assert any("PyInit__serving" in s or s.startswith("b2a_prefill") for s in symbols)
    own = [s for s in symbols if "basic_ostream" in s or "num_put" in s or "logic_error" in s]
    assert not own, own[:5]
