"""The built kernels hold no packed float32 instructions: hipcc makes them from ordinary float code unless it is told not to, and some of
their forms have given wrong results now and then."""
import os
import re
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nrhints_amd", "csrc")
OBJ = os.path.join(CSRC, "..", "lib", "obj")
LLVM = "/opt/rocm/llvm/bin"
UNITS = ("nrh_api", "nrh_small", "nrh_wide", "nrh_wide1", "nrh_linear", "nrh_embedding")


def test_every_unit_is_compiled_without_them():
    text = open(os.path.join(CSRC, "Makefile")).read()
    flags = re.search(r"^FLAGS \?= (.*)$", text, re.M).group(1)
    assert "-Xclang -target-feature -Xclang -packed-fp32-ops" in flags
    compiled = [line for line in text.splitlines() if "$(HIPCC)" in line and " -c " in line]
    assert len(compiled) >= 2 * len(UNITS) and all("$(FLAGS)" in line for line in compiled)


@pytest.mark.parametrize("unit", UNITS)
def test_no_packed_float32_in_the_objects(unit, tmp_path):
    obj = os.path.join(OBJ, unit + ".o")
    if not (os.path.exists(obj) and os.path.exists(os.path.join(LLVM, "llvm-objdump"))):
        pytest.skip("no object of this unit here")
    bundle, code = str(tmp_path / "bundle"), str(tmp_path / "code")
    subprocess.run([os.path.join(LLVM, "llvm-objcopy"), f"--dump-section=.hip_fatbin={bundle}", obj, os.devnull], check=True)
    subprocess.run([os.path.join(LLVM, "clang-offload-bundler"), "--type=o", "--unbundle", f"--input={bundle}", f"--output={code}",
                    "--targets=hipv4-amdgcn-amd-amdhsa--gfx950"], check=True)
    listing = subprocess.run([os.path.join(LLVM, "llvm-objdump"), "-d", code], check=True, capture_output=True, text=True).stdout
    assert listing.count("s_endpgm") > 0
    assert not re.search(r"v_pk_(add|mul|fma)_f32", listing)
