"""CPU test of the assembly of csrc/int8.hip.  Matrix instructions run for the whole wave whatever exec holds, so none may stand
behind a test of lanes: a block that the compiler guards with exec (s_cbranch_execz) may lose its branch and run masked,
which skips vector instructions, but not products.  Whether a product runs has to be a scalar branch."""

import pathlib
import re
import shutil
import subprocess

import pytest

ROOT = pathlib.Path(__file__).resolve().parents[1]
CSRC = ROOT / "alpha-fly_amd" / "csrc"


def test_products_stand_behind_scalar_branches(tmp_path):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not pathlib.Path(hipcc).exists():
        pytest.skip("hipcc is not installed")
    out = tmp_path / "int8.s"
    subprocess.run([hipcc, "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang", "-target-feature", "-Xclang",
                    "-packed-fp32-ops", f"-I{ROOT / 'include'}", "--cuda-device-only", "-S", "-x", "hip",
                    str(CSRC / "int8.hip"), "-o", str(out)], check=True, capture_output=True)
    products, masked, last = 0, {}, ""
    for line in out.read_text().splitlines():
        kernel = re.match(r"(_Z\w+):", line)
        if kernel:
            name, last = kernel.group(1), ""
        word = line.split(";")[0].split()
        if not word:
            continue
        if word[0].startswith(("s_cbranch", "s_branch", "s_endpgm")) or word[:2] == ["s_or_b64", "exec,"]:
            last = word[0]
        if word[0].startswith("v_mfma"):
            products += 1
            if last == "s_cbranch_execz":
                masked[name] = masked.get(name, 0) + 1
    assert products > 1000
    assert not masked, masked
