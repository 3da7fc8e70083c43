"""The token operators' kernels on the CPU: every address that a call touches lies inside its buffers."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(HERE)
CLANG = "/opt/rocm/lib/llvm/bin/clang++"
CSRC = os.path.join("pcd_reg_hregnet_amd", "csrc")


@pytest.mark.parametrize("source", ["tok_elem", "tok_attn"])
def test_kernels_stay_inside_their_buffers(source, tmp_path):
    """the source built for the CPU without optimisation (a load whose value is not used stays), each buffer at the
    edge of a page that cannot be read: widths, lengths, masks, strides and launch plans of every kind, forward and
    backward"""
    (tmp_path / "hip").mkdir()
    (tmp_path / "hip" / "hip_runtime.h").write_text("")  # (host_hip.h gives what is needed of it)
    (tmp_path / CSRC).mkdir(parents=True)
    shutil.copytree(os.path.join(REPO, "include"), tmp_path / "include")
    for name in ("common.h", "tokens.h", source + ".hip"):
        with open(os.path.join(REPO, CSRC, name)) as f:
            text = f.read()
        # the launch's LDS is a buffer like the others; registers are not the GPU's
        text = text.replace("extern __shared__ __attribute__((aligned(16))) uint16_t lds[];", "uint16_t *const lds = host_lds;")
        text = text.replace('asm volatile("" : "+v"(row), "+v"(col));', "")
        (tmp_path / CSRC / name).write_text(text)
    exe = str(tmp_path / "bounds")
    subprocess.check_call([CLANG, "-x", "c++", "-std=c++17", "-O0", "-Wno-everything", "-I", str(tmp_path), "-I", HERE,
                           os.path.join(HERE, source + "_host.cpp"), "-o", exe])
    r = subprocess.run([exe], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0 and "inside their buffers" in r.stdout, r.stdout
