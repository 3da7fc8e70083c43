"""The block boundary's kernels on the CPU: every address that a call touches lies inside its buffers."""
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))
CLANG = "/opt/rocm/lib/llvm/bin/clang++"


def test_block_kernels_stay_inside_their_buffers(tmp_path):
    """tok_elem.hip built for the CPU without optimisation (a load whose value is not used stays), each
    buffer at the edge of a page that cannot be read: widths that fill their threads and widths that
    leave threads behind the row's end, all forms of the call, forward and backward"""
    (tmp_path / "hip").mkdir()
    (tmp_path / "hip" / "hip_runtime.h").write_text("")  # (the build gives its own forms of what it names)
    exe = str(tmp_path / "bounds")
    subprocess.check_call([CLANG, "-x", "c++", "-std=c++17", "-O0", "-Wno-everything", "-I", str(tmp_path),
                           os.path.join(HERE, "tok_elem_host.cpp"), "-o", exe])
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "inside their buffers" in r.stdout, r.stdout
