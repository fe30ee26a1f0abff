"""Build libdsx.so in-tree with hipcc for gfx950, and the autograd nodes of the
block operators (_block_autograd.so, host C++).

    python -m distributedspeed_amd.build

The flags that matter for correctness:
  -ffp-contract=off   (the optimizer step) no implicit fused multiply-adds:
                      each operation rounds where torch's kernels round
                      (explicit fmaf only)
  -Xclang -target-feature -Xclang -packed-fp32-ops
                      no packed fp32 instructions (v_pk_*_f32)
and for speed:
  -mllvm -amdgpu-kernarg-preload-count=16
                      a kernel's leading arguments (the buffers and sizes) are
                      in scalar registers when its waves start, instead of
                      being the first trip to memory of each: flat steps on
                      MI355X 9.5 -> 9.2 us at 9.0e5 elements, 12.9 -> 12.6 at
                      1.9e6, 18.5 -> 18.0 at 3.0e6, nothing from 7.1e6 on (8,
                      14 and 16 registers alike)
HIP's defaults keep fp32 division and sqrt correctly rounded and fp32
denormals intact, which the element math relies on.
"""
from __future__ import annotations

import os
import subprocess
import sys
import sysconfig
import tempfile
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(ROOT, "include")
OUT = os.path.join(HERE, "libdsx.so")
AUTOGRAD = os.path.join(HERE, "_block_autograd.so")
ARCH = os.environ.get("DSX_OFFLOAD_ARCH", "gfx950")

# source -> its own flags. The optimizer step rounds where torch rounds; the
# block and Muon kernels have no such partner and may contract.
SOURCES = {
    "dsx_step.hip": ["-ffp-contract=off"],
    "dsx_muon.hip": [],
    "dsx_ffn.hip": [],
    "dsx_norm.hip": [],
}


def hipcc() -> str:
    for cand in (os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "bin", "hipcc"), "hipcc"):
        if os.path.sep not in cand or os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found")


def command(source: str, out: str, extra: list[str] | None = None) -> list[str]:
    """The compile command of one source to an object file."""
    return [hipcc(), f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC", "-c", *SOURCES[source],
            "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
            "-mllvm", "-amdgpu-kernarg-preload-count=16",
            "-Wall", "-Wno-unused-function",
            f"-I{INCLUDE}", f"-I{CSRC}", os.path.join(CSRC, source), "-o", out] + list(extra or [])


def autograd_command(out: str) -> list[str]:
    """The compile command of the autograd nodes of the block operators: host
    C++ against torch, calling libdsx through addresses bound at load."""
    import torch
    from torch.utils import cpp_extension
    includes = [*cpp_extension.include_paths(), sysconfig.get_paths()["include"], INCLUDE]
    return ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
            *[a for i in includes for a in ("-isystem" if "torch" in i else "-I", i)],
            os.path.join(CSRC, "block_autograd.cpp"), "-o", out,
            *[f"-L{d}" for d in cpp_extension.library_paths()], "-lc10", "-ltorch", "-ltorch_cpu", "-ltorch_python"]


def _run(cmd: list[str]) -> list[str]:
    res = subprocess.run(cmd, capture_output=True, text=True)
    # hipcc's host pass warns that it does not know the packed-fp32 feature: harmless.
    noise = [ln for ln in (res.stderr or "").splitlines() if "packed-fp32-ops" not in ln and ln.strip()]
    if res.returncode != 0:
        raise RuntimeError(f"{os.path.basename(cmd[0])} failed:\n" + "\n".join(noise))
    return noise


def build(out: str = OUT, autograd: str = AUTOGRAD, verbose: bool = False) -> str:
    with tempfile.TemporaryDirectory(prefix="dsx_build_") as tmp:
        objects = {src: os.path.join(tmp, src + ".o") for src in SOURCES}
        jobs = [command(src, objects[src]) for src in SOURCES] + [autograd_command(autograd + ".tmp")]
        with ThreadPoolExecutor(max_workers=min(5, len(jobs))) as pool:
            noise = [ln for got in pool.map(_run, jobs) for ln in got]
        _run([hipcc(), f"--offload-arch={ARCH}", "-fPIC", "-shared", *objects.values(), "-o", out + ".tmp"])
    if verbose and noise:
        print("\n".join(noise), file=sys.stderr)
    os.replace(out + ".tmp", out)
    os.replace(autograd + ".tmp", autograd)
    return out


if __name__ == "__main__":
    print(build(verbose=True))
