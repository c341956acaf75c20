"""Build the HIP library ``lucid_amd/liblucid_amd.so`` for gfx950 (in-tree).

Usage: ``python -m lucid_amd.build``.  hipcc cross-compiles without a GPU.
"""
from __future__ import annotations

import concurrent.futures
import os
import subprocess
import sys
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
ARCH = os.environ.get("LUCID_OFFLOAD_ARCH", "gfx950")

# Every HIP translation unit is compiled with packed-fp32 instructions disabled.  Host code
# gets hidden symbol visibility: each library exports only the extern "C" entry points its
# header declares, so two libraries loaded into one process (RTLD_GLOBAL included) never
# bind each other's internal helpers or their static state.
HIPCC_FLAGS = [
    f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Xarch_host", "-fvisibility=hidden", "-Xarch_host", "-fvisibility-inlines-hidden",
]

# Sources of each library: one translation unit each, compiled side by side.
TARGETS = {
    "liblucid_amd.so": ["lucid_capi.hip", "prompt_capi.hip"],
    "liblucid_path.so": ["path_capi.hip"],
}


def _run(cmd: list[str], what: str, verbose: bool) -> None:
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"hipcc failed for {what}:\n{res.stderr}")


def build(verbose: bool = False) -> list[str]:
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    built = []
    with tempfile.TemporaryDirectory() as tmp:
        objects = {src: os.path.join(tmp, src + ".o") for srcs in TARGETS.values() for src in srcs}

        def compile_one(src: str) -> None:
            _run([hipcc, *HIPCC_FLAGS, "-c", "-o", objects[src], os.path.join(CSRC, src)], src, verbose)

        with concurrent.futures.ThreadPoolExecutor() as pool:
            list(pool.map(compile_one, objects))
        for out, srcs in TARGETS.items():
            dst = os.path.join(HERE, out)
            _run([hipcc, *HIPCC_FLAGS, "-shared", "-o", dst + ".tmp", *(objects[s] for s in srcs)], out, verbose)
            os.replace(dst + ".tmp", dst)
            built.append(dst)
    return built


if __name__ == "__main__":
    for p in build(verbose="-v" in sys.argv):
        print("built", p)
