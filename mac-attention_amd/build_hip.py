"""Builds the libraries for gfx950 with hipcc (no CMake, no JIT):

* libmac_hip.so -- the product: decode step, ring-cache ops, prefill
  rectification, decode RoPE, the 8-bit paged cache and the paged chunk
  attention;
* libmac_noalloc.so -- the decode step with its workspaces in a static device
  array (linked against libmac_hip.so; only processes that load it reserve
  the array);
* libmac_bench.so -- measurement helpers (streaming read; the decode step
  timed kernel by kernel, from the same decode source with its C ABI hidden).
"""

from __future__ import annotations

import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(HERE)
SOURCES = [os.path.join(HERE, "csrc", f) for f in ("mac_decode.hip", "mac_cache_ops.hip", "mac_prefill.hip", "mac_rope.hip",
                                                   "mac_paged_cache.hip", "mac_paged_api.hip")]
# the paged chunk attention's kernels, compiled once per variant (queries' type,
# cache of that type or e4m3), with the type codes of mac_attention_amd.h
PAGED_SOURCE = os.path.join(HERE, "csrc", "mac_paged_attention.hip")
PAGED_VARIANTS = {"bf16": ("MAC_DTYPE_BF16", 0), "f16": ("MAC_DTYPE_F16", 0),
                  "bf16_fp8": ("MAC_DTYPE_BF16", 1), "f16_fp8": ("MAC_DTYPE_F16", 1)}
OUTPUT = os.path.join(HERE, "libmac_hip.so")
NOALLOC_SOURCES = [os.path.join(HERE, "csrc", "mac_noalloc.hip")]
NOALLOC_OUTPUT = os.path.join(HERE, "libmac_noalloc.so")
BENCH_SOURCES = [os.path.join(HERE, "csrc", "mac_bench.hip"), os.path.join(HERE, "csrc", "mac_decode.hip")]
BENCH_OUTPUT = os.path.join(HERE, "libmac_bench.so")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")

FLAGS = [
    "-O3",
    "-std=c++17",
    # keep the compiler from forming packed-fp32 VALU ops (some of their forms
    # have given wrong results on the target machines, without any error)
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-fvisibility=hidden",
    # MFMA accumulators in VGPRs: the online-softmax rescale then works on
    # them in place instead of copying them through AGPRs every block
    "-mllvm", "-amdgpu-mfma-vgpr-form",
    "-I", os.path.join(REPO, "include"),
    "-I", os.path.join(HERE, "csrc"),
]


def _hipcc(sources: list[str], output: str, verbose: bool, extra: list[str] | None = None) -> str:
    linking = all(x.endswith(".o") or x.startswith("-") for x in sources)
    flags = [] if linking else FLAGS
    cmd = [HIPCC, "--offload-arch=gfx950", "-fPIC", *flags, *sources, "-o", output, *(extra or [])]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    noise = "'-packed-fp32-ops' is not a recognized feature"
    err = "\n".join(l for l in res.stderr.splitlines() if noise not in l)
    if res.returncode != 0:
        raise RuntimeError(f"hipcc failed ({res.returncode}):\n{err}")
    if verbose and err.strip():
        print(err, file=sys.stderr)
    return output


def _objects(folder: str) -> list[tuple[list[str], str]]:
    """(hipcc arguments, object) of the decode library's compilations."""
    jobs = [([src], os.path.join(folder, os.path.basename(src) + ".o")) for src in SOURCES]
    for name, (t, f8) in PAGED_VARIANTS.items():
        jobs.append(([f"-DMAC_PAGED_NAME={name}", f"-DMAC_PAGED_T={t}", f"-DMAC_PAGED_F8={f8}", PAGED_SOURCE],
                     os.path.join(folder, f"mac_paged_attention_{name}.o")))
    return jobs


def build(verbose: bool = False) -> str:
    """All three libraries; returns the decode library's path."""
    import tempfile
    from concurrent.futures import ThreadPoolExecutor

    with tempfile.TemporaryDirectory() as folder, ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as pool:
        # the decode library's C ABI stays hidden in the measurement library
        bench = pool.submit(_hipcc, ["-shared", *BENCH_SOURCES], BENCH_OUTPUT, verbose, ["-DMAC_API="])
        parts = [pool.submit(_hipcc, ["-c", *args], obj, verbose) for args, obj in _objects(folder)]
        _hipcc(["-shared", *(p.result() for p in parts)], OUTPUT, verbose)
        _hipcc(["-shared", *NOALLOC_SOURCES], NOALLOC_OUTPUT, verbose, ["-L" + HERE, "-lmac_hip", "-Wl,-rpath,$ORIGIN"])
        bench.result()
    return OUTPUT


if __name__ == "__main__":
    print(build(verbose=True))
