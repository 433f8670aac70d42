"""Build the gfx950 HIP library ``libffamd.so`` in-tree with hipcc.

Each ``csrc/*.hip`` file is compiled to an object for ``--offload-arch=gfx950``
and the objects are linked into ``fastforward_amd/libffamd.so`` (a plain C-ABI
shared library; no torch headers). Run ``python -m fastforward_amd.build``.
"""
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libffamd.so")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")

# -ffp-contract=off keeps each rounding point where the source writes it.
# Packed fp32 instructions are disabled for every device compile.
FLAGS = ["--offload-arch=gfx950", "-O3", "-fPIC", "-std=c++17", "-ffp-contract=off",
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
         "-Wno-unused-result", "-I", os.path.join(HERE, "..", "include")]

# The block-scaled products add each matrix instruction's result to sums in ordinary
# registers; left to itself the compiler writes the result to accumulation registers
# where a wave may use more than 256, and reads every value back for its add.
_VGPR_RESULTS = ["-mllvm", "-amdgpu-mfma-vgpr-form=1"]
# Paged attention: the scores go through the softmax, which reads ordinary registers.
EXTRA_FLAGS = {"ff_gemm_fp8_block.hip": _VGPR_RESULTS, "ff_moe.hip": _VGPR_RESULTS,
               "ff_attention_paged.hip": _VGPR_RESULTS}


def sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".hip"))


def _compile(src):
    obj = os.path.join(OBJ, os.path.basename(src)[:-4] + ".o")
    cmd = [HIPCC, *FLAGS, *EXTRA_FLAGS.get(os.path.basename(src), []), "-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src}:\n{r.stderr}")
    return obj


def build(verbose=True):
    os.makedirs(OBJ, exist_ok=True)
    srcs = sources()
    with ThreadPoolExecutor(max_workers=min(8, len(srcs))) as ex:
        objs = list(ex.map(_compile, srcs))
    tmp = LIB + ".tmp"
    cmd = [HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", tmp, *objs]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stderr}")
    os.replace(tmp, LIB)
    if verbose:
        print(f"built {LIB} from {len(srcs)} sources")
    return LIB


if __name__ == "__main__":
    build()
    sys.exit(0)
