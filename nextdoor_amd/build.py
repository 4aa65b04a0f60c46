"""Builds libnextdoor_amd.so (HIP kernels + C ABI) for gfx950 with hipcc, in-tree."""
import os
import shutil
import subprocess
from concurrent.futures import ThreadPoolExecutor

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG_DIR, "csrc")
OBJ_DIR = os.path.join(PKG_DIR, "build")
LIB_PATH = os.path.join(PKG_DIR, "libnextdoor_amd.so")

SOURCES = ["nd_capi.hip", "nd_graph.cpp", "nd_check.cpp", "nd_dropout.hip", "nd_attention.hip",
           "nd_vocabulary_loss.hip", "nd_layer_norm.hip", "nd_linear.hip", "nd_linear_bf16.hip", "nd_linear_f16.hip"]

# -ffp-contract=off: the samplers compare single IEEE float operations bit for bit with
# the CPU checker.  The target-feature pair switches packed-fp32 code generation off.
HIPCC_FLAGS = [
    "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-shared", "-ffp-contract=off",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
]


def find_hipcc():
    for cand in (shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found")


def _run(cmd):
    proc = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    # the host pass warns that it does not know the packed-fp32 feature; that is expected
    log = "\n".join(l for l in proc.stdout.splitlines() if "packed-fp32-ops" not in l)
    if proc.returncode != 0:
        raise RuntimeError("hipcc failed:\n" + log)
    return log


def _compile(source):
    obj = os.path.join(OBJ_DIR, source + ".o")
    return obj, _run([find_hipcc()] + [f for f in HIPCC_FLAGS if f != "-shared"] +
                     ["-c", os.path.join(CSRC, source), "-o", obj])


def build(verbose=False):
    """Compiles every HIP source of the package, side by side; raises on failure.  Returns the .so path."""
    os.makedirs(OBJ_DIR, exist_ok=True)
    with ThreadPoolExecutor(min(len(SOURCES), os.cpu_count() or 1)) as pool:
        done = list(pool.map(_compile, SOURCES))
    log = [text for _, text in done]
    log.append(_run([find_hipcc()] + HIPCC_FLAGS + [obj for obj, _ in done] + ["-o", LIB_PATH, "-lpthread"]))
    if verbose and any(text.strip() for text in log):
        print("\n".join(text for text in log if text.strip()))
    return LIB_PATH


if __name__ == "__main__":
    print(build(verbose=True))
