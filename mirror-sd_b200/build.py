"""Build the sm_100a CUDA library ``lib/libdflash_b200.so`` in-tree with nvcc,
and ``lib/dflash_paged.so``, the Python binding of its paged-cache and decode operators.

    python mirror-sd_b200/build.py [--force] [--verbose]

Only nvcc is needed for the library (no GPU), which is what the Python host
(`_native.py`) loads with ctypes and what the C ABI in include/dflash_b200.h
describes.  The binding needs g++ and the headers of Python and torch besides;
without torch it is left out, and when it does not compile the library is there
all the same (and the build says so and fails).
"""
import argparse
import hashlib
import importlib.util
import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
LIB_DIR = os.path.join(HERE, "lib")
LIB = os.path.join(LIB_DIR, "libdflash_b200.so")
BINDING = os.path.join(LIB_DIR, "dflash_paged.so")
BINDING_SOURCE = "paged_binding.cpp"
SOURCES = ["quant.cu", "w8_tc.cu", "attention.cu", "attention_tc.cu", "tc_gemm.cu", "lm_head.cu", "misc.cu", "anchor.cu",
           "f32_path.cu", "paged.cu", "paged_share.cu", "prefix_plan.cu", "q4_cache.cu", "q4_attention.cu", "q4_attention_tc.cu", "rope.cu", "verify.cu",
           "dflash_api.cu", "paged_api.cu", "decode_api.cu"]
HEADERS = ["common.cuh", "kernels.cuh", "q4.cuh", "q4_attn.cuh", "paged_scan.cuh", "decode.cuh", "api_error.cuh"]
NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-lineinfo", "-std=c++17",
              "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr", "-Xptxas", "-warn-spills"]


def _nvcc():
    for cand in [os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", "nvcc"]:
        if cand and (os.path.isabs(cand) and os.path.exists(cand) or not os.path.isabs(cand)):
            return cand
    return "nvcc"


def _torch_dir():
    spec = importlib.util.find_spec("torch")
    return spec and os.path.dirname(spec.origin)


def _torch_version():
    with open(os.path.join(_torch_dir(), "version.py")) as fh:
        return fh.read()


def _binding_command(out):
    torch = _torch_dir()
    return ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-isystem", os.path.join(torch, "include"), "-isystem",
            os.path.join(torch, "include", "torch", "csrc", "api", "include"), "-I" + sysconfig.get_paths()["include"],
            "-I" + os.path.join(os.path.dirname(os.path.dirname(_nvcc())) or "/usr/local/cuda", "include"),
            os.path.join(CSRC, BINDING_SOURCE), "-L" + os.path.join(torch, "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu",
            "-ltorch_python", "-o", out]


def _digest(sources, *how):
    h = hashlib.sha256(" ".join(how).encode())
    for f in sources:
        with open(os.path.join(CSRC, f), "rb") as fh:
            h.update(fh.read())
    with open(os.path.join(ROOT, "include", "dflash_b200.h"), "rb") as fh:
        h.update(fh.read())
    return h.hexdigest()


def _stamped(path, digest):
    if not os.path.exists(path) or not os.path.exists(path + ".sha256"):
        return False
    with open(path + ".sha256") as fh:
        return fh.read().strip() == digest


def _stamp(path, digest):
    with open(path + ".sha256", "w") as fh:
        fh.write(digest)


def build(force=False, verbose=False, jobs=None):
    os.makedirs(LIB_DIR, exist_ok=True)
    lib_digest = _digest(SOURCES + HEADERS, *NVCC_FLAGS)
    if force or not _stamped(LIB, lib_digest):
        _build_library(verbose)
        _stamp(LIB, lib_digest)
    if _torch_dir() is None:
        print(f"torch is not installed: {os.path.basename(BINDING)} (the paged operators' Python binding) is left out")
        return LIB
    # (an upgrade in place keeps torch's path, but not its headers)
    binding_digest = _digest([BINDING_SOURCE], _torch_version(), sys.version, *_binding_command(""))
    if force or not _stamped(BINDING, binding_digest):
        r = subprocess.run(_binding_command(BINDING + ".tmp"), capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"{LIB} is built, its Python binding is not:\n--- {BINDING_SOURCE}\n{r.stdout}\n{r.stderr}")
        os.replace(BINDING + ".tmp", BINDING)
        _stamp(BINDING, binding_digest)
    return LIB


def _build_library(verbose):
    objs = []
    procs = []
    for src in SOURCES:
        obj = os.path.join(LIB_DIR, src.replace(".cu", ".o"))
        cmd = [_nvcc(), *NVCC_FLAGS, "-c", os.path.join(CSRC, src), "-o", obj]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
            print(" ".join(cmd))
        procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)))
        objs.append(obj)
    failed = []
    for src, p in procs:
        out, _ = p.communicate()
        txt = out.decode(errors="replace")
        if p.returncode != 0:
            failed.append((src, txt))
        elif verbose and txt.strip():
            print(txt)
    if failed:
        msg = "\n".join(f"--- {s}\n{t}" for s, t in failed)
        raise RuntimeError(f"compilation failed:\n{msg}")
    tmp = LIB + ".tmp"
    link = [_nvcc(), "-shared", "-gencode", "arch=compute_100a,code=sm_100a", *objs, "-o", tmp]
    r = subprocess.run(link, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, LIB)
    for o in objs:
        os.remove(o)


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    a = ap.parse_args()
    print(build(force=a.force, verbose=a.verbose))
    sys.exit(0)
