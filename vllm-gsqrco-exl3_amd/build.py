"""Builds libgguf_mi355x.so (the C-ABI library of include/gguf_mi355x.h) for gfx950 with hipcc,
and the torch op registration over it.

    python vllm-gsqrco-exl3_amd/build.py [--jobs N]

Each csrc/*.hip is compiled to an object in _build/ (in parallel), then linked into
vllm_gguf_plugin/libgguf_mi355x.so, in-tree, where vllm_gguf_plugin._capi loads it.
csrc/torch_ops.cpp (host C++ against PyTorch-ROCm's headers) is compiled alongside into
vllm_gguf_plugin/_C_gguf_ops.so, which links libgguf_mi355x.so next to it and registers
torch.ops._C_gguf when vllm_gguf_plugin._C_gguf loads it. csrc/bench/peaks.hip (bench.py's
measurement kernels, outside the C ABI) is built into vllm_gguf_plugin/libgguf_peaks.so.

csrc/decoder/*.hip (rotation into the 8-bit cache, attention over it and kept paths of drafts, block norms, the gated
delta rule, log probabilities) become
vllm_gguf_plugin/libgguf_decoder.so, the C ABI of include/gguf_decoder.h, and csrc/decoder/torch_ops.cpp
its registration _C_gguf_decoder_ops.so, which vllm_gguf_plugin.decoder loads.
"""

import argparse
import concurrent.futures as cf
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
BUILD = os.path.join(HERE, "_build")
OUT = os.path.join(HERE, "vllm_gguf_plugin", "libgguf_mi355x.so")
OPS_OUT = os.path.join(HERE, "vllm_gguf_plugin", "_C_gguf_ops.so")
# bench.py's measurement kernels (streaming-read floor, MFMA peak): not part of the C ABI
PEAKS_SRC = os.path.join(CSRC, "bench", "peaks.hip")
PEAKS_OUT = os.path.join(HERE, "vllm_gguf_plugin", "libgguf_peaks.so")
DECODER_CSRC = os.path.join(CSRC, "decoder")
DECODER_OUT = os.path.join(HERE, "vllm_gguf_plugin", "libgguf_decoder.so")
DECODER_OPS_OUT = os.path.join(HERE, "vllm_gguf_plugin", "_C_gguf_decoder_ops.so")
CXX = os.environ.get("CXX", "g++")
ARCH = os.environ.get("GGUF_OFFLOAD_ARCH", "gfx950")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")

FLAGS = [
    f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC",
    # no packed fp32 instructions in device code (v_pk_*_f32)
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-fvisibility=hidden", "-Wall", "-Wno-unused-function", "-Wno-unused-variable",
]


def sources(csrc=CSRC):
    return sorted(os.path.join(csrc, f) for f in os.listdir(csrc) if f.endswith(".hip"))


def _compile(src):
    name = os.path.relpath(src, CSRC)[:-4].replace(os.sep, "_")
    obj = os.path.join(BUILD, name + ".o")
    cmd = [HIPCC, *FLAGS, "-c", src, "-o", obj]
    p = subprocess.run(cmd, capture_output=True, text=True)
    # hipcc's host pass warns about the device-only target feature: not an error
    noise = "is not a recognized feature for this target"
    err = "\n".join(l for l in (p.stderr or "").splitlines() if noise not in l)
    if p.returncode != 0:
        raise RuntimeError(f"hipcc failed on {src}:\n{err}")
    return obj, err


def _torch_flags():
    """Include / library directories and ABI flag of the installed PyTorch (ROCm build)."""
    import torch

    tdir = os.path.dirname(torch.__file__)
    inc = [os.path.join(tdir, "include"), os.path.join(tdir, "include", "torch", "csrc", "api", "include"),
           "/opt/rocm/include"]
    abi = int(torch._C._GLIBCXX_USE_CXX11_ABI)
    return inc, os.path.join(tdir, "lib"), abi


def _compile_ops(src):
    """A torch_ops.cpp -> its object (host C++ only)."""
    inc, _, abi = _torch_flags()
    obj = os.path.join(BUILD, os.path.relpath(src, CSRC)[:-4].replace(os.sep, "_") + ".o")
    cmd = [CXX, "-O2", "-std=c++17", "-fPIC", "-c", src, "-o", obj,
           "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1", f"-D_GLIBCXX_USE_CXX11_ABI={abi}",
           "-Wall", "-Wno-unused-function", *[f"-I{d}" for d in inc]]
    p = subprocess.run(cmd, capture_output=True, text=True)
    if p.returncode != 0:
        raise RuntimeError(f"{CXX} failed on {src}:\n{p.stderr}")
    return obj, p.stderr


def _link(objs, out):
    tmp = out + ".tmp"
    cmd = [HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", tmp, *objs]
    p = subprocess.run(cmd, capture_output=True, text=True)
    if p.returncode != 0:
        raise RuntimeError(f"link of {os.path.basename(out)} failed:\n{p.stderr}")
    os.replace(tmp, out)


def _link_ops(obj, lib, out):
    """An op registration, linked to the library `lib` next to it."""
    _, libdir, _ = _torch_flags()
    tmp = out + ".tmp"
    cmd = [CXX, "-shared", "-fPIC", "-o", tmp, obj, f"-L{os.path.dirname(out)}",
           f"-l{os.path.basename(lib)[3:-3]}",
           f"-L{libdir}", "-lc10", "-lc10_hip", "-ltorch", "-ltorch_cpu", "-ltorch_hip",
           "-L/opt/rocm/lib", "-lamdhip64", "-Wl,-rpath,$ORIGIN", f"-Wl,-rpath,{libdir}"]
    p = subprocess.run(cmd, capture_output=True, text=True)
    if p.returncode != 0:
        raise RuntimeError(f"link of {os.path.basename(out)} failed:\n{p.stderr}")
    os.replace(tmp, out)


def _build_peaks():
    """csrc/bench/peaks.hip -> libgguf_peaks.so (one step: compile and link)."""
    tmp = PEAKS_OUT + ".tmp"
    cmd = [HIPCC, *FLAGS, "-shared", PEAKS_SRC, "-o", tmp]
    p = subprocess.run(cmd, capture_output=True, text=True)
    if p.returncode != 0:
        raise RuntimeError(f"hipcc failed on {PEAKS_SRC}:\n{p.stderr}")
    os.replace(tmp, PEAKS_OUT)


def build(jobs: int = 8, verbose: bool = False) -> str:
    os.makedirs(BUILD, exist_ok=True)
    srcs, dec_srcs = sources(), sources(DECODER_CSRC)
    with cf.ThreadPoolExecutor(max_workers=max(1, min(jobs, len(srcs) + len(dec_srcs) + 3))) as ex:
        ops = [ex.submit(_compile_ops, os.path.join(d, "torch_ops.cpp")) for d in (CSRC, DECODER_CSRC)]
        peaks = ex.submit(_build_peaks)
        results = list(ex.map(_compile, srcs + dec_srcs))
        (ops_obj, ops_err), (dec_ops_obj, dec_ops_err) = (f.result() for f in ops)
        peaks.result()
    objs = [o for o, _ in results]
    if verbose:
        for err in [e for _, e in results] + [ops_err, dec_ops_err]:
            if err.strip():
                print(err, file=sys.stderr)
    _link(objs[:len(srcs)], OUT)
    _link(objs[len(srcs):], DECODER_OUT)
    _link_ops(ops_obj, OUT, OPS_OUT)
    _link_ops(dec_ops_obj, DECODER_OUT, DECODER_OPS_OUT)
    return OUT


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--jobs", type=int, default=min(8, os.cpu_count() or 1))
    ap.add_argument("-v", "--verbose", action="store_true")
    a = ap.parse_args()
    print(build(a.jobs, a.verbose))
