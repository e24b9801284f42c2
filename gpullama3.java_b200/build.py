"""Builds libb200llama.so in-tree with nvcc for sm_100a (no JIT cache: the .so travels with
the repo snapshot to the GPU box)."""
from __future__ import annotations

import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(CSRC, "libb200llama.so")
SOURCES = ["plan.cu", "operators.cu", "serving.cu"]


# Headers that plan.cu does not read: its object is not rebuilt for them.
OPERATOR_HEADERS = {"operators.cu": ("kv4.cuh", "kv4_chunk.cuh", "logprobs.cuh", "operator_util.cuh"),
                    "serving.cu": ("kv4.cuh", "kv4_chunk.cuh", "logprobs.cuh", "operator_util.cuh", "paged.cuh", "paged_chunk.cuh", "verify.cuh")}


def _deps(source: str | None = None):
    """What the library, or the object of one of its sources, is made from."""
    d = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    if source in OPERATOR_HEADERS:
        d = [f for f in d if os.path.basename(f) in (*OPERATOR_HEADERS[source], "common.cuh", "operators.h")]
    elif source is not None:
        d = [f for f in d if not any(os.path.basename(f) in h for h in OPERATOR_HEADERS.values())]
    d += [os.path.join(CSRC, f) for f in SOURCES if source in (None, f)]
    exp = os.path.join(CSRC, "experimental")
    if os.path.isdir(exp):
        d += [os.path.join(exp, f) for f in os.listdir(exp) if f.endswith((".cuh", ".h"))]
    d.append(os.path.join(HERE, "..", "include", "b200llama.h"))
    return d


NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
    # Java never contracts a*b+c; the kernels reproduce the CPU path's float order exactly.
    "-fmad=false", "-prec-div=true", "-prec-sqrt=true", "-ftz=false",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-pthread", "-Xptxas", "-v",
]


STAMP = os.path.join(CSRC, ".build_defines")


def _defines() -> list[str]:
    """Opt-in experimental code paths: B200_NVCC_DEFINES="B200_SEQSUM_V2[,...]" (default: none)."""
    return [d for d in os.environ.get("B200_NVCC_DEFINES", "").replace(",", " ").split() if d]


def needs_build() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    built_with = open(STAMP).read().split() if os.path.exists(STAMP) else []
    if built_with != _defines():
        return True
    return any(os.path.getmtime(d) > t for d in _deps()) or os.path.getmtime(__file__) > t


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and not needs_build():
        return LIB
    nvcc = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
    built_with = open(STAMP).read().split() if os.path.exists(STAMP) else []
    running, objects, log = [], [], ""
    for s in SOURCES:  # one compiler per source, at the same time
        obj = os.path.join(CSRC, os.path.splitext(s)[0] + ".o")
        objects.append(obj)
        stale = force or built_with != _defines() or not os.path.exists(obj) or any(os.path.getmtime(d) > os.path.getmtime(obj) for d in [*_deps(s), __file__])
        if stale:
            cmd = [nvcc, *NVCC_FLAGS, *[f"-D{d}" for d in _defines()], "-c", "-o", obj, os.path.join(CSRC, s)]
            running.append((s, obj, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
    failed = []
    for s, obj, p in running:
        out = p.communicate()[0]
        log += out
        if p.returncode != 0:
            failed.append(s)
            if os.path.exists(obj):
                os.remove(obj)
        if verbose or p.returncode != 0:
            sys.stderr.write(out)
    if not failed:
        r = subprocess.run([nvcc, *NVCC_FLAGS[:2], "-Xcompiler", "-fPIC", "-Xcompiler", "-pthread", "-shared", "-o", LIB, *objects, "-lcudart"], capture_output=True, text=True)
        if r.returncode != 0:
            sys.stderr.write(r.stdout + r.stderr)
            failed.append("libb200llama.so")
    if failed:
        raise RuntimeError(f"nvcc failed building {', '.join(failed)}")
    with open(os.path.join(CSRC, "ptxas.log"), "w") as f:
        f.write(log)
    with open(STAMP, "w") as f:
        f.write(" ".join(_defines()))
    return LIB


OPS_LIB = os.path.join(CSRC, "_b200ops.so")
OPS_SRC = os.path.join(CSRC, "torch_ops.cpp")


def _ops_command() -> list[str]:
    import sysconfig

    import torch
    from torch.utils import cpp_extension

    lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    # torch's own libstdc++ (the shared one), also where the compiler would link a static copy into a shared object: two of them do not share their streams' tables
    inc = [f"-I{d}" for d in [*cpp_extension.include_paths(), "/usr/local/cuda/include", sysconfig.get_paths()["include"]]]
    return [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-w", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", *inc, "-o", OPS_LIB, OPS_SRC,
            f"-L{CSRC}", "-l:libb200llama.so", f"-L{lib}", "-lc10", "-lc10_cuda", "-ltorch_cuda", "-ltorch_cpu", "-ltorch", "-ltorch_python", "-nostdlib++", "-l:libstdc++.so.6", "-lm", "-Wl,-rpath,$ORIGIN",
            f"-Wl,-rpath,{lib}"]


def build_operators(force: bool = False) -> str:
    """_b200ops.so: the operators on torch tensors (csrc/torch_ops.cpp), linked against libb200llama.so next to it."""
    hdr = os.path.join(HERE, "..", "include", "b200llama.h")
    if not force and os.path.exists(OPS_LIB) and os.path.getmtime(OPS_LIB) >= max(os.path.getmtime(f) for f in (OPS_SRC, hdr, __file__)):
        return OPS_LIB
    r = subprocess.run(_ops_command(), capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise RuntimeError("g++ failed building _b200ops.so")
    return OPS_LIB


TOK_LIB = os.path.join(CSRC, "libb200tok.so")
TOK_SRC = os.path.join(CSRC, "tokenizer.cpp")


def build_tokenizer(force: bool = False) -> str:
    """libb200tok.so: the native BPE tokenizer (CPU only, plain g++)."""
    hdr = os.path.join(HERE, "..", "include", "b200tok.h")
    if not force and os.path.exists(TOK_LIB) and os.path.getmtime(TOK_LIB) >= max(os.path.getmtime(TOK_SRC), os.path.getmtime(hdr)):
        return TOK_LIB
    cxx = os.environ.get("CXX", "g++")
    r = subprocess.run([cxx, "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-o", TOK_LIB, TOK_SRC], capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise RuntimeError("g++ failed building libb200tok.so")
    return TOK_LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
    print(build_operators(force="--force" in sys.argv))
    print(build_tokenizer(force="--force" in sys.argv))
