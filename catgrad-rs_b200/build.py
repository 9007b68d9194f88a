"""nvcc recipe for libcatgrad_cuda.so (sm_100a only), built in-tree beside this file."""
from __future__ import annotations

import concurrent.futures as cf
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(HERE, "build")
LIB = os.path.join(HERE, "libcatgrad_cuda.so")
SOURCES = ["runtime.cu", "eager.cu", "gemm_tc.cu", "gemm_tcp.cu", "gemm_tcp2.cu", "gemm_dec.cu", "fused.cu", "attention.cu", "attention_fa.cu", "attn_decode.cu", "decoder.cu", "decoder_mixed.cu", "mixed_rows.cu", "depth_rows.cu", "lru.cu", "rows_attn.cu", "latent.cu", "latent_decode.cu", "recurrent.cu", "recurrent_chunk.cu", "channel_chunk.cu", "decode_resident.cu", "safetensors.cu", "lazy.cu", "comm.cu", "moe.cu", "noalloc.cu", "paged.cu", "paged_attn.cu", "paged_fa.cu", "paged_dec.cu", "beam.cu"]
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
    "-ccbin", "/usr/bin/g++", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
]


def _stale(target: str, deps: list[str]) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def build(verbose: bool = False, force: bool = False) -> str:
    os.makedirs(OBJ, exist_ok=True)
    headers = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".h", ".cuh"))]
    headers.append(os.path.join(HERE, "..", "include", "catgrad_cuda.h"))
    srcs = [s for s in SOURCES if os.path.exists(os.path.join(CSRC, s))]
    jobs = []
    for s in srcs:
        src = os.path.join(CSRC, s)
        obj = os.path.join(OBJ, s.replace(".cu", ".o"))
        if force or _stale(obj, [src] + headers):
            cmd = [NVCC, *FLAGS, "-c", src, "-o", obj]
            if verbose:
                cmd.insert(1, "-Xptxas")
                cmd.insert(2, "-v")
            jobs.append((s, cmd))

    def run(job):
        name, cmd = job
        r = subprocess.run(cmd, capture_output=True, text=True)
        return name, r.returncode, r.stdout + r.stderr

    failed = False
    with cf.ThreadPoolExecutor(max_workers=8) as ex:
        for name, rc, out in ex.map(run, jobs):
            if verbose or rc != 0:
                sys.stderr.write(f"--- {name}\n{out}\n")
            failed |= rc != 0
    if failed:
        raise RuntimeError("nvcc failed")
    objs = [os.path.join(OBJ, s.replace(".cu", ".o")) for s in srcs]
    if jobs or not os.path.exists(LIB):
        # link beside the library and rename: a reader (a process loading it, a copy of the tree)
        # sees the old file or the new one, never a partly written one
        tmp = LIB + ".tmp"
        cmd = [NVCC, "-shared", "-ccbin", "/usr/bin/g++", "-o", tmp, *objs, "-ldl"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError("link failed:\n" + r.stdout + r.stderr)
        os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv, force="-f" in sys.argv))
