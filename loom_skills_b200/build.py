"""Build liblk.so in-tree with nvcc for sm_100a (no torch extension machinery: the library is a plain C ABI)."""
import os
import re
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "liblk.so")
SOURCES = ["lk_api.cu", "lk_dequant.cu", "lk_mv.cu", "lk_mvq8.cu","lk_gemm.cu", "lk_mxfp4.cu", "lk_moe.cu", "lk_peer.cu",
           "lk_noalloc.cu", "lk_mvmx.cu", "lk_mvg.cu", "lk_moeq8.cu", "lk_mvq8g.cu", "lk_norm.cu",
           "lk_mvx.cu", "lk_mv1.cu", "lk_gemmx.cu"]
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-Xcompiler", "-fPIC",
         "--expt-relaxed-constexpr", "-Xptxas", "-warn-spills"]


# Registers a thread that a kernel must be launched with at least: k_mvx's consumer warps take theirs from the launch's
# total, and a smaller one would leave them waiting (lk_mvx.cu, kLaunchRegs).
LAUNCH_REGISTERS = {"lk_mvx.cu": ("k_mvx", 96)}


def check_registers(src, ptxas):
    """Holds the registers that ptxas -v reports for the kernels of `src` against LAUNCH_REGISTERS."""
    if src not in LAUNCH_REGISTERS:
        return
    kernel, least = LAUNCH_REGISTERS[src]
    names = re.findall(r"Compiling entry function '(\w+)'", ptxas)
    used = [int(n) for n in re.findall(r"Used (\d+) registers", ptxas)]
    if len(names) != len(used) or not any(kernel in n for n in names):
        raise RuntimeError(f"{src}: ptxas reported no registers of {kernel}")
    few = [n for n, r in zip(names, used) if kernel in n and r < least]
    if few:
        raise RuntimeError(f"{src}: fewer than {least} registers a thread in {', '.join(few)}")


def _write_iq3s_grid(bdir):
    """The IQ3_S codebook (512 entries of four odd magnitudes 1..15; ggml's iq3s_grid, which the reference embeds in
    quant_values.loom:5-6) as the device table lk_formats.cuh includes: taken from gguf-py 0.19.0's IQ3_S grid (the
    format's pinned definition; gguf-py is the reference's dequantiser) at build time, one little-endian u32 per entry
    (byte i = magnitude i), so no copy of the table is kept in this tree."""
    from gguf.quants import IQ3_S
    IQ3_S.init_grid()
    g = IQ3_S.grid.reshape(512, 4).astype(int)
    assert set(g.reshape(-1).tolist()) <= set(range(1, 16, 2))
    words = [int(r[0] | (r[1] << 8) | (r[2] << 16) | (r[3] << 24)) for r in g]
    body = ",\n".join(", ".join(f"0x{w:08x}u" for w in words[i:i + 8]) for i in range(0, 512, 8))
    text = ("// generated by build.py from gguf-py's IQ3_S grid: do not edit\n"
            "static __device__ __align__(16) const unsigned int kIq3sGrid[512] = {\n" + body + "};\n")
    path = os.path.join(bdir, "lk_iq3s_grid.inc")
    if not os.path.exists(path) or open(path).read() != text:
        with open(path, "w") as f:
            f.write(text)


def _stale():
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    deps = [os.path.join(CSRC, f) for f in os.listdir(CSRC)] + [os.path.join(HERE, "..", "include", "lk.h")]
    return any(os.path.getmtime(d) > t for d in deps if os.path.exists(d))


def build(force=False, verbose=False, jobs=None):
    """Compile every .cu under csrc/ to an object, then link liblk.so. Objects go to csrc/_build (git-ignored)."""
    if not force and not _stale():
        return LIB
    bdir = os.path.join(CSRC, "_build")
    os.makedirs(bdir, exist_ok=True)
    _write_iq3s_grid(bdir)
    procs = []
    objs = []
    for src in SOURCES:
        obj = os.path.join(bdir, src.replace(".cu", ".o"))
        objs.append(obj)
        check = ["-Xptxas", "-v"] if src in LAUNCH_REGISTERS else []
        cmd = [NVCC, *FLAGS, *check, "-I", bdir, "-c", os.path.join(CSRC, src), "-o", obj]
        if verbose:
            print(" ".join(cmd), flush=True)
        procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
    failed = []
    for src, p in procs:
        out, _ = p.communicate()
        if verbose or p.returncode:
            sys.stdout.write(out)
        if p.returncode:
            failed.append(src)
        else:
            check_registers(src, out)
    if failed:
        raise RuntimeError("nvcc failed for " + ", ".join(failed))
    tmp = LIB + ".tmp"
    cmd = [NVCC, "-shared", "-gencode", "arch=compute_100a,code=sm_100a", *objs, "-o", tmp, "-lcudart"]
    subprocess.check_call(cmd)
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
