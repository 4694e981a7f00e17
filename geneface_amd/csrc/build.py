"""hipcc build of libgeneface_hip.so (gfx950 only, in-tree so it travels with the repo snapshot).

    python -m geneface_amd.csrc.build [--force]

Every translation unit is compiled to an object (cached by mtime of the source and the headers),
then linked into geneface_amd/csrc/libgeneface_hip.so.  No torch headers are involved: the library
is a plain C-ABI (include/geneface_hip.h) consumed through ctypes.
"""
import glob
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
OUT = os.path.join(HERE, "libgeneface_hip.so")
OBJ_DIR = os.path.join(HERE, "_obj")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
ARCH = "gfx950"

COMMON = ["-O3", "-std=c++17", "-fPIC", "-fvisibility=hidden", f"--offload-arch={ARCH}",
          "-fhip-fp32-correctly-rounded-divide-sqrt", "-Wall", "-Wno-unused-function"]


# EVERY translation unit is built WITHOUT the SLP vectoriser, i.e. without packed-FP32 VALU instructions (v_pk_fma_f32 / v_pk_mul_f32 /
# v_pk_add_f32).  In k_head_phase<true> the low half of one v_pk_fma_f32 of the 2-D grid lookup -- the one fed by a broadcast-form
# v_pk_mul_f32 ... op_sel:[0,1] op_sel_hi:[0,1] -- intermittently lost its product in lanes 32..63 whenever two workgroups shared a CU
# (NOTES.md 4.7, tools/fast_diag.py).  The mechanism is not established, so since round 3 the instruction class is banned from the whole
# library, not just from the kernel it was caught in (encoders.hip's k_encode8<2> held two instances of exactly that pair):
# tests/test_build_invariants.py disassembles every code object and asserts the count is zero.  Scalar FMAs compute the same values (the
# packed form was only ever two independent FMAs); measured cost: head fp32 719 vs 717 fps, fast tier 1890 vs 1845 fps (round 2, A/B on
# one box), stand-alone ops and the training step within noise (round 3, profiles/round3/).
COMMON.append("-fno-slp-vectorize")
PER_FILE = {}


def sources():
    return sorted(glob.glob(os.path.join(HERE, "*.hip")) + glob.glob(os.path.join(HERE, "*.cpp")))


def headers():
    return sorted(glob.glob(os.path.join(HERE, "*.hpp")) + glob.glob(os.path.join(HERE, "*.inc")) + [os.path.join(HERE, "..", "..", "include", "geneface_hip.h")])


# The operators of a training step (train/: AdamW, block-scaled 8-bit products) are translation units of the same library with a public header of
# their own.  Nothing above includes from there and they include only common.hpp, so neither side's edits rebuild the other, and the digest
# below, which stamps measurements of the frame and field kernels, does not move with them.  They are compiled without the packed-FP32 feature:
# the same ban as -fno-slp-vectorize for code that is written on vectors.
TRAIN_DIR = os.path.join(HERE, "train")
TRAIN_FLAGS = ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", "-Wno-unknown-warning-option"]


HOST_SOURCE = os.path.join(TRAIN_DIR, "host.cpp")      # the one file that includes torch's headers: a Python module of its own
HOST_OUT = os.path.join(HERE, "_train_host.so")


def train_sources():
    return sorted({*glob.glob(os.path.join(TRAIN_DIR, "*.hip")), *glob.glob(os.path.join(TRAIN_DIR, "*.cpp"))} - {HOST_SOURCE})


def train_headers():
    return sorted(glob.glob(os.path.join(TRAIN_DIR, "*.hpp")) + [os.path.join(HERE, "common.hpp"), os.path.join(HERE, "..", "..", "include", "geneface_train_hip.h")])


def source_digest() -> str:
    """sha256 (16 hex digits) over every source, header and table of the library's frame, field and stand-alone kernels plus the compile flags: what a measurement taken on
    one tree stamps itself with (tools/pmc_summary.py) and what bench.py compares a committed PMC summary against (`traffic_stale`).
    Content, not mtimes: a snapshot on the GPU box or a fresh checkout has new mtimes and the same digest."""
    import hashlib
    h = hashlib.sha256()
    for path in sorted(sources() + headers()):
        h.update(os.path.basename(path).encode())
        with open(path, "rb") as f:
            h.update(f.read())
    h.update(" ".join(COMMON).encode())
    return h.hexdigest()[:16]


def _run(cmd, out, what):
    """Run a compiler with `-o out`, completely or not at all: other processes (ranks that start together) load and link what lies at `out`."""
    part = f"{out}.{os.getpid()}.part"
    try:
        r = subprocess.run([*cmd, "-o", part], capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"{what}:\n{r.stdout}\n{r.stderr}")
        os.replace(part, out)
    finally:
        if os.path.exists(part):
            os.remove(part)
    return r


def _compile(src, force, extra=(), obj_dir=OBJ_DIR, drop=()):
    obj = os.path.join(obj_dir, os.path.basename(src) + ".o")
    train = os.path.dirname(src) == TRAIN_DIR
    if train:
        obj_dir = os.path.join(obj_dir, "train")
        obj = os.path.join(obj_dir, os.path.basename(src) + ".o")
        extra = (*extra, *TRAIN_FLAGS)
    newest = max(os.path.getmtime(p) for p in [src, __file__, *(train_headers() if train else headers())])
    if not force and os.path.exists(obj) and os.path.getmtime(obj) >= newest:
        return obj, False
    cmd = [HIPCC, *[f for f in COMMON if f not in drop], *PER_FILE.get(os.path.basename(src), ()), *extra, "-x", "hip", "-c", src, "-I", HERE,
           "-I", os.path.join(HERE, "..", "..", "include")]
    r = _run(cmd, obj, f"hipcc failed for {src}")
    said = "".join(line for line in r.stderr.splitlines(True) if "packed-fp32-ops" not in line)      # the host pass does not know the feature
    if said.strip():
        sys.stderr.write(said)
    return obj, True


def build_host(force: bool = False) -> str:
    """_train_host.so: the operators' argument checks and calls in C++ against this interpreter's torch (lib.host() loads it)."""
    newest = max(os.path.getmtime(p) for p in [HOST_SOURCE, __file__, *train_headers()])
    if not force and os.path.exists(HOST_OUT) and os.path.getmtime(HOST_OUT) >= newest:
        return HOST_OUT
    import sysconfig
    import torch
    home = os.path.join(os.path.dirname(torch.__file__))
    inc = [os.path.join(home, "include"), os.path.join(home, "include", "torch", "csrc", "api", "include"), sysconfig.get_paths()["include"],
           "/opt/rocm/include", os.path.join(HERE, "..", "..", "include")]
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-DTORCH_EXTENSION_NAME=_train_host", *[f"-I{i}" for i in inc], HOST_SOURCE,
           f"-L{os.path.join(home, 'lib')}", "-ltorch_python", "-ltorch_cpu", "-lc10_hip", "-lc10"]
    _run(cmd, HOST_OUT, f"g++ failed for {HOST_SOURCE}")
    return HOST_OUT


def build(force: bool = False, verbose: bool = False, trace: bool = False, variant: str = None, defines=(), drop_flags=()) -> str:
    """trace=True builds the instrumented variant (-DGF_TRACE: per-round s_memtime timeline of the head kernel, read by
    tools/trace_head.py) into libgeneface_hip_trace.so; the product library never contains the instrumentation.
    variant="x", defines=("-DFOO",) builds an experiment library libgeneface_hip_x.so (A/B runs select it with GF_HIP_LIB);
    drop_flags=("-fno-slp-vectorize",) removes flags of COMMON for that variant (tools/pk_regress.py: the packed-FP32 probe build)."""
    if drop_flags and not variant:
        raise ValueError("drop_flags is for experiment variants only: the product library is always built with COMMON")
    tag = "trace" if trace else variant
    obj_dir = OBJ_DIR + (f"_{tag}" if tag else "")
    out = OUT.replace(".so", f"_{tag}.so") if tag else OUT
    extra = (("-DGF_TRACE",) if trace else ()) + tuple(defines)
    os.makedirs(os.path.join(obj_dir, "train"), exist_ok=True)
    with ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as ex:
        host = ex.submit(build_host, force) if not tag else None
        results = list(ex.map(lambda s: _compile(s, force, extra, obj_dir, tuple(drop_flags)), [*sources(), *train_sources()]))
    objs = [o for o, _ in results]
    if force or any(ch for _, ch in results) or not os.path.exists(out):
        cmd = [HIPCC, "-shared", "-fPIC", f"--offload-arch={ARCH}", *objs, "-lz", "-lpthread"]   # zlib: the PNG frame writer (png_writer.cpp)
        _run(cmd, out, "link failed")
        if verbose:
            print("linked", out)
    if host is not None and host.exception() is not None:      # the C ABI needs neither g++ nor Python's and torch's headers: lib.host() says what is missing when it is asked for
        sys.stderr.write(f"geneface_amd: {out} is built, the Python side of the training operators is not: {host.exception()}\n")
        if os.path.exists(HOST_OUT):      # of older sources: it must not be loaded beside this library
            os.remove(HOST_OUT)
    return out


if __name__ == "__main__":
    _variant = sys.argv[sys.argv.index("--variant") + 1] if "--variant" in sys.argv else None
    _defs = tuple(a for a in sys.argv[1:] if a.startswith(("-D", "-f")))   # e.g. --variant slp -fslp-vectorize for an A/B library
    print(build(force="--force" in sys.argv, verbose=True, trace="--trace" in sys.argv, variant=_variant, defines=_defs))
