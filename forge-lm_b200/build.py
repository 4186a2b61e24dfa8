"""Builds libforge_b200.so in-tree for sm_100a (B200).

Steps:
  1. gen_expf_fixups (host gcc) -> csrc/generated/expf_fixups.inc: the inputs
     where the host libm expf differs from the correctly rounded exponential
     (the on-device sampler reproduces the host expf bit for bit).
  2. nvcc -gencode arch=compute_100a,code=sm_100a: one object per .cu file
     (in csrc/generated/), linked to libforge_b200.so.
  3. g++ csrc/serving_binding.cpp -> _serving.so, the serving operators' calls
     on torch tensors, where torch is installed.
No fast-math: the sampler's division and exponentials must round as IEEE.
"""
from __future__ import annotations

import hashlib
import importlib.metadata
import importlib.util
import json
import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
GEN = os.path.join(CSRC, "generated")
OBJ = GEN  # the objects lie with the other generated files
LIB = os.path.join(HERE, "libforge_b200.so")
BINDING = os.path.join(HERE, "_serving.so")
ROOT = os.path.dirname(HERE)

NVCC_FLAGS = [
    "-O3", "-std=c++17", "-lineinfo",
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-Xcompiler", "-fPIC,-O3,-fvisibility=hidden",
    "--expt-relaxed-constexpr",
    "-Xptxas", "-warn-spills",
]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def _newer(target: str, sources: list[str]) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(s) > t for s in sources)


def gen_fixups(verbose: bool = False) -> str:
    os.makedirs(GEN, exist_ok=True)
    src = os.path.join(CSRC, "gen_expf_fixups.c")
    out = os.path.join(GEN, "expf_fixups.inc")
    if not _newer(out, [src]):
        return out
    exe = os.path.join(GEN, "gen_expf_fixups")
    subprocess.run(["gcc", "-O2", "-fopenmp", "-ffp-contract=off", src, "-o", exe, "-lm"], check=True)
    r = subprocess.run([exe, out], check=True, capture_output=True, text=True)
    if verbose:
        print(r.stdout.strip())
    os.remove(exe)
    return out


def _flags() -> list[str]:
    """nvcc flags; FORGE_B200_PHASE_TRACE=1 adds the persistent kernel's
    per-phase stamps (a diagnostic build: the stamps cost throughput)."""
    flags = list(NVCC_FLAGS)
    if os.environ.get("FORGE_B200_PHASE_TRACE") == "1":
        flags.append("-DFB2_MK_PHASE_TRACE")
    return flags


def _sources() -> list[str]:
    sources = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh", ".hpp"))]
    sources += [os.path.join(ROOT, "include", h) for h in ("forge_b200.h", "forge_b200_testing.h")]
    sources.append(os.path.join(GEN, "expf_fixups.inc"))
    return sorted(sources)


def source_fingerprint(flags: list[str], sources: list[str]) -> str:
    """SHA-256 of the nvcc flags and every source file (path and contents):
    names the build independently of the binary, which nvcc does not
    reproduce byte for byte."""
    h = hashlib.sha256(" ".join(flags).encode())
    for path in sources:
        h.update(os.path.relpath(path, ROOT).encode())
        with open(path, "rb") as f:
            h.update(f.read())
    return h.hexdigest()


def stamp_path(lib: str = LIB) -> str:
    """The JSON beside the library: the flags and source fingerprint it was built from."""
    return lib + ".flags"


def read_stamp(lib: str = LIB) -> dict:
    try:
        with open(stamp_path(lib)) as f:
            return json.load(f)
    except (OSError, ValueError):
        return {}


def _compile(unit: str, flags: list[str], force: bool, verbose: bool) -> str:
    """One translation unit's object file, compiled again where the unit or a
    file it included the last time (nvcc's dependency list) is newer."""
    obj = os.path.join(OBJ, os.path.basename(unit) + ".o")
    deps = obj + ".d"
    try:
        with open(deps) as f:
            listed = f.read().replace("\\\n", " ").split(":", 1)[1].split()
        stale = _newer(obj, [unit] + [d for d in listed if d.startswith(ROOT)])
    except (OSError, IndexError):
        stale = True
    if force or stale:
        cmd = [_nvcc(), *flags, "-c", "-MD", "-MF", deps, "-o", obj, unit]
        if verbose:
            print(" ".join(cmd))
        subprocess.run(cmd, check=True)
    return obj


def _binding_command(out: str) -> list[str]:
    """g++ for the Python extension _serving: torch's headers, the library
    beside it (found through the extension's own folder)."""
    import torch
    from torch.utils import cpp_extension

    includes = cpp_extension.include_paths() + [sysconfig.get_paths()["include"], "/usr/local/cuda/include"]
    libs = os.path.join(os.path.dirname(torch.__file__), "lib")
    return ["g++", "-O2", "-std=c++20", "-shared", "-fPIC", "-fvisibility=hidden", "-w",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *[f"-isystem{i}" for i in includes],
            os.path.join(CSRC, "serving_binding.cpp"), "-o", out, f"-L{HERE}", "-l:libforge_b200.so", f"-L{libs}",
            "-ltorch_python", "-ltorch_cuda", "-ltorch_cpu", "-lc10_cuda", "-lc10", "-Wl,-rpath,$ORIGIN"]


def build_binding(verbose: bool = False, force: bool = False) -> str | None:
    """The extension module, compiled again where its source or the C header is
    newer or it was built for another torch or Python (the JSON beside it says
    for which).  None without torch: the C library does not need it."""
    if importlib.util.find_spec("torch") is None:
        print("torch is not installed: the serving operators' Python calls (_serving.so) are not built")
        return None
    sources = [os.path.join(CSRC, "serving_binding.cpp"), os.path.join(ROOT, "include", "forge_b200.h")]
    made_for = {"torch": importlib.metadata.version("torch"), "python": sysconfig.get_config_var("EXT_SUFFIX")}
    if force or _newer(BINDING, sources) or read_stamp(BINDING) != made_for:
        cmd = _binding_command(BINDING + ".tmp")
        if verbose:
            print(" ".join(cmd))
        subprocess.run(cmd, check=True)
        os.replace(BINDING + ".tmp", BINDING)
        with open(stamp_path(BINDING), "w") as f:
            json.dump(made_for, f)
    return BINDING


def build(verbose: bool = False, force: bool = False) -> str:
    gen_fixups(verbose)
    sources = _sources()
    flags = _flags()
    same_flags = read_stamp().get("flags") == flags
    if not force and same_flags and not _newer(LIB, sources):
        build_binding(verbose)
        return LIB
    os.makedirs(OBJ, exist_ok=True)
    units = [os.path.join(CSRC, f) for f in sorted(os.listdir(CSRC)) if f.endswith(".cu")]
    with ThreadPoolExecutor(len(units)) as pool:  # each runs an nvcc of its own
        objects = list(pool.map(lambda u: _compile(u, flags, force or not same_flags, verbose), units))
    subprocess.run([_nvcc(), *flags, "-shared", "-o", LIB + ".tmp", *objects], check=True)
    os.replace(LIB + ".tmp", LIB)
    with open(stamp_path(), "w") as f:
        json.dump({"flags": flags, "sources_sha256": source_fingerprint(flags, sources)}, f)
    build_binding(verbose, force)
    return LIB


if __name__ == "__main__":
    print(build(verbose=True, force="--force" in sys.argv))
