"""Builds libstrassen_hip.so (gfx950) from csrc/ with hipcc.

    python build.py            # rebuild what changed
    python build.py --force    # rebuild everything

The fused kernel is instantiated once per (element type, algorithm) pair; the units
plus the C-ABI front end compile in parallel and are linked into one shared library next to
this file.  Object files go to csrc/build/ (git-ignored).  _sthip_torch.so beside it holds the
torch side of the operators in csrc/sthip_torch.cpp (host code only, compiled by the host compiler);
where torch cannot be imported it is left out, and the library with its C ABI is built alone.
"""
from __future__ import annotations

import hashlib
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(CSRC, "build")
LIB = os.path.join(HERE, "libstrassen_hip.so")
TORCH_LIB = os.path.join(HERE, "_sthip_torch.so")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
ARCH = "gfx950"
# Packed fp32 VALU ops are disabled on purpose (hipcc's host pass prints a harmless note
# that it does not know the feature).
FLAGS = ["-O3", "-fPIC", "-std=c++17", f"--offload-arch={ARCH}",
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
         "-Wno-unused-command-line-argument", "-I", CSRC]


def _units():
    units = [("sthip_api.o", "sthip_api.hip", [])]
    for t in range(3):
        for a in range(3):
            units.append((f"sthip_inst_{t}_{a}.o", "sthip_inst.hip",
                          [f"-DSTHIP_INST_TYPE={t}", f"-DSTHIP_INST_ALGO={a}"]))
    for t in (1, 2):
        for a in range(3):
            units.append((f"sthip_inst2_{t}_{a}.o", "sthip_inst2.hip",
                          [f"-DSTHIP_INST_TYPE={t}", f"-DSTHIP_INST_ALGO={a}"]))
    for t in (1, 2):
        for a in range(3):
            units.append((f"sthip_inst3_{t}_{a}.o", "sthip_inst3.hip",
                          [f"-DSTHIP_INST_TYPE={t}", f"-DSTHIP_INST_ALGO={a}"]))
        units.append((f"sthip_inst4_{t}.o", "sthip_inst4.hip", [f"-DSTHIP_INST_TYPE={t}"]))
        units.append((f"sthip_inst5_{t}.o", "sthip_inst5.hip", [f"-DSTHIP_INST_TYPE={t}"]))
    units.append(("sthip_inst4_0.o", "sthip_inst4.hip", ["-DSTHIP_INST_TYPE=0"]))
    units.append(("sthip_inst6.o", "sthip_inst6.hip", []))
    units.append(("sthip_ops.o", "sthip_ops.hip", []))
    # the longest first
    return [(f"sthip_inst7_{t}_{part}.o", "sthip_inst7.hip", [f"-DSTHIP_INST_TYPE={t}", f"-DSTHIP_INST_PART={part}"])
            for part in range(3) for t in (1, 2, 0)] + units


def _digest(extra):
    h = hashlib.sha256()
    for name in sorted(os.listdir(CSRC)):
        path = os.path.join(CSRC, name)
        if os.path.isfile(path) and name != "sthip_torch.cpp":   # _torch_digest has that one
            h.update(name.encode())
            h.update(open(path, "rb").read())
    for hdr in ("strassen_hip.h", "strassen_hip_debug.h"):
        h.update(open(os.path.join(HERE, "..", "include", hdr), "rb").read())
    h.update(" ".join(FLAGS + extra).encode())
    return h.hexdigest()


def _compile(unit, force):
    obj, src, defs = unit
    out = os.path.join(OBJ, obj)
    stamp = out + ".sha"
    dig = _digest(defs)
    if not force and os.path.exists(out) and os.path.exists(stamp) and open(stamp).read() == dig:
        return obj, "cached"
    cmd = [HIPCC, *FLAGS, *defs, "-c", os.path.join(CSRC, src), "-o", out]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed for {obj}:\n{r.stderr[-4000:]}")
    open(stamp, "w").write(dig)
    return obj, "built"


def _torch_commands():
    """Compiling and linking the torch side (None without torch); it links against the library, whose symbols it needs and whose code it does not."""
    import sysconfig
    try:
        import torch
    except ImportError:
        return None
    from torch.utils.cpp_extension import include_paths, library_paths
    cxx, obj = os.environ.get("CXX", "g++"), os.path.join(OBJ, "sthip_torch.oo")
    compile_cmd = [cxx, "-O2", "-fPIC", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-DUSE_ROCM", "-DTORCH_API_INCLUDE_EXTENSION_H",
                   "-DTORCH_EXTENSION_NAME=_sthip_torch", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
    for d in include_paths("cuda"):
        compile_cmd += ["-isystem", d]
    compile_cmd += ["-I", sysconfig.get_paths()["include"], "-c", os.path.join(CSRC, "sthip_torch.cpp"), "-o", obj]
    link_cmd = [cxx, "-shared", obj, "-o", TORCH_LIB]
    for d in library_paths("cuda"):
        link_cmd += ["-L", d]
    link_cmd += ["-lc10", "-lc10_hip", "-ltorch", "-ltorch_cpu", "-ltorch_hip", "-ltorch_python", "-L", HERE, "-lstrassen_hip", "-Wl,-rpath,$ORIGIN"]
    return compile_cmd, link_cmd


def _run_torch(cmd, what):
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{what} sthip_torch.cpp failed:\n{r.stderr[-4000:]}")


def _torch_digest(commands):
    h = hashlib.sha256(repr(commands).encode())
    for path in (os.path.join(CSRC, "sthip_torch.cpp"), os.path.join(HERE, "..", "include", "strassen_hip.h")):
        h.update(open(path, "rb").read())
    return h.hexdigest()


def build(force: bool = False, jobs: int | None = None, verbose: bool = True) -> str:
    os.makedirs(OBJ, exist_ok=True)
    jobs = jobs or min(8, os.cpu_count() or 1)
    units = _units()
    commands = _torch_commands()
    torch_stamp, torch_digest = os.path.join(OBJ, "sthip_torch.sha"), commands and _torch_digest(commands)
    torch_new = commands and (force or not (os.path.exists(TORCH_LIB) and os.path.exists(torch_stamp) and open(torch_stamp).read() == torch_digest))
    with ThreadPoolExecutor(max_workers=jobs) as ex:
        torch_object = ex.submit(_run_torch, commands[0], "compiling") if torch_new else None
        results = list(ex.map(lambda u: _compile(u, force), units))
        if torch_object:
            torch_object.result()
    if verbose:
        print("objects:", ", ".join(f"{o}:{s}" for o, s in results))
    if force or not os.path.exists(LIB) or any(s == "built" for _, s in results):
        objs = [os.path.join(OBJ, u[0]) for u in units]
        cmd = [HIPCC, "-shared", "-fPIC", f"--offload-arch={ARCH}", *objs, "-o", LIB]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stderr[-4000:]}")
        if verbose:
            print("linked", LIB)
    if torch_new:
        _run_torch(commands[1], "linking")
        open(torch_stamp, "w").write(torch_digest)
    if verbose:
        print(TORCH_LIB, "built" if torch_new else "cached" if commands else "left out: torch cannot be imported")
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv)
