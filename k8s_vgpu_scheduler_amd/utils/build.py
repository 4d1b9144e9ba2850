"""Native build driver: the shim, the governor code object and the HIP op library.

Everything is built IN-TREE under ``k8s_vgpu_scheduler_amd/lib`` (shipped to
the GPU box with the repo snapshot) for gfx950 only.  Builds are incremental
(mtime based) and serialised with a file lock so parallel test workers do not
race.  Reference counterpart: ``docker/Dockerfile.hamicore`` builds libvgpu.so
with CMake (``bash ./build.sh``); here the same role is played by this module,
called from ``__graft_entry__.build()`` and ``python -m k8s_vgpu_scheduler_amd.utils.build``.
"""

from __future__ import annotations

import fcntl
import os
import shutil
import subprocess
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parents[2]
PKG = ROOT / "k8s_vgpu_scheduler_amd"
LIB = PKG / "lib"
CSRC = ROOT / "csrc"
BUILD = ROOT / "build"
ROCM = Path(os.environ.get("ROCM_PATH", "/opt/rocm"))
ARCH = "gfx950"
# No packed fp32 vector instructions in device code: some of their forms have given wrong results now and then.
# (The host pass warns that it does not know the feature: harmless.)
NO_PACKED_FP32 = ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]

SHIM_SO = LIB / "libmivgpu.so"
BOARDD = LIB / "mivgpu-boardd"
OPS_SO = LIB / "libmivgpu_ops.so"
GOV_HSACO = BUILD / "governor.hsaco"
GOV_INC = BUILD / "gen" / "governor_hsaco.inc"
MOCK_DIR = BUILD / "mockhip"
MOCK_LIB = MOCK_DIR / "libamdhip64.so"
MOCK_DRIVER = MOCK_DIR / "shim_driver"
MOCK_ROCTX = MOCK_DIR / "libmockroctx.so"
MOCK_SMI = MOCK_DIR / "libmocksmi.so"


def _hipcc() -> str:
    p = ROCM / "bin" / "hipcc"
    return str(p) if p.exists() else (shutil.which("hipcc") or "hipcc")


def _stale(out: Path, deps) -> bool:
    if not out.exists():
        return True
    t = out.stat().st_mtime
    return any(Path(d).stat().st_mtime > t for d in deps)


def _run(cmd, cwd=None):
    r = subprocess.run(cmd, cwd=cwd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"build command failed ({r.returncode}): {' '.join(map(str, cmd))}\n{r.stdout}")
    return r.stdout


class _Lock:
    def __init__(self, name: str):
        BUILD.mkdir(parents=True, exist_ok=True)
        self.path = BUILD / f".{name}.lock"

    def __enter__(self):
        self.fd = open(self.path, "w")
        fcntl.flock(self.fd, fcntl.LOCK_EX)
        return self

    def __exit__(self, *a):
        fcntl.flock(self.fd, fcntl.LOCK_UN)
        self.fd.close()


def build_governor() -> Path:
    """Compile governor.hip to a gfx950 code object and embed it as a C array."""
    src = CSRC / "kernels" / "governor.hip"
    if _stale(GOV_INC, [src, Path(__file__)]):
        GOV_INC.parent.mkdir(parents=True, exist_ok=True)
        _run([_hipcc(), f"--offload-arch={ARCH}", *NO_PACKED_FP32, "--genco", "-O3", "-o", str(GOV_HSACO), str(src)])
        data = GOV_HSACO.read_bytes()
        lines = []
        for i in range(0, len(data), 24):
            lines.append(",".join(str(b) for b in data[i:i + 24]))
        GOV_INC.write_text(
            "// generated by k8s_vgpu_scheduler_amd/utils/build.py from csrc/kernels/governor.hip\n"
            f"alignas(4096) static const unsigned char mivgpu_governor_hsaco[{len(data)}] = {{\n"
            + ",\n".join(lines) + "\n};\n")
    return GOV_INC


SHIM_FLOOR = CSRC / "shim" / "glibc_floor.h"
# The shim's ABI floor (glibc_floor.h): no libc import newer than this, no
# shared libstdc++/libgcc_s; libpthread.so.0 / libdl.so.2 NEEDED so glibc < 2.34
# (where pthread_* / dl* live there) resolves the old-versioned imports.
SHIM_GLIBC_FLOOR = (2, 17)
SHIM_LINK = ["-static-libstdc++", "-static-libgcc", "-Wl,--no-as-needed", "-l:libpthread.so.0", "-l:libdl.so.2",
             "-Wl,--as-needed"]


def build_shim() -> Path:
    srcs = [CSRC / "shim" / "mivgpu_shim.cpp", CSRC / "shim" / "mivgpu_shim.map",
            CSRC / "include" / "mivgpu" / "shared_region.h", SHIM_FLOOR, CSRC / "shim" / "board.h"]
    with _Lock("shim"):
        inc = build_governor()
        if _stale(SHIM_SO, srcs + [inc, Path(__file__)]):
            LIB.mkdir(parents=True, exist_ok=True)
            cxx = shutil.which("g++") or "c++"
            tmp = SHIM_SO.with_suffix(".so.tmp")
            _run([cxx, "-std=c++17", "-O2", "-g", "-fPIC", "-shared", "-fvisibility=hidden",
                  "-D__HIP_PLATFORM_AMD__", "-DMIVGPU_GLIBC_FLOOR", "-include", str(SHIM_FLOOR), f"-I{ROCM / 'include'}",
                  f"-I{CSRC / 'include'}", f"-I{inc.parent}", str(srcs[0]),
                  f"-Wl,--version-script={srcs[1]}", "-Wl,-z,now", *SHIM_LINK,
                  "-o", str(tmp)])
            os.replace(tmp, SHIM_SO)
    return SHIM_SO


def build_boardd() -> Path:
    """The node's share-board owner (csrc/shim/boardd.cpp): one wave-occupancy
    sampler per GPU, started by the monitor."""
    srcs = [CSRC / "shim" / "boardd.cpp", CSRC / "shim" / "board.h", CSRC / "include" / "mivgpu" / "shared_region.h"]
    with _Lock("boardd"):
        if _stale(BOARDD, srcs + [Path(__file__)]):
            LIB.mkdir(parents=True, exist_ok=True)
            cxx = shutil.which("g++") or "c++"
            tmp = BOARDD.with_suffix(".tmp")
            _run([cxx, "-std=c++17", "-O2", "-g", "-Wall", f"-I{CSRC / 'include'}", f"-I{CSRC / 'shim'}",
                  str(srcs[0]), "-static-libstdc++", "-static-libgcc", "-o", str(tmp)])
            os.replace(tmp, BOARDD)
    return BOARDD


DIAG_DIR = BUILD / "diag"


def build_hook_diag(level: int) -> Path:
    """Cost-attribution variant of the shim's launch path (MIVGPU_HOOK_DIAG,
    mivgpu_shim.cpp): 1 = forward only, 2 = + guard and lazy init, 3 = +
    launch counters.  Measurement only: built under build/diag, never
    installed or mounted into a container."""
    if level not in (1, 2, 3):
        raise ValueError(level)
    out = DIAG_DIR / f"libmivgpu_diag{level}.so"
    srcs = [CSRC / "shim" / "mivgpu_shim.cpp", CSRC / "shim" / "mivgpu_shim.map",
            CSRC / "include" / "mivgpu" / "shared_region.h", SHIM_FLOOR]
    with _Lock("diag"):
        inc = build_governor()
        if _stale(out, srcs + [inc, Path(__file__)]):
            DIAG_DIR.mkdir(parents=True, exist_ok=True)
            cxx = shutil.which("g++") or "c++"
            _run([cxx, "-std=c++17", "-O2", "-fPIC", "-shared", "-fvisibility=hidden", "-D__HIP_PLATFORM_AMD__",
                  "-DMIVGPU_GLIBC_FLOOR", f"-DMIVGPU_HOOK_DIAG={level}", "-include", str(SHIM_FLOOR),
                  f"-I{ROCM / 'include'}", f"-I{CSRC / 'include'}", f"-I{inc.parent}", str(srcs[0]),
                  f"-Wl,--version-script={srcs[1]}", "-Wl,-z,now", *SHIM_LINK, "-o", str(out)])
    return out


VARIANT_DIR = BUILD / "variants"


def build_shim_variant(name: str, defines: list[str]) -> Path:
    """The shim built with extra -D defines under build/variants (A/B runs of
    compile-time defaults; measurement only, never installed)."""
    out = VARIANT_DIR / f"libmivgpu_{name}.so"
    srcs = [CSRC / "shim" / "mivgpu_shim.cpp", CSRC / "shim" / "mivgpu_shim.map",
            CSRC / "include" / "mivgpu" / "shared_region.h", SHIM_FLOOR]
    with _Lock("variants"):
        inc = build_governor()
        if _stale(out, srcs + [inc, Path(__file__)]):
            VARIANT_DIR.mkdir(parents=True, exist_ok=True)
            cxx = shutil.which("g++") or "c++"
            _run([cxx, "-std=c++17", "-O2", "-g", "-fPIC", "-shared", "-fvisibility=hidden", "-D__HIP_PLATFORM_AMD__",
                  "-DMIVGPU_GLIBC_FLOOR", *[f"-D{d}" for d in defines], "-include", str(SHIM_FLOOR),
                  f"-I{ROCM / 'include'}", f"-I{CSRC / 'include'}", f"-I{inc.parent}", str(srcs[0]),
                  f"-Wl,--version-script={srcs[1]}", "-Wl,-z,now", *SHIM_LINK, "-o", str(out)])
    return out


def build_mock() -> tuple[Path, Path]:
    """Mock HIP runtime + driver for the CPU test-suite (never shipped)."""
    d = CSRC / "mockhip"
    with _Lock("mock"):
        MOCK_DIR.mkdir(parents=True, exist_ok=True)
        cxx = shutil.which("g++") or "c++"
        common = ["-std=c++17", "-O1", "-g", "-fPIC", "-D__HIP_PLATFORM_AMD__",
                  f"-I{ROCM / 'include'}"]
        if _stale(MOCK_LIB, [d / "mock_amdhip.cpp", d / "mock_amdhip.map"]):
            # -Bsymbolic: like the real runtime, the mock's own references
            # (hipGetProcAddress' table) name its own functions, never an interposer's
            _run([cxx, *common, "-shared", "-fvisibility=hidden", str(d / "mock_amdhip.cpp"),
                  f"-Wl,--version-script={d / 'mock_amdhip.map'}", "-Wl,-soname,libamdhip64.so", "-Wl,-Bsymbolic",
                  "-o", str(MOCK_LIB)])
        if _stale(MOCK_DRIVER, [d / "shim_driver.cpp", MOCK_LIB]):
            _run([cxx, *common, str(d / "shim_driver.cpp"), f"-L{MOCK_DIR}", "-lamdhip64", "-ldl",
                  "-Wl,--disable-new-dtags", f"-Wl,-rpath,{MOCK_DIR}", "-o", str(MOCK_DRIVER)])
        if _stale(MOCK_SMI, [d / "mock_smi.cpp"]):
            _run([cxx, *common, "-shared", "-fvisibility=hidden", str(d / "mock_smi.cpp"), "-o", str(MOCK_SMI)])
        if _stale(MOCK_ROCTX, [d / "mock_roctx.cpp"]):
            _run([cxx, *common, "-shared", "-fvisibility=hidden", str(d / "mock_roctx.cpp"), "-o", str(MOCK_ROCTX)])
    return MOCK_LIB, MOCK_DRIVER


SAN_DIR = BUILD / "san"
SAN_RUNTIME = {"address": "libasan.so.6", "thread": "libtsan.so.0"}


def build_sanitized(kind: str) -> dict:
    """Host-side sanitizer build of the shim, the mock HIP
    runtime and the driver: -fsanitize=address|thread.  GPU sanitizers are
    not available on this pool; these cover the shim's host code (locks,
    accounting, shared region) under concurrent processes and threads."""
    if kind not in SAN_RUNTIME:
        raise ValueError(kind)
    d = SAN_DIR / kind
    md = CSRC / "mockhip"
    shim_srcs = [CSRC / "shim" / "mivgpu_shim.cpp", CSRC / "shim" / "mivgpu_shim.map",
                 CSRC / "include" / "mivgpu" / "shared_region.h", SHIM_FLOOR]
    out = {"shim": d / "libmivgpu.so", "mock": d / "libamdhip64.so", "driver": d / "shim_driver",
           "runtime": SAN_RUNTIME[kind]}
    with _Lock(f"san-{kind}"):
        inc = build_governor()
        d.mkdir(parents=True, exist_ok=True)
        cxx = shutil.which("g++") or "c++"
        flags = ["-std=c++17", "-O1", "-g", "-fPIC", f"-fsanitize={kind}", "-fno-omit-frame-pointer",
                 "-D__HIP_PLATFORM_AMD__", f"-I{ROCM / 'include'}"]
        if _stale(out["shim"], shim_srcs + [inc]):
            _run([cxx, *flags, "-shared", "-fvisibility=hidden", "-include", str(SHIM_FLOOR),
                  f"-I{CSRC / 'include'}", f"-I{inc.parent}",
                  str(shim_srcs[0]), f"-Wl,--version-script={shim_srcs[1]}", "-ldl", "-lpthread",
                  "-o", str(out["shim"])])
        if _stale(out["mock"], [md / "mock_amdhip.cpp", md / "mock_amdhip.map"]):
            _run([cxx, *flags, "-shared", "-fvisibility=hidden", str(md / "mock_amdhip.cpp"),
                  f"-Wl,--version-script={md / 'mock_amdhip.map'}", "-Wl,-soname,libamdhip64.so", "-Wl,-Bsymbolic",
                  "-o", str(out["mock"])])
        if _stale(out["driver"], [md / "shim_driver.cpp", out["mock"]]):
            _run([cxx, *flags, str(md / "shim_driver.cpp"), f"-L{d}", "-lamdhip64", "-ldl", "-lpthread",
                  "-Wl,--disable-new-dtags", f"-Wl,-rpath,{d}", "-o", str(out["driver"])])
    return {k: str(v) for k, v in out.items()}


def build_ops() -> Path:
    """HIP kernels for the workload model and load generators (gfx950)."""
    srcs = sorted((CSRC / "ops").glob("*.hip"))
    hdrs = sorted((CSRC / "ops").glob("*.h"))
    if not srcs:
        return OPS_SO
    with _Lock("ops"):
        if _stale(OPS_SO, srcs + hdrs + [Path(__file__)]):
            LIB.mkdir(parents=True, exist_ok=True)
            obj_dir = BUILD / "ops"
            obj_dir.mkdir(parents=True, exist_ok=True)
            flags = [f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC", "-munsafe-fp-atomics",
                     *NO_PACKED_FP32, f"-I{CSRC / 'include'}"]
            # one object per source, compiled in parallel (the sources share no
            # device code); only the stale ones are rebuilt
            objs = [obj_dir / (src.stem + ".o") for src in srcs]
            todo = [(src, o) for src, o in zip(srcs, objs) if _stale(o, [src, *hdrs, Path(__file__)])]
            from concurrent.futures import ThreadPoolExecutor
            jobs = max(1, min(len(todo), int(os.environ.get("MAX_JOBS", "0") or 0) or (os.cpu_count() or 4)))
            with ThreadPoolExecutor(max_workers=jobs) as ex:
                list(ex.map(lambda so: _run([_hipcc(), *flags, "-c", str(so[0]), "-o", str(so[1])]), todo))
            tmp = OPS_SO.with_suffix(".so.tmp")
            _run([_hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", *map(str, objs), "-o", str(tmp)])
            os.replace(tmp, OPS_SO)
    return OPS_SO


LAUNCH_BENCH = BUILD / "bench" / "launch_bench"


def build_launch_bench() -> Path:
    """Per-launch overhead microbenchmark (csrc/bench/launch_bench.hip)."""
    src = CSRC / "bench" / "launch_bench.hip"
    with _Lock("launch-bench"):
        if _stale(LAUNCH_BENCH, [src, Path(__file__)]):
            LAUNCH_BENCH.parent.mkdir(parents=True, exist_ok=True)
            tmp = LAUNCH_BENCH.with_suffix(".tmp")
            _run([_hipcc(), f"--offload-arch={ARCH}", "-O2", "-std=c++17", *NO_PACKED_FP32, str(src), "-o",
                  str(tmp)])
            os.replace(tmp, LAUNCH_BENCH)
    return LAUNCH_BENCH


RCCL_CHECK = LIB / "mivgpu-rccl-check"


def build_rccl_check() -> Path:
    """The native RCCL collective validator (csrc/bench/rccl_check.cpp)."""
    src = CSRC / "bench" / "rccl_check.cpp"
    with _Lock("rccl-check"):
        if _stale(RCCL_CHECK, [src, Path(__file__)]):
            LIB.mkdir(parents=True, exist_ok=True)
            tmp = RCCL_CHECK.with_suffix(".tmp")
            _run([_hipcc(), f"--offload-arch={ARCH}", "-O2", "-std=c++17", *NO_PACKED_FP32, "-x", "hip", str(src),
                  f"-L{ROCM / 'lib'}", "-lrccl", f"-Wl,-rpath,{ROCM / 'lib'}", "-o", str(tmp)])
            os.replace(tmp, RCCL_CHECK)
    return RCCL_CHECK


def build_all(include_ops: bool = True, include_mock: bool = True) -> dict:
    out = {"shim": str(build_shim()), "boardd": str(build_boardd())}
    if include_ops:
        out["ops"] = str(build_ops())
        out["launch_bench"] = str(build_launch_bench())
        out["rccl_check"] = str(build_rccl_check())
    if include_mock:
        out["mock"] = tuple(str(p) for p in build_mock())
    return out


if __name__ == "__main__":
    what = sys.argv[1:] or ["all"]
    for w in what:
        if w == "all":
            print(build_all())
        elif w == "shim":
            print(build_shim())
        elif w == "boardd":
            print(build_boardd())
        elif w == "ops":
            print(build_ops())
        elif w == "mock":
            print(build_mock())
        elif w == "launch-bench":
            print(build_launch_bench())
        elif w == "rccl-check":
            print(build_rccl_check())
        elif w == "diag":
            print([str(build_hook_diag(lv)) for lv in (1, 2, 3)])
        elif w in ("asan", "tsan"):
            print(build_sanitized({"asan": "address", "tsan": "thread"}[w]))
