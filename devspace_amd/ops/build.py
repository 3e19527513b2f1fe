"""Compile the HIP sources in this directory for gfx950 (in-tree .so files that travel with the repo).

* gpuprobe.hip  -> libgpuprobe.so           C ABI, loaded with ctypes by devspace_amd.gpucheck
* FUSED_SOURCES -> _fused_ops<EXT_SUFFIX>   PyTorch extension (ATen + pybind11), compiled directly
                                            with hipcc against the installed torch headers/libs,
                                            one object per source, in parallel
"""

import os
import shutil
import subprocess
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
FUSED_SOURCES = ("fused_ops.hip", "rotary.hip", "dropout.hip", "cross_attention.hip")
FUSED_HEADERS = ("fused_common.h",)
ARCH = os.environ.get("PYTORCH_ROCM_ARCH", "gfx950")
# No packed fp32 instructions (v_pk_add/mul/fma_f32), which the compiler would otherwise make from
# ordinary float code: some of their forms have given wrong results now and then on these parts.
# The host pass warns that it does not know the feature; that is harmless.
NO_PACKED_FP32 = ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


def hipcc():
    for cand in (shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if cand and os.path.exists(cand):
            return cand
    raise FileNotFoundError("hipcc not found")


def lib_path(name="gpuprobe"):
    return os.path.join(HERE, f"lib{name}.so")


def fused_path():
    return os.path.join(HERE, "_fused_ops" + sysconfig.get_config_var("EXT_SUFFIX"))


def _stale(out, *srcs):
    return not os.path.exists(out) or any(os.path.getmtime(out) < os.path.getmtime(s) for s in srcs)


def _run(cmd, verbose):
    if verbose:
        print("+", " ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)


def build_probe(verbose=False, force=False):
    src = os.path.join(HERE, "gpuprobe.hip")
    out = lib_path()
    if force or _stale(out, src):
        _run([hipcc(), "-O3", f"--offload-arch={ARCH}", *NO_PACKED_FP32, "-shared", "-fPIC", "-Wno-unused-value",
              "-o", out, src], verbose)
    return out


def _fused_files():
    return [os.path.join(HERE, n) for n in FUSED_SOURCES + FUSED_HEADERS]


def source_sha(path=None) -> str:
    """SHA-256 of the extension's sources (of the one file `path`, if given), compiled into it
    (`_fused_ops.source_sha`)."""
    import hashlib

    h = hashlib.sha256()
    for p in [path] if path else _fused_files():
        with open(p, "rb") as f:
            h.update(f.read())
    return h.hexdigest()


def _fused_tag():
    """Cache key of a fused-ops build: source bytes, torch build, target arch, flags, Python ABI."""
    import hashlib

    import torch

    key = (source_sha(), torch.__version__, torch.version.hip, ARCH, NO_PACKED_FP32, sysconfig.get_config_var("EXT_SUFFIX"))
    return hashlib.sha256("|".join(map(str, key)).encode()).hexdigest()[:16]


def fused_cache_path():
    """Where a vendored copy (a project made by `devspace init`, running in its pod) keeps the
    extension it compiled: $DEVSPACE_OPS_CACHE or ~/.cache/devspace_amd, keyed by _fused_tag()."""
    base = os.environ.get("DEVSPACE_OPS_CACHE") or os.path.join(os.path.expanduser("~"), ".cache", "devspace_amd")
    return os.path.join(base, "fused-" + _fused_tag(), "_fused_ops" + sysconfig.get_config_var("EXT_SUFFIX"))


def ensure_fused_cached(verbose=True):
    """Compiles the extension into the cache unless it is there (minutes: done at image build by
    the rocm-pytorch Dockerfile, else once on the first pod start). Returns its path."""
    out = fused_cache_path()
    if not os.path.exists(out):
        os.makedirs(os.path.dirname(out), exist_ok=True)
        tmp = out + f".tmp{os.getpid()}"
        if verbose:
            print(f"[devspace_amd] compiling the fused gfx950 ops ({ARCH}) into {out} ...", flush=True)
        build_fused(verbose=False, force=True, out=tmp)
        os.replace(tmp, out)  # concurrent ranks: whoever finishes first wins, the rest overwrite
    return out


def build_fused(verbose=False, force=False, out=None):
    """Compiles the sources that changed (all of them with `force`) and links the extension."""
    import tempfile

    import torch  # headers + libraries of the torch this extension is loaded into

    out = out or fused_path()
    if not (force or _stale(out, *_fused_files())):
        return out
    troot = os.path.dirname(torch.__file__)
    tlib = os.path.join(troot, "lib")
    cxx11 = int(torch._C._GLIBCXX_USE_CXX11_ABI)
    base = [hipcc(), "-O3", f"--offload-arch={ARCH}", *NO_PACKED_FP32, "-std=c++17", "-fPIC",
            "-DUSE_ROCM=1", "-DTORCH_EXTENSION_NAME=_fused_ops", "-DTORCH_API_INCLUDE_EXTENSION_H",
            f"-D_GLIBCXX_USE_CXX11_ABI={cxx11}", "-Wno-unused-result",
            "-I" + os.path.join(troot, "include"), "-I" + os.path.join(troot, "include", "torch", "csrc", "api", "include"),
            "-I" + sysconfig.get_paths()["include"]]
    # objects of the in-tree build stay (a change of one source compiles that one); others are temporary
    with tempfile.TemporaryDirectory() as tmp:
        objdir = os.path.join(HERE, "_obj") if out == fused_path() else tmp
        os.makedirs(objdir, exist_ok=True)
        objs, running = [], []
        headers = [os.path.join(HERE, n) for n in FUSED_HEADERS]
        for name in FUSED_SOURCES:
            src, obj = os.path.join(HERE, name), os.path.join(objdir, name + ".o")
            objs.append(obj)
            if force or _stale(obj, src, os.path.abspath(__file__), *headers):
                cmd = base + ["-c", src, "-o", obj + ".tmp"]
                if verbose:
                    print("+", " ".join(cmd), flush=True)
                running.append((subprocess.Popen(cmd), cmd, obj))
        failed = [(p.returncode, cmd) for p, cmd, obj in running if p.wait()]
        if failed:
            raise subprocess.CalledProcessError(*failed[0])
        for _, _, obj in running:
            os.replace(obj + ".tmp", obj)
        sha = os.path.join(tmp, "source_sha.cpp")
        with open(sha, "w") as f:
            f.write(f'extern const char devspace_source_sha[];\nconst char devspace_source_sha[] = "{source_sha()}";\n')
        _run([hipcc(), "-shared", "-fPIC", "-x", "c++", sha, "-x", "none", *objs,
              "-L" + tlib, "-lc10", "-lc10_hip", "-ltorch", "-ltorch_cpu", "-ltorch_hip", "-ltorch_python",
              "-Wl,-rpath," + tlib, "-o", out], verbose)
    return out


def build(verbose=False, force=False):
    out = build_probe(verbose=verbose, force=force)
    build_fused(verbose=verbose, force=force)
    return out


def main(argv=None):
    import argparse

    p = argparse.ArgumentParser(prog="devspace_amd.ops.build", description=__doc__.split("\n")[0])
    p.add_argument("--fused", action="store_true", help="the fused training ops")
    p.add_argument("--probe", action="store_true", help="the GPU probe library")
    p.add_argument("--cache", action="store_true",
                   help="build the fused ops into the cache (image build of a vendored copy) instead of in place")
    a = p.parse_args(argv)
    if a.probe:
        print(build_probe(verbose=True))
    if a.fused:
        print(ensure_fused_cached() if a.cache else build_fused(verbose=True))
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
