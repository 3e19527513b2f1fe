"""Compile the HIP sources in this directory for gfx950 (in-tree .so files that travel with the repo).

* gpuprobe.hip  -> libgpuprobe.so           C ABI, loaded with ctypes by devspace_amd.gpucheck
* FUSED_SOURCES -> _fused_ops<EXT_SUFFIX>   PyTorch extension (ATen + pybind11), compiled directly
                                            with hipcc against the installed torch headers/libs,
                                            one object per source, in parallel
"""

import contextlib
import hashlib
import os
import shutil
import subprocess
import sysconfig
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))
FUSED_SOURCES = ("fused_ops.hip", "rotary.hip", "dropout.hip", "cross_attention.hip")
FUSED_HEADERS = ("fused_common.h",)
ARCH = os.environ.get("PYTORCH_ROCM_ARCH", "gfx950")
# No packed fp32 instructions (v_pk_add/mul/fma_f32), which the compiler would otherwise make from
# ordinary float code: some of their forms have given wrong results now and then on these parts.
# The host pass warns that it does not know the feature; that is harmless.
NO_PACKED_FP32 = ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]
FUSED_FLAGS = ["-O3", *NO_PACKED_FP32, "-std=c++17", "-fPIC", "-DUSE_ROCM=1", "-DTORCH_EXTENSION_NAME=_fused_ops",
               "-DTORCH_API_INCLUDE_EXTENSION_H", "-Wno-unused-result"]


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


def _fused_contents():
    """name -> bytes of the extension's sources and headers, in their order."""
    out = {}
    for n in FUSED_SOURCES + FUSED_HEADERS:
        with open(os.path.join(HERE, n), "rb") as f:
            out[n] = f.read()
    return out


def _sha(*parts) -> str:
    h = hashlib.sha256()
    for p in parts:
        h.update(p if isinstance(p, bytes) else repr(p).encode())
    return h.hexdigest()


def _contents_sha(contents) -> str:
    return _sha(*contents.values(), FUSED_FLAGS)


def source_sha(path=None) -> str:
    """SHA-256 of the extension's sources and flags, linked into it (`_fused_ops.source_sha`); of the one file `path`,
    if given."""
    if path:
        with open(path, "rb") as f:
            return _sha(f.read())
    return _contents_sha(_fused_contents())


def _fused_tag():
    """Cache key of a fused-ops build: source bytes and flags, torch build, target arch, Python ABI."""
    import torch

    return _sha(source_sha(), torch.__version__, torch.version.hip, ARCH, sysconfig.get_config_var("EXT_SUFFIX"))[:16]


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


def _compiler():
    """What tells one compiler from another at the same path."""
    return subprocess.run([hipcc(), "--version"], check=True, capture_output=True).stdout


@contextlib.contextmanager
def _alone(directory):
    """One build at a time works in `directory`; another one waits."""
    import fcntl

    os.makedirs(directory, exist_ok=True)
    with open(os.path.join(directory, "lock"), "w") as f:
        fcntl.flock(f, fcntl.LOCK_EX)
        yield


def build_fused(verbose=False, force=False, out=None):
    """Compiles what has changed (everything with `force`) and links the extension. The in-tree build keeps its objects,
    each under a hash of all that goes into it (source, headers, command, compiler and torch), never by a time stamp: an
    edit with an old time, another ARCH or another torch finds no object and is compiled."""
    out = out or fused_path()
    if out != fused_path():
        with tempfile.TemporaryDirectory() as objdir:
            return _build_fused(out, objdir, verbose, force)
    objdir = os.path.join(HERE, "_obj")
    with _alone(objdir):
        return _build_fused(out, objdir, verbose, force)


def _build_fused(out, objdir, verbose, force):
    import torch  # headers + libraries of the torch this extension is loaded into

    troot = os.path.dirname(torch.__file__)
    tlib = os.path.join(troot, "lib")
    base = [hipcc(), f"--offload-arch={ARCH}", *FUSED_FLAGS, f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
            "-I" + os.path.join(troot, "include"), "-I" + os.path.join(troot, "include", "torch", "csrc", "api", "include"),
            "-I" + sysconfig.get_paths()["include"]]
    libs = ["-L" + tlib, "-lc10", "-lc10_hip", "-ltorch", "-ltorch_cpu", "-ltorch_hip", "-ltorch_python", "-Wl,-rpath," + tlib]
    contents = _fused_contents()
    around = (base, _compiler(), torch.__version__, torch.version.hip, *(contents[h] for h in FUSED_HEADERS))
    objs = {n: os.path.join(objdir, f"{n}.{_sha(contents[n], *around)[:16]}.o") for n in FUSED_SOURCES}
    linked = os.path.join(objdir, "linked")  # which objects the extension was linked from, and its own hash
    stamp = _sha([os.path.basename(o) for o in objs.values()], _contents_sha(contents), libs)
    if not force and _read(linked) == f"{stamp} {_sha(_read(out, 'rb') or b'')}":
        return out
    # all that is written becomes visible in one step, when it is whole and belongs to the sources as they were read
    with tempfile.TemporaryDirectory(dir=objdir) as tmp:
        running = []
        for name, obj in objs.items():
            if force or not os.path.exists(obj):
                cmd = base + ["-c", os.path.join(HERE, name), "-o", os.path.join(tmp, name + ".o")]
                if verbose:
                    print("+", " ".join(cmd), flush=True)
                running.append((subprocess.Popen(cmd), cmd, name))
        failed = [(p.returncode, cmd) for p, cmd, _ in running if p.wait()]
        if failed:
            raise subprocess.CalledProcessError(*failed[0])
        if _fused_contents() != contents:
            raise RuntimeError("the fused ops' sources changed while they were being compiled: build again")
        for _, _, name in running:
            os.replace(os.path.join(tmp, name + ".o"), objs[name])
        sha = os.path.join(tmp, "source_sha.cpp")
        with open(sha, "w") as f:
            f.write(f'extern const char devspace_source_sha[];\nconst char devspace_source_sha[] = "{_contents_sha(contents)}";\n')
        lib = os.path.join(tmp, "lib.so")
        _run([hipcc(), "-shared", "-fPIC", "-x", "c++", sha, "-x", "none", *objs.values(), *libs, "-o", lib], verbose)
        record = f"{stamp} {_sha(_read(lib, 'rb'))}"
        os.makedirs(os.path.dirname(out), exist_ok=True)
        shutil.move(lib, out + ".new")  # another file system, perhaps
        os.replace(out + ".new", out)
        with open(linked, "w") as f:
            f.write(record)
    for n in os.listdir(objdir):  # what earlier states of the sources left
        if n.endswith(".o") and os.path.join(objdir, n) not in objs.values():
            os.remove(os.path.join(objdir, n))
    return out


def _read(path, mode="r"):
    try:
        with open(path, mode) as f:
            return f.read()
    except FileNotFoundError:
        return None


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
