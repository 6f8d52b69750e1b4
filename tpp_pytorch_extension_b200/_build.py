"""Builds the CUDA library in-tree with nvcc for sm_100a (cross-compiles without a GPU).

`build()` makes the whole library. `ensure(architecture)` is for a command that runs one model in a fresh checkout: it
returns the whole library if that is up to date, else a library of only the sources that model needs.

Every csrc/*.cu is compiled to an object under build/ (in parallel, only where the source or a header is newer than the
object) and the objects are linked into libtpx_b200.so beside this file; csrc/tpx_torch.cpp becomes the extension module _tpx_torch.so, for the torch
and the Python that are there. The library does without the module: where that cannot be built, a warning says so. `TPX_DEBUG=1` in the environment adds
-DTPX_DEBUG, which compiles in the timing-experiment knobs and debug exports; the default build has none of them."""
import concurrent.futures
import contextlib
import fcntl
import glob
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
import warnings

HERE = os.path.dirname(os.path.abspath(__file__))
SO = os.path.join(HERE, "libtpx_b200.so")
TORCH_SO = os.path.join(HERE, "_tpx_torch.so")
OBJ_DIR = os.path.join(HERE, "build")
NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC",
]


# sources of models that do not need the whole library (names without the tpx_ prefix)
COMPONENTS = {"Dofivik": ("api", "linear_bf16", "linear_bf16_pair", "linear_bf16_rows", "linear_f32", "linear_f32_pair", "postnorm", "latent", "latent_tc", "latent_dec", "delta", "delta_chunk"),
              "Vedizen": ("api", "linear_bf16", "linear_bf16_pair", "linear_bf16_rows", "linear_f32", "linear_f32_pair", "postnorm", "dyt", "gla", "diff", "diff_tc", "diff_dec")}


def sources():
    return sorted(glob.glob(os.path.join(HERE, "csrc", "*.cu")))


def _headers():
    return glob.glob(os.path.join(HERE, "csrc", "*.cuh")) + glob.glob(os.path.join(HERE, "..", "include", "*.h"))


def _flags():
    return NVCC_FLAGS + (["-DTPX_DEBUG"] if os.environ.get("TPX_DEBUG", "0") == "1" else [])


def _obj(src):
    tag = "dbg" if os.environ.get("TPX_DEBUG", "0") == "1" else "rel"
    return os.path.join(OBJ_DIR, os.path.basename(src)[:-3] + "." + tag + ".o")


def stale(so=SO, srcs=None):
    if not os.path.exists(so):
        return True
    t = os.path.getmtime(so)
    return any(os.path.getmtime(d) > t for d in (srcs or sources()) + _headers())


def _nvcc():
    return os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")


@contextlib.contextmanager
def _alone():
    """One build at a time: objects are shared."""
    os.makedirs(OBJ_DIR, exist_ok=True)
    with open(os.path.join(OBJ_DIR, "lock"), "w") as lock:
        fcntl.flock(lock, fcntl.LOCK_EX)
        yield


def build(force=False, verbose=False, so=SO, srcs=None):
    srcs = srcs or sources()
    if force or stale(so, srcs):
        with _alone():
            if force or stale(so, srcs):
                _build_library(force, verbose, so, srcs)
    if so == SO:
        try:
            if force or module_stale():
                with _alone():
                    if force or module_stale():
                        _build_module()
        except (OSError, subprocess.CalledProcessError) as e:
            with contextlib.suppress(OSError):
                if os.path.getmtime(TORCH_SO) < _module_sources_time():
                    os.remove(TORCH_SO)  # it may not know the library's structures any more
            warnings.warn(f"the extension module _tpx_torch cannot be built ({e}): the operators on packed sequences will not be there")
    return so


def _build_library(force, verbose, so, srcs):
    nvcc = _nvcc()
    hdr_t = max(os.path.getmtime(h) for h in _headers())
    todo = []
    for s in srcs:
        o = _obj(s)
        if force or not os.path.exists(o) or os.path.getmtime(o) < max(os.path.getmtime(s), hdr_t):
            todo.append((s, o))

    def compile_one(so):
        s, o = so
        cmd = [nvcc] + _flags() + (["-Xptxas", "-v"] if verbose else []) + ["-c", "-o", o, s]
        subprocess.check_call(cmd, stdout=sys.stderr)

    with concurrent.futures.ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as ex:
        list(ex.map(compile_one, todo))
    part = so + f".{os.getpid()}"
    subprocess.check_call([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-shared", "-o", part] + [_obj(s) for s in srcs])
    os.replace(part, so)


def cuda_include():
    """The headers beside the compiler, wherever $NVCC is found."""
    found = shutil.which(_nvcc()) or _nvcc()
    for nvcc in (os.path.abspath(found), os.path.realpath(found), "/usr/local/cuda/bin/nvcc"):
        inc = os.path.join(os.path.dirname(os.path.dirname(nvcc)), "include")
        if os.path.exists(os.path.join(inc, "cuda_runtime_api.h")):
            return inc
    raise FileNotFoundError(f"no CUDA headers beside {_nvcc()}")


def _torch_dir():
    spec = importlib.util.find_spec("torch")
    if spec is None:
        raise FileNotFoundError("torch is not installed")
    return os.path.dirname(spec.origin)


def _made_for():
    """What the module depends on besides its sources."""
    with open(os.path.join(_torch_dir(), "version.py")) as f:
        return f"{sys.version}\n{sysconfig.get_config_var('EXT_SUFFIX')}\n{f.read()}"


def _module_sources_time():
    return max(os.path.getmtime(f) for f in [os.path.join(HERE, "csrc", "tpx_torch.cpp")] + _headers())


def _stamp():
    return os.path.join(OBJ_DIR, os.path.basename(TORCH_SO) + ".made_for")


def module_stale():
    if not os.path.exists(TORCH_SO) or not os.path.exists(_stamp()) or os.path.getmtime(TORCH_SO) < _module_sources_time():
        return True
    with open(_stamp()) as f:
        return f.read() != _made_for()


def _build_module():
    """The extension module csrc/tpx_torch.cpp: operators on torch tensors without ctypes in between (g++, against torch's headers)."""
    torch_dir = _torch_dir()
    inc = [os.path.join(torch_dir, "include"), os.path.join(torch_dir, "include", "torch", "csrc", "api", "include"),
           sysconfig.get_paths()["include"], cuda_include()]
    part = TORCH_SO + f".{os.getpid()}"
    subprocess.check_call(["g++", "-O2", "-std=c++17", "-fPIC", "-shared"] + [f for d in inc for f in ("-isystem", d)] +
                          ["-o", part, os.path.join(HERE, "csrc", "tpx_torch.cpp"), "-L" + os.path.join(torch_dir, "lib"),
                           "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python"], stdout=sys.stderr)
    os.replace(part, TORCH_SO)
    with open(_stamp(), "w") as f:
        f.write(_made_for())


def ensure(architecture):
    """Path of an up-to-date library that serves the named architecture, built now if there is none."""
    if architecture not in COMPONENTS:
        return build()
    if not stale():
        return SO
    srcs = [os.path.join(HERE, "csrc", f"tpx_{n}.cu") for n in COMPONENTS[architecture]]
    so = os.path.join(HERE, f"libtpx_b200_{architecture.lower()}.so")
    with open(so + ".lock", "w") as lock:
        fcntl.flock(lock, fcntl.LOCK_EX)
        return build(so=so, srcs=srcs)


if __name__ == "__main__":
    print(build(force=True, verbose=True))
