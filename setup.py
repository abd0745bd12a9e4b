"""Build the native parts of flodl_b200 in-tree.

Two extensions:

* ``flodl_b200._C``      hand-written sm_100a CUDA kernels (tcgen05 GEMM, flash
  attention, fused norms/losses/optimizers, peer-memory collectives) and their
  torch bindings. Compiled for ``sm_100a`` only.
* ``flodl_b200._native`` the C++ runtime that does not touch the GPU: ``.fdl``
  checkpoint IO, SHA-256/HMAC, graph topology compiler, ElChe cadence
  balancer, CPU averaging reducer and the batch prefetcher.

Usage: ``python setup.py build_ext --inplace -t /tmp/flodl_b200_build`` (``__graft_entry__.build()`` runs
exactly this). Objects are kept per tree under the ``-t`` directory and reused only while what they were
compiled from is the same, whatever the files' times say.
"""
import glob
import hashlib
import os

import torch
from setuptools import setup
from torch.utils.cpp_extension import BuildExtension, CppExtension, CUDAExtension

ROOT = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join("flodl_b200", "csrc")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "--expt-relaxed-constexpr",
    "-diag-suppress", "177",
    "-DNDEBUG",
]
CXX_FLAGS = ["-O3", "-std=c++17", "-DNDEBUG", "-g0"]


def _shared_libstdcxx_dir():
    """Directory holding the SHARED libstdc++ link library.

    A toolchain whose private library directory only carries ``libstdc++.a``
    links a second, static copy of libstdc++ into each extension; that copy's
    iostream/locale state is never initialised, so formatting a number in an
    error message (``TORCH_CHECK(..., n)``) crashes. Putting the system
    directory first makes both extensions use the process-wide libstdc++.so.6
    that torch already loaded.
    """
    import subprocess

    for cxx in ("/usr/bin/g++", "g++", "c++"):
        try:
            out = subprocess.run([cxx, "-print-file-name=libstdc++.so"], capture_output=True,
                                 text=True, timeout=30).stdout.strip()
        except Exception:
            continue
        if os.path.isabs(out) and os.path.exists(out):
            return [os.path.dirname(out)]
    return []


LINK_DIRS = _shared_libstdcxx_dir()
LINK_FLAGS = [f"-L{d}" for d in LINK_DIRS]


def _sources(*patterns):
    out = []
    for p in patterns:
        out.extend(sorted(glob.glob(os.path.join(CSRC, p))))
    return out


ext_modules = [
    CUDAExtension(
        name="flodl_b200._C",
        sources=_sources("bind/*.cpp", "capi/*.cpp", "kernels/*.cu", "comm/*.cu"),
        include_dirs=[os.path.join(ROOT, CSRC)],
        extra_compile_args={"cxx": CXX_FLAGS, "nvcc": NVCC_FLAGS},
        extra_link_args=LINK_FLAGS,
    ),
    CppExtension(
        name="flodl_b200._native",
        sources=_sources("runtime/*.cpp"),
        include_dirs=[os.path.join(ROOT, CSRC)],
        extra_compile_args={"cxx": CXX_FLAGS},
        libraries=["z"],
        extra_link_args=LINK_FLAGS,
    ),
]

def _digest(*parts):
    h = hashlib.sha256()
    for p in parts:
        h.update(len(p).to_bytes(8, "little") + p)
    return h.hexdigest()


def _read(path):
    with open(path, "rb") as f:
        return f.read()


class Build(BuildExtension.with_options(use_ninja=True)):
    """Objects by content.

    ninja compares modification times only: where another version of the tree
    was built at this path before, and the files here carry older times (a
    commit's, as archives and time-preserving copies keep them), it would link
    the other version's objects. So every object has a key beside it, of its
    source, of all headers and of the toolkit, and one whose key differs is
    removed first. Trees do not share a directory.
    """

    def finalize_options(self):
        super().finalize_options()
        self.build_temp = os.path.join(self.build_temp,
                                       "tree-" + _digest(os.path.realpath(ROOT).encode())[:16])

    def build_extension(self, ext):
        headers = sorted(f for f in glob.glob(os.path.join(CSRC, "**", "*"), recursive=True)
                         if os.path.isfile(f) and not f.endswith((".cpp", ".cu")))
        common = [f"{torch.__version__} {torch.version.cuda}".encode()]
        for f in headers:
            common += [f.encode(), _read(f)]
        common = _digest(*common).encode()
        keys = {}
        for src in ext.sources:
            obj = os.path.join(self.build_temp, os.path.splitext(src)[0] + ".o")
            keys[obj] = _digest(common, src.encode(), _read(src)).encode()
            known = os.path.exists(obj + ".key") and _read(obj + ".key") == keys[obj]
            if os.path.exists(obj) and not known:
                os.remove(obj)
        super().build_extension(ext)
        for obj, key in keys.items():
            if not os.path.exists(obj):
                raise RuntimeError(f"{obj} was not built")
            with open(obj + ".key", "wb") as f:
                f.write(key)


setup(
    name="flodl_b200",
    version="0.1.0",
    packages=["flodl_b200"],
    ext_modules=ext_modules,
    cmdclass={"build_ext": Build},
)
