"""Build the native runtime extension in-tree:  python setup.py build_ext --inplace

The extensions are plain C++ (compiled by the host compiler) that link the HIP runtime and
PyTorch's c10_hip directly — no hipify step, no CUDA sources.  The serving operators' gfx950 kernels
(csrc/ops/*.hip) are compiled by hipcc into objects that ``tilelang._tl_ops`` links; they are compiled
every time, the rest when its sources changed.
"""
import glob
import os
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pybind11
from setuptools import Extension, setup, find_packages
from torch.utils.cpp_extension import BuildExtension, CppExtension

ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")

ext = CppExtension(
    "tilelang._tl_runtime",
    ["csrc/tl_runtime.cpp"],
    include_dirs=[os.path.join(ROCM, "include")],
    define_macros=[("__HIP_PLATFORM_AMD__", "1"), ("USE_ROCM", "1")],
    library_dirs=[os.path.join(ROCM, "lib")],
    libraries=["amdhip64", "c10_hip"],
    extra_compile_args=["-O2", "-std=c++17", "-Wno-unused-function"],
)

# host-only compiler core (fragment algebra, LDS model, arena planner, hierarchical layouts)
# (plain pybind11, no torch linkage: the compiler runs without loading the torch/HIP runtime)
core = Extension(
    "tilelang._tl_core",
    ["csrc/core/bindings.cc", "csrc/core/fragment.cc", "csrc/core/lds.cc", "csrc/core/hier.cc"],
    include_dirs=[pybind11.get_include()],
    language="c++",
    extra_compile_args=["-O2", "-std=c++17", "-fvisibility=hidden"],
)

# the serving operators: torch bindings and host forms here, the device kernels from hipcc
ops = CppExtension(
    "tilelang._tl_ops",
    ["csrc/ops/bindings.cpp", "csrc/ops/cpu.cpp"],
    depends=sorted(glob.glob("csrc/ops/*.h")),
    include_dirs=[os.path.join(ROCM, "include")],
    define_macros=[("__HIP_PLATFORM_AMD__", "1"), ("USE_ROCM", "1")],
    library_dirs=[os.path.join(ROCM, "lib")],
    libraries=["amdhip64", "c10_hip", "torch_hip"],
    extra_compile_args=["-O2", "-std=c++17", "-fvisibility=hidden", "-Wno-unused-function"],
)

# packed fp32 instructions stay off: some of their forms have given wrong results on gfx950
HIP_FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-fvisibility=hidden", "-Xclang",
             "-target-feature", "-Xclang", "-packed-fp32-ops"]


class BuildWithKernels(BuildExtension.with_options(use_ninja=False)):

    def build_extensions(self):
        out = os.path.join(self.build_temp, "ops")
        os.makedirs(out, exist_ok=True)

        def compile_kernels(src):
            obj = os.path.join(out, os.path.basename(src)[:-len(".hip")] + ".o")
            subprocess.check_call([os.path.join(ROCM, "bin", "hipcc"), *HIP_FLAGS, "-c", src, "-o", obj])
            return obj

        with ThreadPoolExecutor(4) as pool:
            objs = list(pool.map(compile_kernels, sorted(glob.glob("csrc/ops/*.hip"))))
        ops.extra_objects = objs
        ops.depends = ops.depends + objs
        super().build_extensions()


setup(
    name="tilelang-mi355x",
    version="0.1.7+mi355x",
    packages=find_packages(include=["tilelang", "tilelang.*"]),
    package_data={"tilelang": ["include/tl/*.h"]},
    ext_modules=[ext, core, ops],
    cmdclass={"build_ext": BuildWithKernels},
)
