"""Build the gfx950 HIP extensions in-tree.

python setup.py build_ext --inplace   (PYTORCH_ROCM_ARCH=gfx950)
"""

import hashlib
import os

from setuptools import find_packages, setup

os.environ.setdefault("PYTORCH_ROCM_ARCH", "gfx950")

from torch.utils.cpp_extension import BuildExtension, CUDAExtension  # noqa: E402

CSRC = os.path.join(os.path.dirname(os.path.abspath(__file__)), "beta9_amd", "ops", "csrc")

ext_flags = ["-O3", "-std=c++17"]
# packed fp32 arithmetic is left out of all HIP code: some of its forms have given wrong results on MI355X
hip_flags = ext_flags + ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]

# a changed header changes the command line of every source that may include it, and so builds it again
paged_sources = ("bind.cpp", "tables.hip", "write.hip", "decode.hip", "prompt.hip")
paged_headers = hashlib.sha256()
for name in ("paged.h", "device.h"):
    with open(os.path.join(CSRC, "paged", name), "rb") as f:
        paged_headers.update(f.read())
paged_define = [f"-DPAGED_HEADERS={paged_headers.hexdigest()[:16]}"]

setup(
    name="beta9-amd",
    version="0.1.0",
    packages=find_packages(include=["beta9_amd", "beta9_amd.*"]),
    entry_points={"console_scripts": ["b9 = beta9_amd.cli.main:main"]},
    ext_modules=[
        CUDAExtension(
            name="beta9_amd.ops._hipsnap_ext",
            sources=[os.path.join(CSRC, "hipsnap.hip")],
            extra_compile_args={"cxx": ext_flags, "nvcc": hip_flags},
        ),
        CUDAExtension(
            name="beta9_amd.ops._gemm_ext",
            sources=[os.path.join(CSRC, "gemm.hip")],
            extra_compile_args={"cxx": ext_flags, "nvcc": hip_flags},
        ),
        CUDAExtension(
            name="beta9_amd.ops._paged_ext",
            sources=[os.path.join(CSRC, "paged", name) for name in paged_sources],
            extra_compile_args={"cxx": ext_flags + paged_define, "nvcc": hip_flags + paged_define},
        ),
    ],
    cmdclass={"build_ext": BuildExtension.with_options(no_python_abi_suffix=True)},
)
