"""In-tree build of the deepof_amd HIP extension for gfx950.

    PYTORCH_ROCM_ARCH=gfx950 python setup.py build_ext --inplace

The .so lands in deepof_amd/ops/hip/ so it travels with the repo
snapshot to GPU boxes (no JIT cache dependence).
"""

import glob
import os

os.environ.setdefault("PYTORCH_ROCM_ARCH", "gfx950")

from setuptools import setup
from torch.utils.cpp_extension import BuildExtension, CUDAExtension

ROOT = os.path.dirname(os.path.abspath(__file__))
SRC = os.path.join("deepof_amd", "ops", "hip")

# the generated build file does not know which headers an object was built
# from: objects older than a header are built again
newest = max(os.path.getmtime(h) for h in glob.glob(os.path.join(ROOT, SRC, "*.h")))
for obj in glob.glob(os.path.join(ROOT, "build", "temp.*", SRC, "*.o")):
    if os.path.getmtime(obj) < newest:
        os.remove(obj)

ext = CUDAExtension(
    name="deepof_amd.ops.hip._deepof_hip",
    sources=[
        os.path.join(SRC, "ext.cpp"),
        os.path.join(SRC, "loss_kernels.hip"),
        os.path.join(SRC, "correlation.hip"),
        os.path.join(SRC, "adam.hip"),
        os.path.join(SRC, "conv_mfma.hip"),
        os.path.join(SRC, "conv_wrw2.hip"),
        os.path.join(SRC, "group_norm.cpp"),
        os.path.join(SRC, "group_norm_f32.hip"),
        os.path.join(SRC, "group_norm_f16.hip"),
        os.path.join(SRC, "group_norm_bf16.hip"),
        os.path.join(SRC, "dropout.hip"),
        os.path.join(SRC, "autograd.cpp"),
    ],
    extra_compile_args={
        "cxx": ["-O3", "-std=c++17"],
        # packed fp32 arithmetic is kept out of device code: some of its
        # forms have returned wrong sums on gfx950
        "nvcc": ["-O3", "-std=c++17", "--offload-arch=gfx950",
                 "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"],
    },
)

setup(
    name="deepof_amd",
    version="0.1.0",
    packages=["deepof_amd"],
    ext_modules=[ext],
    cmdclass={"build_ext": BuildExtension.with_options(use_ninja=True)},
)
