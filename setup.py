"""In-tree build of the CDNA4 HIP extension.

    PYTORCH_ROCM_ARCH=gfx950 python setup.py build_ext --inplace

The built blades_amd/_hip_ops*.so travels with the repo snapshot to GPU
boxes (it is git-ignored but NOT gpurun-ignored).
"""
import os

from setuptools import setup

os.environ.setdefault("PYTORCH_ROCM_ARCH", "gfx950")

from torch.utils.cpp_extension import BuildExtension, CUDAExtension

setup(
    name="blades_amd",
    version="0.1.0",
    packages=["blades_amd", "blades"],
    ext_modules=[
        CUDAExtension(
            name="blades_amd._hip_ops",
            sources=["csrc/blades_kernels.hip", "csrc/token_bindings.cpp",
                     "csrc/layer_norm.hip", "csrc/act8.hip",
                     "csrc/token_gemm.hip"],
            depends=["csrc/token_ops.h", "csrc/token_device.h"],
            extra_compile_args={
                # stands in only where no other path has such a header
                "cxx": ["-O3", "-idirafter", os.path.join(
                    os.path.dirname(os.path.abspath(__file__)), "csrc",
                    "compat")],
                # no packed fp32 instructions: some of their forms have
                # given wrong results on this hardware
                "nvcc": ["-O3", "-std=c++17", "-Xclang", "-target-feature",
                         "-Xclang", "-packed-fp32-ops"],
            },
        ),
    ],
    cmdclass={"build_ext": BuildExtension},
)
