# Copyright 2026. Licensed under the Apache License, Version 2.0.
"""Build the bluefog_amd native HIP extension in-tree.

    PYTORCH_ROCM_ARCH=gfx950 python setup.py build_ext --inplace

Produces bluefog_amd/_C.*.so (gfx950-only; no CUDA path, no generic
multi-arch fatbin — this framework targets MI355X)."""

import glob
import os

from setuptools import setup

os.environ.setdefault("PYTORCH_ROCM_ARCH", "gfx950")

from torch.utils.cpp_extension import BuildExtension, CUDAExtension

# Objects of HIP sources carry no record of the headers they include: those
# older than the newest header are built again.
_here = os.path.dirname(os.path.abspath(__file__))
_headers = glob.glob(os.path.join(_here, "bluefog_amd", "csrc", "*.h"))
_newest = max(map(os.path.getmtime, _headers), default=0)
for _object in glob.glob(os.path.join(_here, "build", "temp*", "bluefog_amd", "csrc", "*.o")):
    if os.path.getmtime(_object) < _newest:
        os.remove(_object)

ext = CUDAExtension(
    name="bluefog_amd._C",
    sources=[
        "bluefog_amd/csrc/bindings.cpp",
        "bluefog_amd/csrc/bluefog_kernels.hip",
        "bluefog_amd/csrc/transformer_ops.cpp",
        "bluefog_amd/csrc/attention.hip",
        "bluefog_amd/csrc/norm.hip",
    ],
    depends=_headers,
    extra_compile_args={
        "cxx": ["-O3", "-std=c++17"],
        # no packed 32-bit float instructions: some of their forms have given
        # wrong results on gfx950, without an error and not reproducibly
        "nvcc": ["-O3", "-std=c++17",
                 "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"],
    },
)

setup(
    name="bluefog_amd",
    version="0.1.0",
    description="MI355X-native decentralized deep-learning training framework",
    packages=[
        "bluefog_amd",
        "bluefog_amd.ops",
        "bluefog_amd.parallel",
        "bluefog_amd.utils",
        "bluefog_amd.models",
        "bluefog_amd.run",
        "bluefog_amd.torch",
    ],
    ext_modules=[ext],
    cmdclass={"build_ext": BuildExtension},
)
