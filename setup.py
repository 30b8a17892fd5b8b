# -*- coding: utf-8 -*-
"""Build the in-tree HIP extension for gfx950.

    PYTORCH_ROCM_ARCH=gfx950 python setup.py build_ext --inplace

Produces ``stoke/_C.cpython-*.so`` next to the package so it travels with
repo snapshots (no JIT cache dependence).
"""

import os

from setuptools import setup

from torch.utils import cpp_extension

os.environ.setdefault("PYTORCH_ROCM_ARCH", "gfx950")



def drop_old_objects(folder, headers):
    """Objects that are older than a header: the generated build rules know
    which source an object comes from, not what the source includes."""
    newest = max(os.path.getmtime(h) for h in headers)
    for root, _, names in os.walk(folder):
        for name in names:
            path = os.path.join(root, name)
            if name.endswith(".o") and os.path.getmtime(path) <= newest:
                os.remove(path)


class BuildExtension(cpp_extension.BuildExtension):
    def build_extensions(self):
        for ext in self.extensions:
            drop_old_objects(self.build_temp, ext.depends)
        super().build_extensions()


if __name__ == "__main__":
    setup(
        name="stoke-amd",
        version="0.1.0",
        description="MI355X-native declarative training wrapper for PyTorch-ROCm",
        packages=[
            "stoke",
            "stoke.runtime",
            "stoke.comm",
            "stoke.ddp",
            "stoke.shard",
            "stoke.amp",
            "stoke.ops",
            "stoke.nn",
        ],
        ext_modules=[
            cpp_extension.CUDAExtension(
                name="stoke._C",
                sources=["csrc/stoke_kernels.hip", "csrc/fused_bn.hip",
                         "csrc/fused_rmsnorm.hip",
                         "csrc/fused_rope.hip",
                         "csrc/fused_swiglu.hip",
                         "csrc/fused_layernorm.hip",
                         "csrc/fa_fwd.hip",
                         "csrc/fa_bwd.hip",
                         "csrc/fp8_quant.hip",
                         "csrc/fused_ce.hip",
                         "csrc/act8.hip",
                         "csrc/token_loss.hip",
                         "csrc/qk_norm_rope.hip"],
                depends=["csrc/elem.h"],
                extra_compile_args={
                    "cxx": ["-O3"],
                    # scalar fp32 only: some packed fp32 forms that the compiler
                    # makes by itself are not reliable on this target
                    "nvcc": ["-O3", "-std=c++17", "-Xclang", "-target-feature",
                             "-Xclang", "-packed-fp32-ops"],
                },
            )
        ],
        cmdclass={"build_ext": BuildExtension},
    )
