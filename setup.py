"""Build the rl_amd native extension (CPU segment trees + CDNA4 HIP kernels).

In-tree build: ``python setup.py build_ext --inplace`` produces
``rl_amd/_C*.so`` next to the package so it ships with the source tree.
Target arch is gfx950 only (MI355X) — set via PYTORCH_ROCM_ARCH.
"""
import glob
import os
import sys

os.environ.setdefault("PYTORCH_ROCM_ARCH", "gfx950")

from setuptools import setup  # noqa: E402

import torch  # noqa: E402
from torch.utils import cpp_extension  # noqa: E402

ROOT = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(ROOT, "rl_amd", "csrc")

with_hip = torch.version.hip is not None

# Objects that hipcc made know no headers: what is older than one is compiled again
# (the two sides of a launch must agree on its structs).
headers = glob.glob(os.path.join(CSRC, "*.h"))
newest = max((os.path.getmtime(h) for h in headers), default=0.0)
for obj in glob.glob(os.path.join(ROOT, "build", "temp*", "**", "*.o"), recursive=True):
    if os.path.getmtime(obj) < newest:
        os.remove(obj)

sources = [
    os.path.join(CSRC, "bindings.cpp"),
    os.path.join(CSRC, "llm_bindings.cpp"),
]
extra_cflags = ["-O3", "-std=c++17"]
define_macros = []

if with_hip:
    sources += [
        os.path.join(CSRC, "value_scan.hip"),
        os.path.join(CSRC, "segment_tree_hip.hip"),
        os.path.join(CSRC, "rnn_scan.hip"),
        os.path.join(CSRC, "fused_actor.hip"),
        os.path.join(CSRC, "wgrad.hip"),
        os.path.join(CSRC, "env_step.hip"),
        os.path.join(CSRC, "loss_ops.hip"),
        os.path.join(CSRC, "fused_mlp.hip"),
        os.path.join(CSRC, "rollout_fused.hip"),
        os.path.join(CSRC, "token_loss.hip"),
        os.path.join(CSRC, "paged_kv.hip"),
    ]
    define_macros.append(("RL_AMD_WITH_HIP", None))
    ext_cls = cpp_extension.CUDAExtension
    extra = {
        "extra_compile_args": {
            "cxx": extra_cflags,
            # no packed fp32 instructions: some of their forms have given wrong
            # results on this hardware now and then
            "nvcc": [
                "-O3", "-std=c++17", "--offload-arch=gfx950",
                "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
            ],
        }
    }
else:
    ext_cls = cpp_extension.CppExtension
    extra = {"extra_compile_args": {"cxx": extra_cflags}}

setup(
    name="rl_amd_C",
    ext_modules=[
        ext_cls(
            name="rl_amd._C",
            sources=sources,
            depends=headers,
            define_macros=define_macros,
            **extra,
        )
    ],
    cmdclass={"build_ext": cpp_extension.BuildExtension.with_options(no_python_abi_suffix=False)},
)
