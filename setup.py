"""Build the in-tree gfx950 HIP extension: python setup.py build_ext --inplace

The resulting zaremba_amd/_hip*.so travels with the repo snapshot to GPU
boxes (no JIT cache involved). hipcc cross-compiles without a GPU.
"""

import glob
import os

from setuptools import setup

os.environ.setdefault("PYTORCH_ROCM_ARCH", "gfx950")

from torch.utils.cpp_extension import BuildExtension, CUDAExtension  # noqa: E402

here = os.path.dirname(os.path.abspath(__file__))


def drop_stale_objects():
    """The build knows of no header that a HIP source includes: an object
    older than one of them would keep the old structs and constants, beside
    objects that have the new ones. Such objects are compiled again."""
    headers = glob.glob(os.path.join(here, "zaremba_amd/csrc/*.h"))
    newest = max(map(os.path.getmtime, headers))
    objects = os.path.join(here, "build/temp.*/**/*.o")
    for path in glob.glob(objects, recursive=True):
        if os.path.getmtime(path) < newest:
            os.remove(path)


drop_stale_objects()

ext = CUDAExtension(
    name="zaremba_amd._hip",
    sources=[
        "zaremba_amd/csrc/ext_bind.hip",
        "zaremba_amd/csrc/gemm.hip",
        "zaremba_amd/csrc/lstm.hip",
        "zaremba_amd/csrc/lstm_persistent.hip",
        "zaremba_amd/csrc/elementwise.hip",
        "zaremba_amd/csrc/adamw.hip",
        "zaremba_amd/csrc/adamw_bind.hip",
        "zaremba_amd/csrc/glr.hip",
        "zaremba_amd/csrc/glr_bind.hip",
    ],
    extra_compile_args={
        "cxx": ["-O3", "-std=c++17"],
        # packed f32 instructions stay off: some of their forms have given
        # wrong results on this hardware now and then
        "nvcc": ["-O3", "-std=c++17", "--offload-arch=gfx950",
                 "-Xclang", "-target-feature", "-Xclang",
                 "-packed-fp32-ops"],
    },
)

setup(
    name="zaremba_amd",
    version="0.1.0",
    packages=["zaremba_amd"],
    ext_modules=[ext],
    cmdclass={"build_ext": BuildExtension},
)
