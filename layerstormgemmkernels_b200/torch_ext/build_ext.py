"""Builds the PyTorch extension modules in-tree, linked against layerstormgemmkernels_b200/liblsg_b200.so:

  <repo>/sm120_gemm_kernels.so                             the reference's module name and operators
  layerstormgemmkernels_b200/torch_ext/lsg_torch_ops.so    host side of the eager operators of
                                                           ops.py that have no counterpart there

    python -m layerstormgemmkernels_b200.torch_ext.build_ext
"""
import os
import shutil
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
PKG = os.path.dirname(HERE)
ROOT = os.path.dirname(PKG)


def _build(name, source, out, verbose):
    from torch.utils.cpp_extension import load
    bdir = os.path.join(HERE, "_build", name)
    os.makedirs(bdir, exist_ok=True)
    up = os.path.relpath(PKG, os.path.dirname(out))
    load(name=name, sources=[os.path.join(HERE, source)],
         extra_include_paths=[os.path.join(ROOT, "include")],
         extra_cflags=["-O2", "-std=c++17"],
         # the library beside the module, wherever the tree lies ($$ for ninja, quotes for the shell)
         extra_ldflags=[f"-L{PKG}", "-llsg_b200", f"-Wl,-rpath,'$$ORIGIN/{up}'", f"-Wl,-rpath,{PKG}"],
         build_directory=bdir, with_cuda=True, is_python_module=False, verbose=verbose)
    shutil.copyfile(os.path.join(bdir, name + ".so"), out)
    return out


def build(verbose=False):
    from .. import build as libbuild
    libbuild.build()
    build_ops(verbose)
    return _build("sm120_gemm_kernels", "bindings_python.cpp", os.path.join(ROOT, "sm120_gemm_kernels.so"), verbose)


def build_ops(verbose=False):
    return _build("lsg_torch_ops", "int8_moe_ops.cpp", os.path.join(HERE, "lsg_torch_ops.so"), verbose)


if __name__ == "__main__":
    print(build(verbose="--verbose" in sys.argv))
