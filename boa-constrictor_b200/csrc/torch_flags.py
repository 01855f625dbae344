"""Compiler and linker flags for a CPython module on the installed torch."""
import os
import sysconfig

import torch

base = os.path.dirname(torch.__file__)
cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
inc = [sysconfig.get_paths()["include"], os.path.join(base, "include"),
       os.path.join(base, "include", "torch", "csrc", "api", "include"), os.path.join(cuda, "include")]
lib = os.path.join(base, "lib")
print(" ".join([f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"] + [f"-isystem {p}" for p in inc]
               + [f"-L{lib}", f"-Wl,-rpath,{lib}", "-ltorch_python", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-lc10",
                  "-lc10_cuda"]))
