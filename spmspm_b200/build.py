"""In-tree build of libSpMM_API.so (nvcc, sm_100a only) and of the extension that calls its 4-bit operators from tensors."""
import os
import subprocess
import sysconfig

_HERE = os.path.dirname(os.path.abspath(__file__))


def ext_flags():
    """Compiler flags of the extension, by their names in the Makefile."""
    import torch
    from torch.utils.cpp_extension import include_paths, library_paths
    return dict(EXT_INCLUDES=" ".join("-isystem " + d for d in include_paths("cuda") + [sysconfig.get_paths()["include"]]),
                EXT_LIBS=" ".join("-L" + d for d in library_paths("cuda")),
                EXT_ABI=f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}")


def build(verbose=False):
    env = dict(os.environ, **ext_flags())
    r = subprocess.run(["make", "-C", os.path.join(_HERE, "csrc"), "-j", "6"], capture_output=True, text=True, env=env)
    if verbose or r.returncode != 0:
        print(r.stdout[-4000:])
        print(r.stderr[-4000:])
    if r.returncode != 0:
        raise RuntimeError("building libSpMM_API.so failed")
    return os.path.join(_HERE, "libSpMM_API.so")
