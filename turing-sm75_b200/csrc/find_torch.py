"""For the Makefile: what the torch module needs of the Python that runs this, without importing torch.

Prints the Python's include directory, its torch's directory, the tag of its extension modules and torch's version
(the last two are what a built module fits); nothing where there is no torch with CUDA.
"""
import importlib.util
import os
import re
import sysconfig

spec = importlib.util.find_spec("torch")
if spec and spec.submodule_search_locations:
    torch = spec.submodule_search_locations[0]
    include = sysconfig.get_paths()["include"]
    needed = (os.path.join(torch, "lib", "libc10_cuda.so"), os.path.join(torch, "include", "c10", "cuda", "CUDAGuard.h"),
              os.path.join(torch, "version.py"), os.path.join(include, "Python.h"))
    if all(map(os.path.exists, needed)):
        with open(needed[2]) as f:
            version = re.search(r"^__version__ = ['\"](.*)['\"]", f.read(), re.M)
        print(include, torch, sysconfig.get_config_var("SOABI"), version.group(1) if version else "unknown")
