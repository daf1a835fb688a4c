"""The name of the native module with the answering operators' ordinary calls (csrc/calls.cpp): it holds the versions whose internals the module
was compiled against, so that a module of another torch, Python or C++ ABI is not found instead of loaded."""
import sysconfig


def calls_name() -> str:
    import torch
    return f"_calls-torch{torch.__version__}-cxxabi{int(torch._C._GLIBCXX_USE_CXX11_ABI)}{sysconfig.get_config_var('EXT_SUFFIX')}"
