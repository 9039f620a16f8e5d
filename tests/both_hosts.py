"""The Python host layer of a module whose names the compiled extension has taken over."""

import importlib.util

import deep_gemm
from deep_gemm import _api


def python_layer(name: str):
    """`deep_gemm.<name>` as it is where the extension has not been built."""
    spec = importlib.util.find_spec('deep_gemm.' + name)
    module = importlib.util.module_from_spec(spec)
    compiled, _api._C = _api._C, None
    try:
        spec.loader.exec_module(module)
    finally:
        _api._C = compiled
    return module


moe_hosts = [deep_gemm, python_layer('moe_ops')]
quant_hosts = [deep_gemm, python_layer('quant_ops')]
