"""B200-native (sm_100a) Ivonar token loop: decode step, prefill and sampler behind the reference
decoder interface. The compute path is libivonar_b200.so (include/ivonar_b200.h); see
``B200Decoder`` (a subclass of the reference's ``StaticDecoder``), ``build_decoder`` and ``KV4Cache``.

The decoder is imported on first use: it needs the reference package, the rest of this one does not."""

from ._native import KernelError
from .kv4 import KV4Cache

__version__ = "0.2.0"

__all__ = ["B200Decoder", "KV4Cache", "KernelError", "build_decoder"]


def __getattr__(name: str):
    if name in ("B200Decoder", "build_decoder", "decoder", "_reference"):
        import importlib

        found = importlib.import_module("._reference" if name == "_reference" else ".decoder", __name__)
        return found if name in ("decoder", "_reference") else getattr(found, name)
    raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
