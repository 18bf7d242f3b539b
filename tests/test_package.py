"""What `import ivonar_inference_b200` gives, with the reference package (a stand-in here) and without."""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]

STAND_IN = """
import sys, types
reference, theirs = types.ModuleType("ivonar_inference"), types.ModuleType("ivonar_inference.decoder")
theirs.StaticDecoder = type("StaticDecoder", (), {})
sys.modules.update({"ivonar_inference": reference, "ivonar_inference.decoder": theirs})
"""


def run(code: str) -> None:
    done = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr


def test_the_package_gives_its_decoder_and_modules() -> None:
    for first in ("package.decoder.B200Decoder", "package.B200Decoder", "package.build_decoder", "package._reference.module('decoder')"):
        run(STAND_IN + f"import ivonar_inference_b200 as package\n{first}\n"
            "assert package.decoder.B200Decoder is package.B200Decoder and package.decoder.build_decoder is package.build_decoder\n"
            "assert package.decoder.DeviceMatrix is package.matrix.DeviceMatrix\n"
            "from ivonar_inference_b200 import *\nassert B200Decoder is package.B200Decoder and KV4Cache is package.KV4Cache")


def test_the_package_without_the_reference() -> None:
    run("import sys\nsys.modules['ivonar_inference'] = None\nimport ivonar_inference_b200 as package\n"
        "package._reference._BUNDLED = package._reference.Path('/nowhere')\npackage.KV4Cache, package.KernelError, package._native\n"
        "for name in ('B200Decoder', 'build_decoder', 'decoder'):\n"
        "    try:\n        getattr(package, name)\n        raise SystemExit(1)\n"
        "    except ImportError as error:\n        assert 'reference package' in str(error)\n"
        "assert not hasattr(package, 'nothing')\nimport ivonar_inference_b200.tp")
