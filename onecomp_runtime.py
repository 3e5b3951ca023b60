"""``import onecomp_runtime`` from the root of a checkout, with nothing on ``PYTHONPATH``.

The package lies in ``onecompression-runtime_b200/onecomp_runtime``; this module puts it in its own place, so
that one package is loaded whichever path finds it first.
"""
import importlib.util
import sys
from pathlib import Path

_home = Path(__file__).resolve().parent / "onecompression-runtime_b200" / "onecomp_runtime"
_spec = importlib.util.spec_from_file_location(__name__, _home / "__init__.py", submodule_search_locations=[str(_home)])
_package = importlib.util.module_from_spec(_spec)
sys.modules[__name__] = _package   # the import statement returns what stands here
_spec.loader.exec_module(_package)
