"""The package and its workload file from the root of a checkout: the root is the working folder and the only
path that is added, so nothing here may lean on the import paths of the test session."""
from __future__ import annotations

import os
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


def from_root(code: str) -> str:
    env = {k: v for k, v in os.environ.items() if k != "PYTHONPATH"}
    code = ("import sys\n"
            "sys.path = [sys.argv[1]] + [p for p in sys.path if 'onecompression' not in p]\n" + code)
    res = subprocess.run([sys.executable, "-c", code, str(ROOT)], cwd=ROOT, env=env, capture_output=True, text=True,
                         timeout=600)
    assert res.returncode == 0, res.stderr[-3000:]
    return res.stdout


def test_package_imports_from_the_root():
    out = from_root("from onecomp_runtime import layers\n"
                    "import onecomp_runtime, onecomp_runtime.layers.rotary as rotary\n"
                    "assert sys.modules['onecomp_runtime'] is onecomp_runtime and onecomp_runtime.layers is layers\n"
                    "assert layers.RotaryEmbedding is rotary.RotaryEmbedding is onecomp_runtime.RotaryEmbedding\n"
                    "print(onecomp_runtime.__file__)\n")
    assert Path(out.strip()) == ROOT / "onecompression-runtime_b200" / "onecomp_runtime" / "__init__.py"


def test_one_package_with_both_paths():
    """The root and the package's own folder on the path, in either order: one module, loaded once."""
    for order in ("[root, pkg]", "[pkg, root]"):
        from_root(f"root = sys.argv[1]; pkg = root + '/onecompression-runtime_b200'\nsys.path[:1] = {order}\n"
                  "import onecomp_runtime as a\nfrom onecomp_runtime import layers\n"
                  "import onecomp_runtime as b\nassert a is b and b.layers is layers\n"
                  "assert len([m for m in sys.modules.values() if getattr(m, '__name__', '') == 'onecomp_runtime']) == 1")


OPERATORS = """
import importlib.util, random, torch
spec = importlib.util.spec_from_file_location("operators", sys.argv[1] + "/perf/operators.py")
ops = importlib.util.module_from_spec(spec)
spec.loader.exec_module(ops)
"""


def test_workload_file_finds_the_layers():
    """Its own calls reach the framework: on CPU tensors they end in the refusal of the device."""
    out = from_root(OPERATORS + """
x, w = torch.zeros(2, 8, dtype=torch.bfloat16), torch.zeros(40, 8, dtype=torch.bfloat16)
try:
    ops._run_own("linear", dict(case=dict(act="none"), x=x, w=w, b=None, r=None))
except RuntimeError as e:
    print(e)
""")
    assert "CUDA" in out


@pytest.mark.gpu
def test_workload_file_runs_its_own_calls(cuda_device):
    """The smallest listed case of each kind and two drawn ones: prepare and run with the framework's calls give
    the shapes and types of the plain form, and values near it."""
    from_root(OPERATORS + """
def flat(y):
    return [y] if isinstance(y, torch.Tensor) else list(y)
cases = [c for c in ops.listed() if c["name"] in ("attn_decode_one", "attn_prompt_chunk", "rope_tokens", "linear_token")]
assert len(cases) == 4
cases += [ops.draw(random.Random(s)) for s in (1, 2)]
for c in cases:
    outs = []
    for ops.own in (False, True):
        outs.append([t.float() for t in flat(ops.run(ops.prepare(c, 5)))])
    for a, b in zip(*outs):
        assert a.shape == b.shape
        # two roundings to 16 bits of values near each other, and of the weights of a mean of values up to 6
        assert bool(((a - b).abs() <= 2.0 ** -7 * (a.abs() + 6.0)).all()), c
""")
