"""The package is found from the repository's root, and from its own folder, as one module either way."""
import os
import pathlib
import subprocess
import sys

import pytest

ROOT = pathlib.Path(__file__).resolve().parents[1]
PKG = ROOT / "kern-glm53_b200"
PROGRAM = """
import sys
sys.path[:0] = sys.argv[1:]
import glmkv.stage
import glmkv
from glmkv import ops
assert glmkv is sys.modules["glmkv"] and glmkv.stage.ops is ops and glmkv.kv4_attn is ops.kv4_attn
print(glmkv.__file__, glmkv.LIB_PATH)
"""


@pytest.mark.parametrize("paths", [[ROOT], [PKG], [ROOT, PKG], [PKG, ROOT]], ids=["root", "folder", "both", "folder first"])
def test_the_package_is_one_module_from_either_path(tmp_path, paths):
    env = {k: v for k, v in os.environ.items() if k != "PYTHONPATH"}
    out = subprocess.run([sys.executable, "-c", PROGRAM, *map(str, paths)], cwd=tmp_path, env=env, check=True,
                         capture_output=True, text=True).stdout.split()
    assert out == [str(PKG / "glmkv" / "__init__.py"), str(PKG / "glmkv" / "libglmkv.so")]
