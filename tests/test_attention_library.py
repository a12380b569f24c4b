"""The package without the library of attention and rotary positions: everything else imports and runs, they say what is missing."""
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

PACKAGE = Path(__file__).resolve().parent.parent / "torchpairwise_b200"
CODE = """
import torch, torchpairwise_b200 as tpw
assert tpw.__file__.startswith({root!r}), tpw.__file__
x = torch.zeros(3, 2, 8)
try:
    tpw.euclidean_distances(x[0], x[0])
except RuntimeError as e:
    assert "CUDA" in str(e), e
for call in (lambda: tpw.attention(x, x, x), lambda: tpw.rotary_embedding(x, None, x[0], x[0]), lambda: tpw.rotary_table(4, 8, device="cpu")):
    try:
        call()
    except ImportError as e:
        assert {text!r} in str(e) and "build.py" in str(e), e
    else:
        raise AssertionError("no ImportError")
print("fine")
"""


@pytest.mark.parametrize("state,text", [("missing", "is missing"), ("of another torch", "does not load")])
def test_the_package_imports_without_the_attention_library(tmp_path, state, text):
    root = tmp_path / "torchpairwise_b200"
    (root / "lib").mkdir(parents=True)
    for source in PACKAGE.glob("*.py"):
        shutil.copy(source, root)
    (root / "lib" / "libtpw_b200.so").symlink_to(PACKAGE / "lib" / "libtpw_b200.so")
    if state != "missing":
        (root / "lib" / "libtpw_b200_attention.so").write_bytes(b"not a library that this interpreter can load")
    r = subprocess.run([sys.executable, "-c", CODE.format(root=str(tmp_path), text=text)], cwd=tmp_path, capture_output=True, text=True)
    assert r.returncode == 0 and "fine" in r.stdout, r.stderr[-2000:]
