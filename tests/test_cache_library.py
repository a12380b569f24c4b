"""The package without the library of the quantised cache: everything else imports and runs, its functions say what is missing."""
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

PACKAGE = Path(__file__).resolve().parent.parent / "torchpairwise_b200"
CODE = """
import torch, torchpairwise_b200 as tpw
assert tpw.__file__.startswith({root!r}), tpw.__file__
x, n = torch.zeros(1, 3, 2, 8), torch.zeros(1, dtype=torch.int32)
cache = tpw.quantized_cache(1, 3, 2, 8, device="cpu")
for call in (lambda: tpw.cache_write(cache, x, x, n), lambda: tpw.cache_read(cache, n), lambda: tpw.cache_attention(x, cache, n)):
    try:
        call()
    except ImportError as e:
        assert {text!r} in str(e) and "build.py" in str(e), e
    else:
        raise AssertionError("no ImportError")
try:
    tpw.attention(x, x, x)
except RuntimeError as e:
    assert "CUDA" in str(e), e
print("fine")
"""


@pytest.mark.parametrize("state,text", [("missing", "is missing"), ("of another torch", "does not load")])
def test_the_package_imports_without_the_cache_library(tmp_path, state, text):
    root = tmp_path / "torchpairwise_b200"
    (root / "lib").mkdir(parents=True)
    for source in PACKAGE.glob("*.py"):
        shutil.copy(source, root)
    for name in ("libtpw_b200.so", "libtpw_b200_attention.so"):
        (root / "lib" / name).symlink_to(PACKAGE / "lib" / name)
    if state != "missing":
        (root / "lib" / "libtpw_b200_cache.so").write_bytes(b"not a library that this interpreter can load")
    r = subprocess.run([sys.executable, "-c", CODE.format(root=str(tmp_path), text=text)], cwd=tmp_path, capture_output=True, text=True)
    assert r.returncode == 0 and "fine" in r.stdout, r.stderr[-2000:]
