"""Which objects a build compiles anew."""
import importlib.util
import os
from pathlib import Path

import pytest

PATH = Path(__file__).resolve().parent.parent / "torchpairwise_b200" / "build.py"


@pytest.fixture
def build(tmp_path):
    script = tmp_path / "build.py"
    script.write_text(PATH.read_text())
    spec = importlib.util.spec_from_file_location("tpw_build_under_test", script)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_an_object_depends_on_its_source_its_headers_and_the_build_script(build, tmp_path):
    src, direct, nested, other, obj = (tmp_path / n for n in ("a.cu", "direct.cuh", "nested.cuh", "other.cuh", "a.o"))
    src.write_text('#include "direct.cuh"\n#include <cstdio>\n')
    direct.write_text('#include "nested.cuh"\n')
    nested.write_text("")
    other.write_text("")
    files = [src, direct, nested, other, Path(build.__file__)]

    def touched(path):
        for f in files:
            os.utime(f, (1000, 1000))
        os.utime(obj, (2000, 2000))
        if path is not None:
            os.utime(path, (3000, 3000))
        return build._obj_stale(src, obj)

    assert build._obj_stale(src, obj)   # there is none yet
    obj.write_text("")
    assert not touched(None) and not touched(other)
    for path in (src, direct, nested, Path(build.__file__)):
        assert touched(path), path.name
