"""The build where a part of it is missing: the library needs nvcc alone, the module for torch tensors g++ and torch as well."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def build():
    from wukong_b200 import build
    build.build()
    return build


@pytest.mark.parametrize("missing", ["import sys; sys.modules['torch'] = None", "import os; os.environ['PATH'] = '/nowhere'"])
def test_the_library_builds_without_torch_and_without_a_host_compiler(build, tmp_path, missing):
    """Only the module is left out then, and the build says so."""
    code = "%s\nfrom wukong_b200 import build\nbuild.CALLS_OUT = %r\nprint(build.build())" % (missing, str(tmp_path / "calls.so"))
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    assert r.stdout.strip() == build.OUT and "_torch_calls" in r.stderr and not (tmp_path / "calls.so").exists()


def test_the_library_loads_without_torch(build):
    code = "import sys; sys.modules['torch'] = None\nimport wukong_b200\nfrom wukong_b200.paged import BlockManager\nprint(BlockManager(4, 2, 1, 4).reserve(0, 3))"
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.strip() == "0", r.stderr
