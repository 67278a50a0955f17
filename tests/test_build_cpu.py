"""The build where a part of it is missing: the library needs nvcc alone, the module for torch tensors g++ and torch as well."""
import os
import subprocess
import sys
from types import SimpleNamespace

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


def test_another_torch_rebuilds_the_module(build, monkeypatch, tmp_path):
    import torch
    ran = []
    monkeypatch.setattr(build, "run_host_compiler", lambda cmd, verbose: ran.append(cmd))
    monkeypatch.setattr(build, "CALLS_FOR", str(tmp_path / "for"))
    build.build_calls()
    assert len(ran) == 1, "nothing says for which torch it was built"
    build.build_calls()
    assert len(ran) == 1
    monkeypatch.setattr(torch, "__version__", "1.0.0+other")
    build.build_calls()
    assert len(ran) == 2 and any("1.0.0+other" in a for a in ran[1])


def test_a_module_for_another_torch_is_refused(build, monkeypatch):
    import torch
    import wukong_b200
    from wukong_b200 import _lib, device
    device._calls()                                        # the one that was built is fine
    monkeypatch.setattr(device, "_calls_module", None)
    fake = SimpleNamespace(torch_version="1.0.0+other", set_error=lambda e: None)
    monkeypatch.setattr(wukong_b200, "_torch_calls", fake, raising=False)
    monkeypatch.setitem(sys.modules, "wukong_b200._torch_calls", fake)
    with pytest.raises(_lib.WukongB200Error, match="1.0.0"):
        device.token_probs(torch.zeros(1, 1))
