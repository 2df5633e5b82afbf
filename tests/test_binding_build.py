"""When the torch binding is built again, checked without a compiler run."""
import os

import pytest

from therock_b200 import build


@pytest.fixture
def compiles(monkeypatch, tmp_path):
    """Counts the compiler's runs; the result and the record go to a folder of the test's."""
    made = []

    def run(cmd, **kw):
        made.append(cmd)
        open(cmd[cmd.index("-o") + 1], "w").close()
        return type("Done", (), {"returncode": 0, "stdout": ""})
    monkeypatch.setattr(build.subprocess, "run", run)
    monkeypatch.setattr(build, "HERE", str(tmp_path))
    monkeypatch.setattr(build, "OBJ_DIR", str(tmp_path / "build"))
    return made


def test_a_binding_of_another_torch_is_built_again(compiles, monkeypatch):
    import torch
    out = build.build_binding()
    assert os.path.exists(out) and len(compiles) == 1
    build.build_binding()
    assert len(compiles) == 1                       # nothing has changed
    monkeypatch.setattr(torch, "__version__", "99.0")
    build.build_binding()
    assert len(compiles) == 2
    build.build_binding()
    assert len(compiles) == 2


def test_a_binding_without_a_record_is_built_again(compiles):
    build.build_binding()
    os.remove(os.path.join(build.OBJ_DIR, "_fmoe_torch.made_for"))
    build.build_binding()
    assert len(compiles) == 2
