"""CPU: when the torch extension is built again (nothing is compiled here: the compiler's call is recorded)."""
import os
import subprocess

import torch

from cpfn_amd import build


def test_the_extension_is_built_again_for_another_torch(tmp_path, monkeypatch):
    calls = []

    def compiler(cmd, **kw):
        calls.append(cmd)
        with open(build.NATIVE, "w") as f:
            f.write("built")
        return subprocess.CompletedProcess(cmd, 0, "", "")
    monkeypatch.setattr(build, "NATIVE", os.path.join(str(tmp_path), "_native.so"))
    monkeypatch.setattr(build, "OBJ", str(tmp_path))
    monkeypatch.setattr(build.subprocess, "run", compiler)
    build._build_native(False)
    assert len(calls) == 1 and calls[0][0] == "g++"
    build._build_native(False)
    assert len(calls) == 1
    monkeypatch.setattr(torch, "__version__", torch.__version__ + ".another")
    build._build_native(False)
    assert len(calls) == 2
    build._build_native(False)
    assert len(calls) == 2
    build._build_native(True)
    assert len(calls) == 3
