"""The build of the serving libraries' torch binding: left out where there is no torch, and never one of another torch or Python."""
import os
import subprocess
import sys
import sysconfig

import torch

from reax_engine_kernels_b200 import build as B

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_libraries_build_without_torch():
    """The C ABI needs no torch: the build ends well where it cannot be imported, and says what it left out."""
    code = ("import sys; sys.modules['torch'] = None\n"
            "from reax_engine_kernels_b200 import build as B\n"
            "B.build_library = lambda name, force=False, verbose=False: 'lib/' + name\n"  # compiled elsewhere
            "print(sorted(B.build_libraries()))")
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    assert "skipped _serving" in r.stdout
    assert r.stdout.strip().splitlines()[-1] == str(sorted("lib/" + n for n in B.LIBRARIES))


def test_no_binding_for_a_torch_without_cuda(monkeypatch, capsys):
    monkeypatch.setattr(torch.version, "cuda", None)
    assert B.build_binding(force=True) is None
    assert "skipped _serving" in capsys.readouterr().out


def test_binding_of_another_torch_or_python_is_not_kept(monkeypatch, tmp_path):
    """What lies there is used again only under the torch and the Python that it was built for; a new one takes the others' place."""
    built = []

    def run(cmd, what):
        built.append(what)
        open(cmd[cmd.index("-o") + 1], "w").close()

    monkeypatch.setattr(B, "LIBDIR", str(tmp_path))
    monkeypatch.setattr(B, "_run", run)
    (tmp_path / "_serving.so").touch()
    first = B.build_binding()
    assert B.build_binding() == first and built == ["_serving"] and os.listdir(tmp_path) == [os.path.basename(first)]
    monkeypatch.setattr(torch, "__version__", "9.9.9+cu999")
    other = B.build_binding()
    assert other != first and built == ["_serving"] * 2 and os.listdir(tmp_path) == [os.path.basename(other)]
    monkeypatch.setattr(sysconfig, "get_config_var", lambda name: "cpython-399")
    third = B.build_binding()
    assert third not in (first, other) and built == ["_serving"] * 3 and os.listdir(tmp_path) == [os.path.basename(third)]
