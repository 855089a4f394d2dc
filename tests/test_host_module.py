"""The host module of the language-model operators: loading and rebuilding, without a GPU."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_host_module_loads_before_torch_is_imported():
    # a process that has not imported torch, with nothing to build
    res = subprocess.run([sys.executable, "-c", "import sys\n"
                          "from mk_iii_technologies_tsrn_b200 import _lib\n"
                          "assert 'torch' not in sys.modules\n"
                          "_lib.host()\n"], cwd=ROOT, capture_output=True, text=True)
    assert res.returncode == 0, res.stderr


def test_host_module_is_rebuilt_for_another_torch(tmp_path, monkeypatch):
    from mk_iii_technologies_tsrn_b200 import build
    module, stamp = tmp_path / "module.so", tmp_path / "module.for"
    monkeypatch.setattr(build, "HOST_PATH", str(module))
    monkeypatch.setattr(build, "HOST_STAMP", str(stamp))
    module.write_bytes(b"")
    assert build.needs_host_build()                       # nothing says what it was built for
    stamp.write_text(build._host_target())
    assert not build.needs_host_build()
    stamp.write_text(build._host_target().replace("torch ", "torch 1."))
    assert build.needs_host_build()
