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
