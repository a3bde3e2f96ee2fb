"""What importing the package does and does not need. Each check runs in an interpreter of its own."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def run(code):
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    return r.stdout


def test_import_maps_no_extension():
    """Binaries are loaded by the first call that needs them."""
    out = run("import rgpt_b200, rgpt_b200.model, rgpt_b200.native, rgpt_b200.optimizer, rgpt_b200.losses, rgpt_b200.trainer\n"
              "import sys\nassert 'rgpt_b200._fastargs' not in sys.modules\n"
              "print([l.split()[-1] for l in open('/proc/self/maps') if 'rgpt_b200' in l])")
    assert out.strip() == "[]"


def test_the_first_call_loads_the_argument_checks():
    run("import importlib.util, sys, torch\nfrom rgpt_b200 import native as nv\n"
        "o = torch.zeros(4)\n"
        "try:\n    nv.token_logprobs(torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64), o)\n"
        "except RuntimeError as e:\n    assert 'CUDA' in str(e)\n"
        "else:\n    raise SystemExit('a CPU tensor went through')\n"
        "if importlib.util.find_spec('rgpt_b200._fastargs'):\n"
        "    from rgpt_b200 import _fastargs\n    assert nv._pack is _fastargs.pack\n")


def test_import_without_cuda_in_torch():
    """A torch built without CUDA lacks these names."""
    run("import torch\n"
        "for n in ('_cuda_getDevice', '_cuda_getCurrentRawStream'):\n"
        "    if hasattr(torch._C, n): delattr(torch._C, n)\n"
        "import rgpt_b200.model, rgpt_b200.optimizer, rgpt_b200.losses\nfrom rgpt_b200 import native as nv\n"
        "o = torch.zeros(4)\n"
        "try:\n    nv.token_logprobs(torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64), o)\n"
        "except RuntimeError as e:\n    assert 'CUDA' in str(e)\n"
        "else:\n    raise SystemExit('a CPU tensor went through')\n")
