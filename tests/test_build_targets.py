"""What needs which built file: the library alone for the C ABI and the network's training, the torch extension for the operators beside it."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _python(code):
    return subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)


def test_training_starts_without_the_extension():
    got = _python("import sys; sys.modules['erfnet_pytorch_amd._host'] = None\n"
                  "from erfnet_pytorch_amd import loss, trainer\n"
                  "loss.CrossEntropyLoss2d()\n"
                  "try:\n    loss.class_log_probs(None)\n"
                  "except ImportError as e:\n    print(e)\n")
    assert got.returncode == 0 and "build it" in got.stdout, got.stderr


def test_operators_that_need_the_extension_say_how_to_build_it():
    for name in ("norm", "optim", "train_ops"):
        got = _python(f"import sys; sys.modules['erfnet_pytorch_amd._host'] = None\nfrom erfnet_pytorch_amd import {name}")
        assert got.returncode != 0 and "build it" in got.stderr


def test_the_operators_are_registered_with_the_loss():
    got = _python("import torch\nfrom erfnet_pytorch_amd import loss\nprint(torch.ops.erfnet_mi355.class_log_probs_fwd.default)")
    assert got.returncode == 0 and "class_log_probs_fwd" in got.stdout, got.stderr


def test_the_library_is_built_without_torch():
    def plan(*args):
        got = subprocess.run(["make", "-C", os.path.join(ROOT, "erfnet_pytorch_amd", "csrc"), "-n", "-B", *args], capture_output=True, text=True)
        assert got.returncode == 0, got.stderr
        return "../libermi355.so" in got.stdout, "../_host.so" in got.stdout
    assert plan() == (True, True) and plan("PY=false") == (True, False) and plan("lib") == (True, False)
