"""What importing the drop-in modules loads, and building the library alone."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "boa-constrictor_b200")


def _python(code):
    env = dict(os.environ, PYTHONPATH=PKG)
    r = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    return r.stdout


def test_operators_are_loaded_on_first_use():
    """The codec's modules do not map the operators' extension; the first operator call does."""
    out = _python("""
import boa, codec, gpu_range_coder, model, train, torch
from boa_b200 import ops
mapped = lambda: '_boa_ops' in open('/proc/self/maps').read()
m = model.BoaConstrictor(64, 1)
print(mapped())
try:
    ops.layer_norm(torch.zeros(2, 8), torch.ones(8))
except RuntimeError as e:
    print('no CPU path' in str(e), mapped())
try:
    ops.layer_norm(torch.zeros(2, 8), torch.ones(7))
except ValueError:
    print('again')
""").split()
    assert out == ["False", "True", "True", "again"]


def test_operators_that_are_not_built_raise():
    out = _python("""
import sys
sys.modules['boa_b200._boa_ops'] = None
import torch, model
from boa_b200 import ops
for _ in range(2):
    try:
        ops.layer_norm(torch.zeros(2, 8), torch.ones(8))
    except RuntimeError as e:
        print('not built' in str(e))
""").split()
    assert out == ["True", "True"]


def test_the_library_is_built_without_torch_headers(tmp_path):
    """`make lib` is every step of libboa_b200.so and none that wants torch or g++."""
    make = ["make", "-n", "-C", os.path.join(PKG, "csrc"), f"BUILD={tmp_path}", f"OUT={tmp_path}/libboa_b200.so",
            "PYTHON=false", "BIND_CXX=no-compiler", "lib"]
    out = subprocess.run(make, capture_output=True, text=True)
    assert out.returncode == 0, out.stderr
    assert "ssm.cu" in out.stdout and "libboa_b200.so" in out.stdout
    assert "no-compiler" not in out.stdout and "ops_bind" not in out.stdout
