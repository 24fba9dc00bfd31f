"""mineral_amd.ops without the library of the memory operators, or with one that this torch cannot load: the operators of the training
loops are there all the same, the others are not, and a warning names the reason."""

import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CODE = """
import os, warnings
import torch
{spoil}
with warnings.catch_warnings(record=True) as seen:
    warnings.simplefilter('always')
    import mineral_amd.ops as ops
assert any('memory operators' in str(w.message) and {reason!r} in str(w.message) for w in seen), [str(w.message) for w in seen]
assert 'gae_finish' in ops.OPS and 'linear_act' not in ops.OPS
assert torch.ops.mineral.param_count.default is not None
try:
    torch.ops.mineral.linear_act
except AttributeError:
    pass
else:
    raise SystemExit('linear_act is registered')
from mineral_amd import _hip
try:
    import mineral_amd.memory_ops
except (_hip.HipLibraryError, OSError):
    print('fine')
"""

MISSING = "real = os.path.exists\nos.path.exists = lambda p: not str(p).endswith('libmineral_torch.so') and real(p)"
FOREIGN = "def refuse(path):\n    raise OSError('undefined symbol')\ntorch.ops.load_library = refuse"


@pytest.mark.parametrize('spoil,reason', [(MISSING, 'not found'), (FOREIGN, 'undefined symbol')], ids=['missing', 'foreign'])
def test_the_other_operators_do_not_need_it(spoil, reason):
    run = subprocess.run([sys.executable, '-c', CODE.format(spoil=spoil, reason=reason)], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.strip() == 'fine', run.stdout + run.stderr
