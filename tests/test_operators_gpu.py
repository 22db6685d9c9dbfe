"""The operators of optim.adamw_step and routing on a real MI355X: the cases of tests/operator_cases.py through the HIP library, and
what only a GPU run shows (streams, recorded graphs)."""
import os

import pytest
import torch

import operator_cases as oc
from mneslam_amd import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def real_library():
    if not torch.cuda.is_available():
        pytest.skip("these tests need an MI355X", allow_module_level=False)
    _lib.unload()
    lib = _lib.load()
    assert os.path.samefile(lib._name, _lib.LIB_PATH)
    yield
    torch.cuda.synchronize()


TYPES = [("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32")]


@pytest.mark.parametrize("ptype,gtype", TYPES)
def test_adamw_32(ptype, gtype):
    oc.check_adamw32(DEV, ptype, gtype)


@pytest.mark.parametrize("ptype,gtype", TYPES)
def test_adamw_8(ptype, gtype):
    oc.check_adamw8(DEV, ptype, gtype)
