"""The operators of optim.adamw_step and routing through the host emulator (tests/hostemu): the same kernel sources on CPU tensors.
The GPU run of the same cases is tests/test_operators_gpu.py."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "hostemu"))

import operator_cases as oc  # noqa: E402
from mneslam_amd import _lib  # noqa: E402

DEV = "cpu"


@pytest.fixture(scope="module", autouse=True)
def emulator_library():
    import build_emu
    from mneslam_amd import build
    build.build_host()
    path = build_emu.build()
    _lib.unload()
    _lib.load(path)
    torch.set_num_threads(2)
    yield
    _lib.unload()


TYPES = [("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32")]


@pytest.mark.parametrize("ptype,gtype", TYPES)
def test_adamw_32(ptype, gtype):
    oc.check_adamw32(DEV, ptype, gtype)


@pytest.mark.parametrize("ptype,gtype", TYPES)
def test_adamw_8(ptype, gtype):
    oc.check_adamw8(DEV, ptype, gtype)
