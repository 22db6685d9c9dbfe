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


SORTS = [(1, 1, 1), (1, 2, 8), (3, 2, 1), (0, 2, 5), (64, 1, 64), (65, 3, 7), (1000, 2, 129), (4097, 4, 33), (777, 8, 2000), (300, 2, 2001),
         (5000, 4, 4096)]


@pytest.mark.parametrize("kind", ["even", "hot", "none", "last", "masked", "outside"])
@pytest.mark.parametrize("n,k,experts", SORTS)
def test_expert_sort(n, k, experts, kind):
    oc.check_expert_sort(DEV, n, k, experts, kind, wide=(n + experts) % 2 == 0 or kind == "outside")


# widths of one element, below and beyond a piece, odd, one wave's columns and more
ROWS = [(1, 2, 8, 1024, 1024), (5, 1, 3, 1, 1), (33, 3, 4, 3, 4), (70, 2, 9, 8, 7), (129, 2, 6, 65, 65), (17, 8, 40, 130, 129),
        (9, 5, 4, 520, 257), (6, 4, 3, 2051, 1030), (40, 6, 5, 16, 16), (0, 2, 3, 8, 8), (4, 2, 3, 0, 0)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kind", ["even", "masked"])
@pytest.mark.parametrize("n,k,experts,width,out_width", ROWS)
def test_expert_rows(dtype, kind, n, k, experts, width, out_width):
    oc.check_expert_rows(DEV, dtype, n, k, experts, width, out_width, kind, odd=(n + width) % 2 == 1 and n > 1)


@pytest.mark.parametrize("dtype,wtype", [("f32", "bf16"), ("bf16", "bf16"), ("f16", "f32")])
@pytest.mark.parametrize("need", [("x",), ("y",), ("w",), ("x", "w"), ("y", "w"), ()])
def test_expert_rows_needed_gradients(dtype, wtype, need):
    oc.check_expert_rows(DEV, dtype, 50, 3, 5, 24, 33, "masked", odd=True, wtype=wtype, need=need)


@pytest.mark.parametrize("kind", ["hot", "none", "outside"])
def test_expert_rows_batches(kind):
    oc.check_expert_rows(DEV, "bf16", 130, 2, 7, 40, 24, kind, odd=False)


# enough tokens for several columns a lane (forms of one to four), with one, two and more choices
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,k,width,out_width", [(9001, 1, 65, 65), (16000, 2, 100, 33), (3001, 5, 512, 1027), (140000, 2, 3, 4), (1025, 3, 1024, 2050)])
def test_expert_rows_large(dtype, n, k, width, out_width):
    oc.check_expert_rows(DEV, dtype, n, k, 37, width, out_width, "masked", odd=width % 2 == 1)


@pytest.mark.parametrize("kind", ["even", "hot", "masked"])
@pytest.mark.parametrize("n,k,experts", [(275200, 2, 8), (1 << 20, 1, 4096), (700001, 3, 100)])
def test_expert_sort_large(n, k, experts, kind):
    oc.check_expert_sort(DEV, n, k, experts, kind, wide=k == 1)
