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


def test_agent_maps(tmp_path):
    oc.check_agent_maps(DEV, tmp_path)


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("ptype", ["f32", "bf16"])
def test_mixture_step(bits, ptype):
    oc.check_mixture_step(DEV, bits, ptype)


def test_adamw_refusals():
    oc.check_adamw_refusals(DEV)


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_nonfinite(bits):
    oc.check_adamw_nonfinite(DEV, bits)


def test_adamw_8_poisoned():
    oc.check_adamw8_poisoned(DEV)


def test_adamw_shared_state():
    oc.check_adamw_shared_state(DEV)


def test_adamw_loads_no_other_rule():
    oc.check_adamw_loads_no_other_rule(DEV)


def test_combine_keeps_what_it_needs():
    oc.check_combine_keeps_what_it_needs(DEV)


def test_adamw_8_small_and_zero():
    oc.check_adamw8_small_and_zero(DEV)


def test_adamw_8_dither():
    oc.check_adamw8_dither(DEV)


def test_fused_adamw():
    oc.check_fused_adamw(DEV)


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_many_tensors(bits):
    oc.check_adamw_many(DEV, 170, bits)


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("ptype", ["f32", "bf16"])
def test_adamw_flat_buffers(bits, ptype):
    oc.check_adamw_flat(DEV, bits, ptype)


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_clock(bits):
    oc.check_adamw_clock(DEV, bits)


def test_routing_refusals():
    oc.check_routing_refusals(DEV)


def test_routing_views():
    oc.check_routing_views(DEV)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("width", [1, 6])
def test_routing_of_negated_views(dtype, width):
    oc.check_negated_rows(DEV, dtype, width)


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_of_negated_views(bits):
    oc.check_negated_adamw(DEV, bits)


def test_operators_are_not_traced():
    oc.check_not_traced(DEV)


def test_zeros_without_memory():
    oc.check_zeros_without_memory(DEV)


def test_rows_are_copied_once():
    oc.check_rows_copied_once(DEV)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_expert_rows_infinite(dtype):
    oc.check_infinite_rows(DEV, dtype)


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("ptype", ["f32", "bf16", "f16"])
def test_adamw_tiny_eps(ptype, bits):
    oc.check_adamw_tiny_eps(DEV, ptype, bits)


def test_adamw_8_quotient():
    oc.check_adamw8_quotient(DEV)


def test_plane_gradients():
    oc.check_plane_gradients(DEV)


def test_plane_gradients_rendered():
    oc.check_plane_gradients_rendered(DEV)


def test_agent_maps_have_no_seam():
    oc.check_agent_maps_have_no_seam(DEV)


def test_fused_adamw_loads_all_or_nothing():
    oc.check_fused_adamw_loads_all_or_nothing(DEV)


def test_fused_adamw_loads_no_other_decay():
    oc.check_fused_adamw_loads_no_other_decay(DEV)


def test_fused_adamw_keeps_its_bits():
    oc.check_fused_adamw_keeps_its_bits(DEV)


def test_fused_adamw_steps_all_or_nothing():
    oc.check_fused_adamw_steps_all_or_nothing(DEV)


def test_adamw_gradient_in_written_memory():
    oc.check_adamw_gradient_in_written_memory(DEV)


def test_adamw_outdates_what_it_writes():
    oc.check_adamw_outdates_what_it_writes(DEV)


def test_plan_tensors_are_apart():
    oc.check_plan_tensors_are_apart(DEV)


def test_adamw_8_follows_32():
    oc.check_adamw8_follows_32(DEV)


def test_fused_adamw_loads_no_scales_with_32_bits():
    oc.check_fused_adamw_loads_no_scales_with_32_bits(DEV)
