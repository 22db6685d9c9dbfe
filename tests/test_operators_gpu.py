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


# ------------------------------------------------------------------------------------------------------------ only on a GPU
def test_adamw_far_elements():
    """Elements beyond 2^31 of one tensor."""
    import numpy as np
    from mneslam_amd import optim
    n = (1 << 31) + (1 << 16) + 77
    for bits in (8, 32):
        p = torch.ones(n, device=DEV, dtype=torch.bfloat16)
        g = torch.full((n,), 0.25, device=DEV, dtype=torch.bfloat16)
        tail = 256 * 40 + 77
        gen = torch.Generator().manual_seed(1)
        p[-tail:] = torch.randn(tail, generator=gen).bfloat16().to(DEV)
        g[-tail:] = torch.randn(tail, generator=gen).bfloat16().to(DEV)
        state = oc._state_for(p, bits, DEV)
        p0, g0 = oc._np(p[-tail:]), oc._np(g[-tail:])
        oc._step([p], [g], bits, DEV, state=[state], seed=3)
        want_p, want_m, want_v = oc.adamw64(p0, g0, np.zeros(tail), np.zeros(tail), 1, 0.01, (0.9, 0.99), 1e-8, 0.0)
        oc.assert_rounded(p[-tail:], want_p, 18 * oc.EPS32 * 0.011 + 4 * oc.EPS32 * np.abs(p0), bits)
        if bits == 32:
            assert np.abs(oc._np(state[0][0][-tail:]) - want_m).max() <= 1e-6 and float(state[0][1][0]) > 0
        else:
            z = np.zeros(tail, np.int8)
            mc, rc, sc, _, _ = oc.adamw8_ieee(g0.astype(np.float32), z, z.astype(np.uint8), np.zeros((41, 2), np.float32), 3, 0, 1, (0.9, 0.99), start=n - tail)
            assert np.array_equal(oc._np(state[0][0][-tail:]), mc) and np.array_equal(oc._np(state[0][1][-tail:]), rc)
            assert np.array_equal(state[1][-41:].cpu().numpy(), sc)
            m, v = optim.adamw_moments(*state[0], state[1])
            assert np.array_equal(oc._np(m[-tail:]), oc.values8(mc, rc, sc)[0].astype(np.float64))
            del m, v
        del p, g, state
        torch.cuda.empty_cache()


def test_expert_rows_far():
    """Rows beyond 4 GB, in and out."""
    from mneslam_amd.routing import expert_combine, expert_dispatch, expert_sort
    n, k, width, experts = 600011, 2, 2048, 16
    gen = torch.Generator(device=DEV).manual_seed(5)
    ids = torch.randint(0, experts, (n, k), generator=gen, device=DEV)
    ids[::17, 1] = -1
    plan = expert_sort(ids, experts)
    x = torch.randn(n, width, generator=gen, device=DEV).bfloat16()
    w = torch.rand(n, k, generator=gen, device=DEV)
    xs = expert_dispatch(x, plan)
    some = torch.cat([torch.randint(0, n, (200,), generator=gen, device=DEV), torch.tensor([0, n - 1], device=DEV)])
    pos = plan.position[some].long()
    held = pos >= 0
    assert torch.equal(xs[pos.clamp(min=0)][held], x[some][:, None].expand(-1, k, -1)[held]) and not xs[int(plan.live):].any()
    # the dispatched rows have far places too: combined with weights, and differentiated
    xs.requires_grad_(True)
    w.requires_grad_(True)
    out = expert_combine(xs, plan, w)
    dy, dw = torch.autograd.grad(out, (xs, w), x)
    share = torch.where(held, w.detach()[some], 0.0)
    want = (share.double().sum(1, keepdim=True) * x[some].double())
    assert ((out.detach()[some].double() - want).abs() <= 2.0 ** -8 * want.abs() * 1.01 + 1e-30).all()
    dots = torch.where(held, x[some].double().square().sum(1, keepdim=True), 0.0)
    assert ((dw[some].double() - dots).abs() <= width * oc.EPS32 * dots).all()
    rows = dy[pos.clamp(min=0)].double()
    want = share.double()[..., None] * x[some].double()[:, None]
    assert ((torch.where(held[..., None], rows, 0.0) - want).abs() <= 2.0 ** -8 * want.abs() * 1.01 + 1e-30).all()
    assert not dy[int(plan.live):].any()


def test_streams():
    """Inputs that another stream still writes: the calls run on the current stream, behind them."""
    from mneslam_amd import optim
    from mneslam_amd.routing import expert_combine, expert_dispatch, expert_sort
    gen = torch.Generator().manual_seed(6)
    ids, x = torch.randint(0, 5, (3000, 2), generator=gen).to(DEV), torch.randn(3000, 33, generator=gen).to(DEV)
    plan = expert_sort(ids, 5)
    want = expert_combine(expert_dispatch(x, plan), plan)
    big = torch.empty(1 << 28, device=DEV)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:                                       # at the same time on two streams
        with torch.cuda.stream(s):
            late_ids, late_x = torch.empty_like(ids).fill_(-1), torch.zeros_like(x)
            for _ in range(8):
                big.fill_(1.0)
            late_ids.copy_(ids)
            late_x.copy_(x)
            a = late_x.requires_grad_(True)
            p = expert_sort(late_ids, 5)
            out = expert_combine(expert_dispatch(a, p), p)
            grad, = torch.autograd.grad(out, a, torch.ones_like(out))
            q, g = torch.ones(5000, device=DEV), torch.zeros(5000, device=DEV)
            big.fill_(2.0)
            g += 1.0
            state = oc._step([q], [g], 8, DEV)
            got.append((out.detach(), grad, q, state[0][0][0]))
    torch.cuda.synchronize()
    for out, grad, q, codes in got:
        assert torch.equal(out, want) and torch.equal(grad, torch.full_like(grad, 2.0))
        assert (q - 0.99).abs().max() < 1e-6 and (codes == 127).all()


def test_routing_recorded():
    """Sort, both row movements and their gradients in a recorded graph, replayed on other inputs between eager calls; two graphs."""
    from mneslam_amd.routing import expert_combine, expert_dispatch, expert_sort
    gen = torch.Generator().manual_seed(9)

    def inputs(n, k, d, experts):
        ids = oc.make_ids("masked", n, k, experts, gen)
        return [ids.to(DEV), torch.randn(n, d, generator=gen).bfloat16().to(DEV), torch.randn(n * k, d, generator=gen).bfloat16().to(DEV),
                torch.rand(n, k, generator=gen).to(DEV), torch.randn(n * k, d, generator=gen).bfloat16().to(DEV),
                torch.randn(n, d, generator=gen).bfloat16().to(DEV)]

    def work(ids, x, y, w, gx, go, experts):
        x, y, w = (t.detach().requires_grad_(True) for t in (x, y, w))
        plan = expert_sort(ids, experts)
        xs, out = expert_dispatch(x, plan), expert_combine(y, plan, w)
        grads = torch.autograd.grad((xs, out), (x, y, w), (gx, go))
        return [plan.order, plan.position, plan.offsets, xs.detach(), out.detach(), *grads]

    graphs = []
    for shape in ((700, 2, 40, 6), (9000, 3, 64, 300)):                   # the short sort and the long one
        static = inputs(*shape)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            work(*static, shape[3])
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            result = work(*static, shape[3])
        graphs.append((shape, static, graph, result))
    for _ in range(4):
        for shape, static, graph, result in graphs:
            fresh = inputs(*shape)
            want = work(*fresh, shape[3])                                  # eager work between the replays
            for s, f in zip(static, fresh):
                s.copy_(f)
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(result, want):
                assert torch.equal(a, b)


def test_routing_recorded_beside_an_eager_graph():
    """Recording a backward pass whose leaves an eager graph on the default stream holds is refused; without that graph it is recorded."""
    from mneslam_amd.routing import expert_combine, expert_dispatch, expert_sort
    ids = torch.tensor([[0, 1], [2, 0], [1, -1]], device=DEV)
    x, w = torch.randn(3, 8, device=DEV, requires_grad=True), torch.rand(3, 2, device=DEV, requires_grad=True)

    def work():
        plan = expert_sort(ids, 3)
        return expert_combine(expert_dispatch(x * 1.0, plan), plan, w)

    eager = work()
    with pytest.raises(RuntimeError, match="default stream"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            torch.autograd.grad(work().sum(), (x, w))
    want = torch.autograd.grad(eager.sum(), (x, w))
    del eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(work().sum(), (x, w))
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_recorded(bits):
    """A step with a clock in a recorded graph equals eager steps; without one it is refused."""
    from mneslam_amd import optim
    clock, offset, table = oc.check_adamw_clock(DEV, bits)
    offset.zero_()
    gen = torch.Generator().manual_seed(10)
    grads = [torch.randn(5000, generator=gen).to(DEV) for _ in range(4)]
    p, q, g = torch.ones(5000, device=DEV), torch.ones(5000, device=DEV), grads[0].clone()
    state = oc._state_for(p, bits, DEV)
    lib = _lib.load()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        oc._step([p], [g], bits, DEV, step=1, state=[state], clock=clock)
        _lib.check(lib.mne_clock_advance(None, offset.data_ptr(), _lib.stream_for(p)), "mne_clock_advance")
    assert (p == 1).all()
    other = None
    for k, fresh in enumerate(grads):
        g.copy_(fresh)
        graph.replay()
        other = oc._step([q], [fresh], bits, DEV, step=1 + k, state=other)
        torch.cuda.synchronize()
        assert torch.equal(p, q) and all(torch.equal(a, b) for a, b in zip(state[0], other[0][0])), k
    graph2 = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="clock"):
        with torch.cuda.graph(graph2):
            oc._step([p], [g], bits, DEV, step=1, state=[state])
    opt = optim.FusedAdamW([torch.nn.Parameter(torch.ones(10, device=DEV))], state_bits=bits)
    opt.param_groups[0]["params"][0].grad = torch.ones(10, device=DEV)
    with pytest.raises(RuntimeError, match="before recording"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step(clock=clock)
    torch.cuda.synchronize()


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
