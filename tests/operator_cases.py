"""Bodies of the operator tests, shared by the host-emulator run (CPU) and the GPU run: each compares an operator with a plain
implementation in 64 bits (codes of 8-bit moments: in IEEE 32-bit arithmetic, bit for bit)."""
import numpy as np
import pytest
import torch

from mneslam_amd import optim

U32 = 0xFFFFFFFF
GOLD, MIX1, MIX2 = 0x9E3779B1, 0x7FEB352D, 0x846CA68B
EPS32 = 2.0 ** -24                      # half a step of fp32, relative
NAMES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ---------------------------------------------------------------------------------------------------------------- AdamW
def constants(step, lr, betas, wd):
    return lr / (1.0 - betas[0] ** step), np.sqrt(1.0 - betas[1] ** step), 1.0 - lr * wd


def adamw64(p, g, m, v, step, lr, betas, eps, wd):
    """One step in 64 bits on float64 arrays -> (p, m, v)."""
    size, root_bc2, decay = constants(step, lr, betas, wd)
    m = betas[0] * m + (1.0 - betas[0]) * g
    v = betas[1] * v + (1.0 - betas[1]) * g * g
    return p * decay - size * (m / (np.sqrt(v) / root_bc2 + eps)), m, v


def mix(h):
    h = ((h ^ (h >> np.uint64(16))) * np.uint64(MIX1)) & np.uint64(U32)
    h = ((h ^ (h >> np.uint64(15))) * np.uint64(MIX2)) & np.uint64(U32)
    return h ^ (h >> np.uint64(16))


def dither(seed, ordinal, step, n):
    """u_m, u_r of the n elements of a tensor (float32, multiples of 2^-16)."""
    i = np.arange(n, dtype=np.uint64)
    key = mix(np.uint64((seed + ordinal * GOLD) & U32))
    key = mix(((key + np.uint64(step * GOLD & U32)) & np.uint64(U32)) ^ mix((i >> np.uint64(8)) & np.uint64(U32)))
    h = (key + (i & np.uint64(255)) * np.uint64(GOLD)) & np.uint64(U32)
    h = ((h ^ (h >> np.uint64(16))) * np.uint64(MIX1)) & np.uint64(U32)
    h = h ^ (h >> np.uint64(15))
    return (h & np.uint64(0xFFFF)).astype(np.float32) / np.float32(65536), (h >> np.uint64(16)).astype(np.float32) / np.float32(65536)


def values8(mc, rc, scales):
    """m and sqrt(v) in fp32 arithmetic, from int8 / uint8 codes and [blocks, 2] scales."""
    n = mc.size
    s = np.repeat(scales.astype(np.float32), 256, 0)[:n]
    c, d = mc.astype(np.float32), rc.astype(np.float32)
    return c * np.abs(c) * s[:, 0], d * d * s[:, 1]


def encode8(x, u, top, most, least):
    """Codes and scales of |m| or sqrt(v), IEEE fp32 as the operator defines it."""
    f, n = np.float32, x.size
    blocks = -(-n // 256)
    pad = np.zeros(blocks * 256, f)
    pad[:n] = x
    pad = pad.reshape(blocks, 256)
    fine = np.isfinite(pad).all(1)
    big = np.where(fine, pad.max(1, initial=0), f(0)).astype(f)
    some = fine & (big > f(least))
    safe = np.where(some, big, f(1))
    inv = np.where(some, f(top) / safe, f(0)).astype(f)
    scale = np.where(fine, np.where(some, safe / f(top), f(0)), f(np.nan)).astype(f)
    y = np.where(some[:, None], pad, f(0)) * inv[:, None]
    c = np.floor(np.sqrt(y.astype(np.float64))).astype(f)
    uu = np.zeros(blocks * 256, f)
    uu[:n] = u
    c = c + (uu.reshape(blocks, 256) * (f(2) * c + f(1)) < y - c * c).astype(f)
    return np.minimum(c, f(most)).reshape(-1)[:n], scale, np.repeat(some, 256)[:n]


def adamw8_ieee(g, mc, rc, scales, seed, ordinal, step, betas):
    """New codes and scales, bit for bit (g float32)."""
    f = np.float32
    b1, o1, b2, o2 = f(betas[0]), f(1.0 - betas[0]), f(betas[1]), f(1.0 - betas[1])
    with np.errstate(all="ignore"):
        m, r = values8(mc, rc, scales)
        m = m * b1 + g * o1
        r = np.sqrt((r * r) * b2 + (g * g) * o2)
        um, ur = dither(seed, ordinal, step, g.size)
        cm, sm, _ = encode8(np.abs(m), um, 16129, 127, 2.0 ** -100)
        cr, sr, some = encode8(r, ur, 65025, 255, 0)
        cr = np.where((cr == 0) & (r > 0) & some, f(1), cr)
        return np.where(m < 0, -cm, cm).astype(np.int8), cr.astype(np.uint8), np.stack([sm, sr], 1), m, r


def _np(t):
    """The tensor's memory in order, as a float64 / integer array."""
    t = t.detach().cpu()
    flat = torch.as_strided(t, (t.numel(),), (1,), t.storage_offset())
    return flat.double().numpy() if flat.is_floating_point() else flat.numpy()


def assert_rounded(t, want, tol, what):
    """``t`` is ``want`` up to ``tol`` (which counts fp32's own roundings), rounded to t's type once: half a step of the type, half of its
    smallest number, and infinity from where half a step above its largest number begins."""
    got, info = _np(t), torch.finfo(t.dtype)
    if t.dtype != torch.float32:
        tol = tol + info.eps / 2 * (np.abs(want) + tol) + info.smallest_normal * info.eps / 2
        edge = info.max * (1.0 + info.eps / 4)
        over = np.isinf(got) & np.isfinite(want) & (np.sign(got) == np.sign(want)) & (np.abs(want) + tol >= edge)
        got = np.where(over, want, got)
    with np.errstate(invalid="ignore"):
        off = np.where(got == want, -1.0, np.abs(got - want) - tol - 1e-44)          # (an infinity that is wanted included)
    assert (off <= 0).all(), (what, int(off.argmax()), got[off.argmax()], want[off.argmax()], tol[off.argmax()])


SHAPES = [(1, 32, 9, 7), (16, 32), (3, 33), (5,), (1,), (0,), (4097,), (256,), (255,), (2, 257)]


def _inputs(ptype, gtype, seed, device, shapes=SHAPES):
    """Tensors of odd sizes; the first is channels_last, one starts at an odd element of its storage, one gradient is transposed."""
    gen = torch.Generator().manual_seed(seed)
    ps, gs = [], []
    for k, s in enumerate(shapes):
        p, g = torch.randn(s, generator=gen), torch.randn(s, generator=gen) * 10.0 ** (k % 4 - 3)
        g = g * (torch.rand(s, generator=gen) > 0.3)
        p, g = p.to(NAMES[ptype]).to(device), g.to(NAMES[gtype]).to(device)
        if k == 0 and len(s) == 4:
            p = p.contiguous(memory_format=torch.channels_last)          # the gradient stays contiguous: copied by the step
        if k == 2:
            base = torch.zeros(p.numel() + 1, dtype=p.dtype, device=device)
            base[1:] = p.reshape(-1)
            p = base[1:].view(p.shape)
        if k == 1:
            g = g.t().contiguous().t()
        ps.append(p)
        gs.append(g)
    return ps, gs


def _as_param(g, p):
    return torch.empty_like(p, dtype=g.dtype).copy_(g)


def check_adamw32(device, ptype, gtype, wd=0.01, eps=1e-8, betas=(0.9, 0.99), steps=(1, 2, 50), lr=0.01):
    ps, gs = _inputs(ptype, gtype, 5, device)
    ms, vs = [torch.zeros_like(p, dtype=torch.float32) for p in ps], [torch.zeros_like(p, dtype=torch.float32) for p in ps]
    for n, step in enumerate(steps):
        before = [(_np(p).copy(), _np(_as_param(g, p)).copy(), _np(m).copy(), _np(v).copy()) for p, g, m, v in zip(ps, gs, ms, vs)]
        last = n == len(steps) - 1
        zero = [_as_param(g, p) for g, p in zip(gs, ps)] if last else gs
        optim.adamw_step(ps, zero, ms, vs, step=step, lr=lr, betas=betas, eps=eps, weight_decay=wd, zero_grad=last)
        for p, m, v, (p0, g0, m0, v0) in zip(ps, ms, vs, before):
            want_p, want_m, want_v = adamw64(p0, g0, m0, v0, step, lr, betas, eps, wd)
            # m, v: three roundings and the two rounded constants; p: those of m, v, the root, two divisions, two products and a
            # difference (at most 16 half steps of the update and 4 of p), and the rounding to p's type
            size, root_bc2, decay = constants(step, lr, betas, wd)
            term_m = betas[0] * np.abs(m0) + (1 - betas[0]) * np.abs(g0)
            assert (np.abs(_np(m) - want_m) <= 5 * EPS32 * term_m + 1e-44).all()
            assert (np.abs(_np(v) - want_v) <= 6 * EPS32 * want_v + 1e-44).all()
            upd = size * term_m / (np.sqrt(want_v) / root_bc2 + eps)
            assert_rounded(p, want_p, 16 * EPS32 * upd + 4 * EPS32 * np.abs(p0), step)
        if last:
            assert all(float(z.float().abs().sum()) == 0.0 for z in zero)


def random_state8(p, gen, device):
    n = p.numel()
    mc = torch.randint(-127, 128, p.shape, generator=gen, dtype=torch.int8)
    rc = torch.randint(0, 256, p.shape, generator=gen, dtype=torch.uint8)
    sc = torch.rand(-(-n // 256), 2, generator=gen) * 1e-5
    m, r = torch.empty_like(p, dtype=torch.int8), torch.empty_like(p, dtype=torch.uint8)
    return m.copy_(mc), r.copy_(rc), sc.to(device)


def check_adamw8(device, ptype, gtype, wd=0.01, eps=1e-8, betas=(0.9, 0.99), steps=(1, 7), lr=0.01, seed=11):
    """Codes and scales bit for bit, parameters in 64 bits, from zero and from random states."""
    for fresh in (True, False):
        ps, gs = _inputs(ptype, gtype, 6, device)
        gen = torch.Generator().manual_seed(7)
        if fresh:
            state = [(torch.zeros_like(p, dtype=torch.int8), torch.zeros_like(p, dtype=torch.uint8),
                      torch.zeros(-(-p.numel() // 256), 2, device=device)) for p in ps]
        else:
            state = [random_state8(p, gen, device) for p in ps]
        ords = [3 * k + 1 for k in range(len(ps))]
        for step in steps:
            before = [[_np(_as_param(g, p)).copy(), _np(p).copy()] + [_np(x).copy() for x in st[:2]] + [st[2].cpu().numpy().copy()]
                      for p, g, st in zip(ps, gs, state)]
            optim.adamw_step(ps, gs, [s[0] for s in state], [s[1] for s in state], [s[2] for s in state], step=step, lr=lr,
                             betas=betas, eps=eps, weight_decay=wd, seed=seed, ordinals=ords)
            for k, (p, st, (g0, p0, mc, rc, sc)) in enumerate(zip(ps, state, before)):
                want_mc, want_rc, want_sc, m, r = adamw8_ieee(g0.astype(np.float32), mc, rc, sc, seed, ords[k], step, betas)
                assert np.array_equal(_np(st[0]), want_mc) and np.array_equal(_np(st[1]), want_rc), (k, step)
                assert np.array_equal(st[2].cpu().numpy(), want_sc), (k, step)
                m0, r0 = values8(mc, rc, sc.astype(np.float32))
                want_p, _, want_v = adamw64(p0, g0, m0.astype(np.float64), r0.astype(np.float64) ** 2, step, lr, betas, eps, wd)
                size, root_bc2, decay = constants(step, lr, betas, wd)
                upd = size * (betas[0] * np.abs(m0) + (1 - betas[0]) * np.abs(g0)) / (np.sqrt(want_v) / root_bc2 + eps)
                # as with 32-bit moments, and two more half steps where a reciprocal stands for a division
                tol = 18 * EPS32 * upd + 4 * EPS32 * np.abs(p0)
                assert_rounded(p, want_p, tol, (k, step))
                got_m, got_v = optim.adamw_moments(*st)
                m1, r1 = values8(want_mc, want_rc, want_sc)
                assert np.array_equal(_np(got_m), m1.astype(np.float64)) and np.array_equal(_np(got_v), (r1 * r1).astype(np.float64))


# -------------------------------------------------------------------------------------------------------------- routing
def plan64(ids, experts):
    """order, position, offsets of int64 ids [N, K] (numpy)."""
    flat = ids.reshape(-1)
    live = (flat >= 0) & (flat < experts)
    slots = np.nonzero(live)[0]
    slots = slots[np.argsort(flat[slots], kind="stable")]
    order = np.full(flat.size, -1, np.int64)
    order[:slots.size] = slots
    position = np.full(flat.size, -1, np.int64)
    position[slots] = np.arange(slots.size)
    offsets = np.concatenate([[0], np.cumsum(np.bincount(flat[slots], minlength=experts))])
    return order, position.reshape(ids.shape), offsets


def make_ids(kind, n, k, experts, gen):
    """Batches that routing goes wrong on: one hot expert, the same expert twice for a token, none at all, ids out of range."""
    if kind == "hot":
        ids = torch.full((n, k), experts // 2, dtype=torch.int64)
    elif kind == "none":
        ids = torch.full((n, k), -1, dtype=torch.int64)
    elif kind == "last":
        ids = torch.full((n, k), experts - 1, dtype=torch.int64)
    else:
        ids = torch.randint(0, experts, (n, k), generator=gen)
        if kind == "masked":
            ids[torch.rand(n, k, generator=gen) < 0.4] = -1
            ids[n // 3:n // 2] = -1                       # whole tokens without an expert
        if kind == "outside" and n:
            ids[::3] = experts
            ids[1::5, 0] = -(1 << 40)
            ids[2::7, -1] = (1 << 33) + 1                 # 32 bits of it would be a valid id
    return ids


def check_expert_sort(device, n, k, experts, kind, wide):
    from mneslam_amd.routing import expert_sort
    gen = torch.Generator().manual_seed(n + 7 * k + experts)
    ids = make_ids(kind, n, k, experts, gen)
    if not wide:
        ids = ids.clamp(-(1 << 31), (1 << 31) - 1).to(torch.int32)
    plan = expert_sort(ids.to(device), experts)
    order, position, offsets = plan64(ids.to(torch.int64).numpy(), experts)
    assert np.array_equal(plan.offsets.cpu().numpy(), offsets)
    assert np.array_equal(plan.order.cpu().numpy(), order)
    assert np.array_equal(plan.position.cpu().numpy(), position)
    assert plan.sizes() == np.diff(offsets).tolist() and int(plan.live) == offsets[-1]


def _rows_of(shape, dtype, gen, device, odd):
    """Rows with a stride and an odd start, or dense ones."""
    n, d = shape
    t = torch.randn(n, d + (3 if odd else 0), generator=gen).to(dtype).to(device)
    return t[:, 1:1 + d] if odd else t


def check_expert_rows(device, dtype, n, k, experts, width, out_width, kind, odd, wtype="f32", need=("x", "y", "w")):
    """dispatch, combine and their gradients against float64; masked slots carry NaN weights and dead rows NaN."""
    from mneslam_amd.routing import expert_combine, expert_dispatch, expert_sort
    dt, wt = NAMES[dtype], NAMES[wtype]
    gen = torch.Generator().manual_seed(n + 31 * k + width)
    ids = make_ids(kind, n, k, experts, gen)
    order, position, offsets = plan64(ids.numpy(), experts)
    live = int(offsets[-1])
    plan = expert_sort(ids.to(device), experts)
    x, y = _rows_of((n, width), dt, gen, device, odd), _rows_of((n * k, out_width), dt, gen, device, odd)
    w = torch.randn(n, k, generator=gen).to(wt)
    w[torch.from_numpy(position) < 0] = float("nan")
    w = w.to(device)
    with torch.no_grad():
        y[live:] = float("nan")
    x, y, w = (t.requires_grad_(name in need) for name, t in (("x", x), ("y", y), ("w", w)))
    xs, out = expert_dispatch(x, plan), expert_combine(y, plan, w)
    gxs, gout = _rows_of((n * k, width), dt, gen, device, odd), _rows_of((n, out_width), dt, gen, device, odd)
    gxs[live:] = float("nan")
    outs = [t for t in (xs, out) if t.requires_grad]
    ins = [t for t in (x, y, w) if t.requires_grad]
    got = dict(zip(need, torch.autograd.grad(outs, ins, [g for t, g in ((xs, gxs), (out, gout)) if t.requires_grad]))) if ins else {}

    f = lambda t: t.detach().cpu().double().numpy()                                   # noqa: E731
    half = lambda t, want: (torch.finfo(t).eps / 2 * np.abs(want) + torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2) * (t != torch.float32)  # noqa: E731
    slot = order[:live]
    tok, w64 = slot // k, f(w).reshape(-1)
    X, Y, GX, GO = f(x), f(y)[:live], f(gxs)[:live], f(gout)

    def near(t, want, scale, terms, what):
        # `terms` roundings of fp32 on sums of magnitudes up to `scale`, and the rounding to the result's type
        tol = terms * EPS32 * scale * 1.01 + half(t.dtype, want) * 1.01 + 1e-44
        assert t.shape == want.shape and (np.abs(f(t) - want) <= tol).all(), what

    def summed(rows, width):
        total = np.zeros((n, width))
        np.add.at(total, tok, rows)
        return total

    def full(rows):
        return np.concatenate([rows, np.zeros((n * k - live, rows.shape[1]))])

    assert xs.dtype == dt and np.array_equal(f(xs), full(X[tok]))
    near(out, summed(w64[slot][:, None] * Y, out_width), summed(np.abs(w64[slot][:, None] * Y), out_width), k, "out")
    if "x" in need:
        near(got["x"], summed(GX, width), summed(np.abs(GX), width), k, "dx")
    if "y" in need:
        want = full(w64[slot][:, None] * GO[tok])
        near(got["y"], want, np.abs(want), 1, "dy")
    if "w" in need:
        want, scale = np.zeros(n * k), np.zeros(n * k)
        want[slot], scale[slot] = (GO[tok] * Y).sum(1), np.abs(GO[tok] * Y).sum(1)
        near(got["w"], want.reshape(n, k), scale.reshape(n, k), out_width, "dw")
        assert got["w"].dtype == wt
