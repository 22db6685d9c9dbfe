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


def dither(seed, ordinal, step, n, start=0):
    """u_m, u_r of the elements start .. start + n - 1 of a tensor (float32, multiples of 2^-16)."""
    i = np.arange(start, start + n, dtype=np.uint64)
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


def adamw8_ieee(g, mc, rc, scales, seed, ordinal, step, betas, start=0):
    """New codes and scales, bit for bit (g float32), of a tensor's blocks from element `start` on."""
    f = np.float32
    b1, o1, b2, o2 = f(betas[0]), f(1.0 - betas[0]), f(betas[1]), f(1.0 - betas[1])
    with np.errstate(all="ignore"):
        m, r = values8(mc, rc, scales)
        m = m * b1 + g * o1
        r = np.sqrt((r * r) * b2 + (g * g) * o2)
        um, ur = dither(seed, ordinal, step, g.size, start)
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


# ----------------------------------------------------------------------------------------------------------- run together
def check_agent_maps(device, tmp_path):
    """Two agents' maps with overlapping boxes, one of them read from its checkpoint: the union's answers against each map queried by
    itself and blended in float64."""
    import parity_cases as pc
    from helpers import load_golden
    from mneslam_amd import configs, slam_glue
    from mneslam_amd.model.agent_maps import AgentMaps
    g = load_golden("fwd_colorplanes")
    cfg = configs.small_test_config(one_grid=False, depth_trunc=3.0)
    cfg["data"]["output"], cfg["data"]["exp_name"] = str(tmp_path), "union"
    own, other = (pc.model_from_golden(g, cfg, device).eval() for _ in range(2))
    box = own.bounding_box.clone()
    with torch.no_grad():
        for p in other.decoder.parameters():
            p.mul_(-0.5)
    own.bounding_box = box.clone()
    own.bounding_box[0, 1] = box[0].mean() + 0.2
    other.bounding_box = box.clone()
    other.bounding_box[0, 0] = box[0].mean() - 0.2
    slam_glue.save_latest_checkpoint(other, cfg, 1)
    union = slam_glue.load_agent_maps(own, cfg, [1], lambda: pc.model_from_golden(g, cfg, device).eval(), torch.device(device))
    gen = torch.Generator().manual_seed(3)
    lo, hi = box[:, 0].float().cpu(), box[:, 1].float().cpu()
    pts = lo + (hi - lo) * (torch.rand(211, 3, generator=gen) * 1.2 - 0.1)        # some in no box
    pts[0], pts[1] = own.bounding_box[:, 1].float().cpu(), float("nan")
    pts = pts.to(device)
    ids, w = union.route(pts)
    raw = union.query_color_sdf(pts)
    with torch.no_grad():
        alone = torch.stack([m.query_color_sdf(torch.nan_to_num(pts)).double() for m in union.models], 1)
    held = ids >= 0
    want = torch.where(held[..., None], alone.gather(1, ids.clamp(min=0).long()[..., None].expand(-1, -1, 4)) * w.double()[..., None], 0.0).sum(1)
    assert torch.equal(union.covered(pts), held[:, 0]) and 0 < int(held[:, 1].sum()) < int(held[:, 0].sum()) < len(pts)
    assert (w.sum(1)[held[:, 0]] - 1).abs().max() < 1e-6 and (raw[~held[:, 0]] == 0).all()
    # the same kernels on the same points (a row's answer does not depend on its neighbours), two fp32 products and their sum
    assert ((raw.double() - want).abs() <= 4 * EPS32 * (alone.abs().amax(1) + 1e-30)).all()
    assert torch.equal(union.query_sdf(pts), raw[:, 3]) and union.query_color(pts).shape == (211, 3)
    assert AgentMaps([own]).top == 1


def check_mixture_step(device, bits, ptype="f32"):
    """A mixture of small experts on grid features, trained for some steps: routing and its gradients, the experts on their runs, one
    AdamW call for all their tensors -- against the same model in float64 (gradients of the first step), with 32-bit moments the
    parameters after each step too."""
    from mneslam_amd.optim import FusedAdamW
    from mneslam_amd.routing import expert_combine, expert_dispatch, expert_sort
    dt = NAMES[ptype]
    gen = torch.Generator().manual_seed(12)
    n, k, e, d, h = 150, 2, 5, 19, 16
    x = torch.randn(n, d, generator=gen).to(dt).to(device).requires_grad_(True)
    target = torch.randn(n, 4, generator=gen).to(device)
    ids = make_ids("masked", n, k, e, gen)
    ids[ids == 3] = 1                                              # an expert without a row
    logits = torch.nn.Parameter((torch.randn(n, k, generator=gen)).to(device))
    experts = [[torch.nn.Parameter((torch.randn(h, d, generator=gen) / d ** 0.5).to(dt).to(device)),
                torch.nn.Parameter((torch.randn(4, h, generator=gen) / h ** 0.5).to(dt).to(device))] for _ in range(e)]
    flat = [p for pair in experts for p in pair]
    opt = FusedAdamW([{"params": [logits], "state_bits": 32}, {"params": flat}], lr=0.01, betas=(0.9, 0.99), weight_decay=0.02, state_bits=bits, seed=4)
    order, position, _ = plan64(ids.numpy(), e)

    def exact_loss(xv, lv, ws):
        out = 0.0
        w = torch.softmax(lv, 1)
        rows = []
        for t in range(n):
            acc = torch.zeros(4, dtype=torch.float64)
            for j in range(k):
                i = int(ids[t, j])
                if i >= 0:
                    acc = acc + w[t, j] * (ws[2 * i + 1] @ torch.tanh(ws[2 * i] @ xv[t]))
            rows.append(acc)
        return torch.square(torch.stack(rows) - target.double().cpu()).mean()

    plan = expert_sort(ids.to(device), e)
    sizes = plan.sizes()
    for step in range(1, 4):
        rows = expert_dispatch(x, plan)
        ys, at = [], 0
        for (a, b), size in zip(experts, sizes):
            ys.append(torch.tanh(rows[at:at + size].float() @ a.float().t()) @ b.float().t())
            at += size
        ys.append(torch.zeros(n * k - at, 4, device=device))
        out = expert_combine(torch.cat(ys), plan, torch.softmax(logits, 1))
        loss = torch.square(out - target).mean()
        opt.zero_grad()
        x.grad = None
        loss.backward()
        if step == 1:
            dbl = [t.detach().double().cpu().requires_grad_(True) for t in [x, logits] + flat]
            want = torch.autograd.grad(exact_loss(dbl[0], dbl[1], dbl[2:]), dbl, allow_unused=True)
            for t, g in zip([x, logits] + flat, want):
                if g is None or not g.abs().max():
                    assert t.grad is None or not t.grad.abs().max()      # the expert without a row
                    continue
                # sums of up to n k d fp32 products; a 16-bit gradient is rounded on its way (rows, and their sum over k)
                tol = (2e-5 if t.dtype == torch.float32 and dt == torch.float32 else 4 * torch.finfo(dt).eps) * float(g.abs().max())
                assert (t.grad.double().cpu() - g).abs().max() <= tol, t.shape
        before = [(_np(p).copy(), _np(p.grad).copy(), [_np(v).copy() for v in opt.moments(p)]) if p.grad is not None and p in opt.state else None for p in flat]
        opt.step()
        for p, b in zip(flat, before):
            if b is None or bits != 32:
                continue
            want_p, _, want_v = adamw64(b[0], b[1], b[2][0], b[2][1], step, 0.01, (0.9, 0.99), 1e-8, 0.02)
            size, root_bc2, _ = constants(step, 0.01, (0.9, 0.99), 0.02)
            upd = size * (0.9 * np.abs(b[2][0]) + 0.1 * np.abs(b[1])) / (np.sqrt(want_v) / root_bc2 + 1e-8)
            assert_rounded(p, want_p, 16 * EPS32 * upd + 4 * EPS32 * np.abs(b[0]), step)
    assert all(torch.isfinite(p).all() for p in flat) and opt.state[flat[0]]["step"] == 3


# ------------------------------------------------------------------------------------------------- AdamW: the rest of its contract
def _state_for(p, bits, device):
    if bits == 32:
        return [torch.zeros_like(p, dtype=torch.float32) for _ in range(2)], None
    return [torch.zeros_like(p, dtype=torch.int8), torch.zeros_like(p, dtype=torch.uint8)], torch.zeros(-(-p.numel() // 256), 2, device=device)


def _step(ps, gs, bits, device, step=1, state=None, **kw):
    state = state or [_state_for(p, bits, device) for p in ps]
    args = dict(step=step, lr=0.01, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.0)
    args.update(kw)
    optim.adamw_step(ps, gs, [s[0][0] for s in state], [s[0][1] for s in state], [s[1] for s in state] if bits == 8 else None, **args)
    return state


def check_adamw_refusals(device):
    p, g = torch.ones(300, device=device), torch.ones(300, device=device)
    before = p.clone()
    m, v = torch.zeros_like(p), torch.zeros_like(p)
    c, d, s = torch.zeros(300, dtype=torch.int8, device=device), torch.zeros(300, dtype=torch.uint8, device=device), torch.zeros(2, 2, device=device)
    ok = dict(step=1, lr=0.1)

    def bad(error, *lists, scales=None, **kw):
        with pytest.raises(error):
            optim.adamw_step(*[[x] if torch.is_tensor(x) else x for x in lists], scales, **{**ok, **kw})

    bad(ValueError, [p, p], g, m, v)
    bad(ValueError, [p, p], [g, g], [m, m.clone()], [v, v.clone()])
    bad(ValueError, [p[:200], p[100:]], [g[:200], g[100:]], [m[:200], m[100:]], [v[:200], v[100:]])          # overlapping
    for kw in (dict(step=0), dict(step=-3), dict(step=1 << 31), dict(lr=-1.0), dict(lr=float("nan")), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)),
               dict(eps=-1e-8), dict(weight_decay=-1.0), dict(seed=-1), dict(seed=1 << 32), dict(ordinals=[-1]), dict(ordinals=[1 << 32]), dict(ordinals=[])):
        bad(ValueError, p, g, m, v, **kw)
    bad(TypeError, p.double(), g, m, v)
    bad(TypeError, p, g.double(), m, v)
    bad(TypeError, p.bfloat16(), g.half(), m, v)
    bad(TypeError, p, g, m.bfloat16(), v)
    bad(TypeError, p, g, m, v, scales=[s])                                   # 32-bit moments with scales
    bad(TypeError, p, g, c, d)                                               # codes without
    bad(ValueError, p, g[:299], m, v)
    bad(ValueError, p, g, m.view(3, 100), v)
    bad(ValueError, p, g, c, d, scales=[s[:1]])
    bad(ValueError, p, g, c, d, scales=[s.t().contiguous().t()])
    bad(ValueError, p, g, c, d, scales=[s.double()])
    wide = torch.ones(300, 2, device=device)
    bad(ValueError, wide[:, 0], g, m, v)                                     # not dense
    bad(ValueError, p[:1].expand(300), g, m, v)
    bad(ValueError, torch.ones(20, 15, device=device), g.view(20, 15), m.view(15, 20).t(), v.view(20, 15))
    bad(ValueError, torch.ones(20, 15, device=device), g.view(15, 20).t(), m.view(20, 15), v.view(20, 15), zero_grad=True)
    bad(ValueError, p, g.to_sparse(), m, v)
    bad(TypeError, p, [None], m, v)
    for args in ((c.float(), d, s), (c, d.to(torch.int8), s), (c, d[:299], s), (c, d, s[:1]), (c[::2], d[::2], s[:1])):
        with pytest.raises((TypeError, ValueError)):
            optim.adamw_moments(*args)
    assert torch.equal(p, before) and not m.any() and not c.any()            # nothing was touched
    optim.adamw_step([], [], [], [], **ok)
    optim.adamw_step([p[:0]], [g[:0]], [m[:0]], [v[:0]], **ok)
    if device != "cpu":
        bad(ValueError, p.cpu(), g, m, v)
        bad(ValueError, p.cpu(), g.cpu(), m.cpu(), v.cpu())


def check_adamw_nonfinite(device, bits):
    """A gradient that is not finite: its own element with 32-bit moments, its block's moments with 8-bit ones, nothing else."""
    for value in (float("nan"), float("inf"), -float("inf"), 1e30):
        p, g = torch.ones(1000, device=device), torch.full((1000,), 0.01, device=device)
        g[300] = value
        state = _step([p], [g], bits, device)
        first = p.clone()
        g[300] = 0.01
        _step([p], [g], bits, device, step=2, state=state)
        assert torch.isfinite(first[:256]).all() and torch.isfinite(p[512:]).all() and torch.isfinite(p[:256]).all()
        if bits == 32:
            m, v = state[0][0]
            ok = torch.ones(1000, dtype=torch.bool, device=device)
            ok[300] = False
            assert torch.isfinite(p[ok]).all() and torch.isfinite(m[ok]).all()
            assert torch.isnan(p[300]) if value != 1e30 else p[300] == first[300] == 1.0       # 1e30 squared is infinite: no update
        else:
            m, v = optim.adamw_moments(*state[0][0], state[0][1])
            assert torch.isfinite(m[:256]).all() and torch.isfinite(v[512:]).all() and torch.isnan(v[256:512]).all()
            assert torch.isnan(m[256:512]).all() == (value != 1e30) and torch.isnan(p[256:512]).all()


def check_adamw8_poisoned(device):
    """A block whose scale of either moment is NaN (a state from elsewhere) stays so, its neighbours do not notice."""
    for which in (0, 1):
        p, g = torch.ones(768, device=device), torch.full((768,), 0.01, device=device)
        state = _step([p], [g], 8, device)
        state[0][1][1, which] = float("nan")
        for step in (2, 3):
            _step([p], [g], 8, device, step=step, state=state)
        values = optim.adamw_moments(*state[0][0], state[0][1])
        assert torch.isnan(values[which][256:512]).all() and torch.isfinite(values[which][:256]).all() and torch.isfinite(values[which][512:]).all()
        assert torch.isfinite(values[1 - which]).all() and torch.isfinite(p[:256]).all() and torch.isfinite(p[512:]).all()


def check_adamw_shared_state(device):
    """What a step writes may not be one tensor's and another's: moments, scales, gradients that it clears."""
    p = [torch.ones(300, device=device) for _ in range(2)]
    g = [torch.ones(300, device=device) for _ in range(2)]
    m, v = ([torch.zeros(300, device=device) for _ in range(2)] for _ in range(2))
    c = [torch.zeros(300, dtype=torch.int8, device=device) for _ in range(2)]
    d = [torch.zeros(300, dtype=torch.uint8, device=device) for _ in range(2)]
    s = [torch.zeros(2, 2, device=device) for _ in range(2)]
    for lists, scales, zero in (([p, g, [m[0], m[0]], v], None, False), ([p, g, m, [v[0], v[0]]], None, False), ([p, g, m, m[::-1]], None, False),
                                ([p, g, [c[0], c[0]], d], s, False), ([p, g, c, [d[0], d[0]]], s, False), ([p, g, c, d], [s[0], s[0]], False),
                                ([p, [g[0], g[0]], m, v], None, True), ([p, g, [p[1], m[1]], v], None, False)):
        with pytest.raises(ValueError, match="overlap"):
            optim.adamw_step(*lists, scales, step=1, lr=0.1, zero_grad=zero)
    assert all((x == 1.0).all() for x in p + g) and not any(x.any() for x in m + v + c + d + s)
    optim.adamw_step(p, [g[0], g[0]], m, v, step=1, lr=0.1)          # a gradient that is only read may be shared
    assert torch.equal(p[0], p[1]) and (p[0] < 1.0).all()


def check_adamw_loads_no_other_rule(device):
    """States of torch.optim.AdamW with another rule than this step's are refused, and nothing is loaded."""
    for kw in (dict(amsgrad=True), dict(maximize=True)):
        p = torch.nn.Parameter(torch.ones(4, device=device))
        ref = torch.optim.AdamW([p], lr=0.5, **kw)
        p.grad = torch.ones_like(p)
        ref.step()
        opt = optim.FusedAdamW([p], lr=0.25)
        with pytest.raises(ValueError, match=next(iter(kw))):
            opt.load_state_dict(ref.state_dict())
        assert opt.param_groups[0]["lr"] == 0.25 and not opt.state


def check_adamw8_small_and_zero(device):
    """Zero blocks stay zero, tiny values neither overflow a scale nor lose the second moment."""
    p, g = torch.ones(1024, device=device), torch.zeros(1024, device=device)
    g[256:512] = 1e-20                                     # the square of its tenth is below fp32's range
    g[512:768] = 1e-34                                     # and this one's moment below what a scale can hold
    g[768] = 1.0
    g[769] = 1e-9                                          # far below its block's largest
    state = _step([p], [g], 8, device)
    (mc, rc), sc = state[0]
    m, v = optim.adamw_moments(mc, rc, sc)
    assert not m[:256].any() and not v[:256].any() and (p[:256] == 1).all() and torch.isfinite(p).all()
    assert (sc[2] == 0).all() and not mc[512:768].any() and float(v[769]) > 0
    want = adamw64(np.ones(256), g[768:].cpu().double().numpy(), np.zeros(256), np.zeros(256), 1, 0.01, (0.9, 0.99), 1e-8, 0.0)[0]
    assert np.abs(p[768:].cpu().double().numpy() - want).max() <= 40 * EPS32
    for step in range(2, 30):
        _step([p], [g], 8, device, step=step, state=state)
    assert torch.isfinite(p).all() and (p[:256] == 1).all()
    assert float((1 - p[769]).abs()) < 0.31                # thirty steps of at most lr each


def check_adamw8_dither(device):
    """Moments that change by less than a code a step still move, by the right amount on average; the codes are a function of seed,
    ordinal, step and element alone."""
    n = 256 * 64
    p, g = torch.zeros(n, device=device), torch.full((n,), 0.5, device=device)
    g[::256] = 1.0                                         # the block's largest, held up by its own gradient
    state = _step([p], [g], 8, device, betas=(0.0, 0.0))   # m = g, sqrt(v) = g
    rest = torch.arange(n, device=device) % 256 != 0
    hold = torch.where(rest, 0.0, 1.0)
    for step in range(2, 202):
        _step([p], [hold], 8, device, step=step, state=state, betas=(0.999, 0.999))
    m, v = optim.adamw_moments(*state[0][0], state[0][1])
    # unbiased: the mean of m over 16320 elements follows 0.5 * 0.999^200.  One step's rounding has at most half a code's standard
    # deviation, (2 c + 1) / (2 * 127^2) with c = 90: 200 steps, 16320 elements, five standard deviations
    want, sd = 0.5 * 0.999 ** 200, 181 / (2 * 16129) * 200 ** 0.5 / 16320 ** 0.5
    assert abs(float(m[rest].double().mean()) - want) < 5 * sd
    # sqrt(v) is what is unbiased: v's mean is above by the variance of sqrt(v), at most 200 codes' of (2 * 180 + 1) / (2 * 255^2) each
    want_r, sd_r = 0.5 * 0.999 ** 100, 361 / (2 * 65025) * 200 ** 0.5
    assert abs(float(v[rest].double().sqrt().mean()) - want_r) < 5 * sd_r / 16320 ** 0.5 + sd_r ** 2 / want_r
    again = {}
    for name, kw in (("same", {}), ("same2", {}), ("seed", dict(seed=1)), ("ordinal", dict(ordinals=[5])), ("step", dict(step=2))):
        st = _step([torch.zeros(n, device=device)], [torch.linspace(0, 1, n, device=device)], 8, device, **{"seed": 0, **kw})
        again[name] = (st[0][0][0], st[0][0][1])
    assert all(torch.equal(a, b) for a, b in zip(again["same"], again["same2"]))
    for name in ("seed", "ordinal", "step"):
        assert all(0.02 < (a != b).float().mean() for a, b in zip(again["same"], again[name])), name


def check_fused_adamw(device):
    """The optimizer against torch.optim.AdamW: groups, steps that skip a tensor, saved and loaded states."""
    gen = torch.Generator().manual_seed(2)
    shapes = [(7, 9), (300,), (1, 4, 6, 5), (1,)]
    start = [torch.randn(s, generator=gen) for s in shapes]
    start[2] = start[2].contiguous(memory_format=torch.channels_last)
    make = lambda dev: [torch.nn.Parameter(t.clone().to(dev)) for t in start]        # noqa: E731
    ours, theirs = make(device), make("cpu")
    groups = lambda ps: [{"params": ps[:2], "lr": 0.02, "weight_decay": 0.1}, {"params": ps[2:], "eps": 1e-6, "betas": (0.5, 0.9)}]  # noqa: E731
    opt, ref = optim.FusedAdamW(groups(ours), lr=0.005), torch.optim.AdamW(groups([p for p in theirs]), lr=0.005)
    versions = [p._version for p in ours]
    for step in range(5):
        for k, (p, q) in enumerate(zip(ours, theirs)):
            grad = None if step in (1, 2) and k == 1 else torch.randn(q.shape, generator=gen)
            q.grad, p.grad = grad, None if grad is None else grad.to(device)
        assert opt.step(lambda: torch.tensor(3.0)) == 3.0
        ref.step()
        if step == 2:                                          # through a saved state, into new objects
            saved = opt.state_dict()
            ours2 = [torch.nn.Parameter(p.detach().clone()) for p in ours]
            opt = optim.FusedAdamW(groups(ours2), lr=0.005)
            opt.load_state_dict(saved)
            ours = ours2
            versions = [p._version for p in ours]
    assert all(p._version > v for p, v in zip(ours, versions))        # what autograd saved of a parameter is out of date
    for p, q in zip(ours, theirs):
        assert (p.detach().cpu() - q.detach()).abs().max() <= 5 * 30 * EPS32 * (q.abs().max() + 1)
    # torch.optim.AdamW's own state
    opt2 = optim.FusedAdamW(groups([torch.nn.Parameter(p.detach().clone()) for p in ours]), lr=0.005)
    opt2.load_state_dict(ref.state_dict())
    for p, q in zip((p for g in opt2.param_groups for p in g["params"]), theirs):
        assert opt2.state[p]["step"] == int(ref.state[q]["step"]) and opt2.state[p]["exp_avg"].dtype == torch.float32
        p.grad = torch.ones_like(p)
    opt2.step(zero_grad=True)
    assert all(not p.grad.any() for g in opt2.param_groups for p in g["params"])
    # 8-bit states of 16-bit parameters survive a round trip bit for bit
    ps = [torch.nn.Parameter(t.clone().bfloat16().to(device)) for t in start]
    opt = optim.FusedAdamW([{"params": ps[:1], "state_bits": 32}, {"params": ps[1:]}], state_bits=8, seed=9)
    for _ in range(2):
        for p in ps:
            p.grad = torch.randn(p.shape, generator=gen).bfloat16().to(device)
        opt.step()
    saved = opt.state_dict()
    other = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    opt_b = optim.FusedAdamW([{"params": other[:1]}, {"params": other[1:]}])
    opt_b.load_state_dict(saved)
    for p, q in zip(ps, other):
        q.grad = p.grad.clone()
        for key, value in opt.state[p].items():
            loaded = opt_b.state[q][key]
            assert loaded == value if key == "step" else (loaded.dtype == value.dtype and loaded.stride() == value.stride() and torch.equal(loaded, value)), key
    opt.step()
    opt_b.step()
    for p, q in zip(ps, other):
        assert torch.equal(p, q) and all(torch.equal(a, b) for a, b in zip(opt.moments(p), opt_b.moments(q)))
    # ... but not into a parameter whose memory has another order: its blocks would be others
    other = [torch.nn.Parameter(p.detach().clone().contiguous()) for p in ps]
    opt_b = optim.FusedAdamW([{"params": other[:1]}, {"params": other[1:]}])
    with pytest.raises(ValueError):
        opt_b.load_state_dict(saved)
    for kw in (dict(lr=-1), dict(betas=(0.9, 1.0)), dict(eps=-1), dict(weight_decay=-1), dict(state_bits=4), dict(seed=-1)):
        with pytest.raises(ValueError):
            optim.FusedAdamW(ps, **kw)
    opt = optim.FusedAdamW([torch.nn.Parameter(torch.ones(3, device=device))])
    with pytest.raises(ValueError):
        opt.add_param_group({"params": [torch.nn.Parameter(torch.ones(2, device=device))], "state_bits": 16})
    assert len(opt.param_groups) == 1
    p = opt.param_groups[0]["params"][0]
    assert not opt.moments(p)[0].any() and not opt.state
    opt.zero_grad()
    opt.step()                                                 # nothing has a gradient
    assert (p == 1).all()


def check_adamw_many(device, count, bits):
    """More tensors than a launch holds, of mixed types and sizes."""
    gen = torch.Generator().manual_seed(8)
    types = [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32)]
    ps, gs = [], []
    for k in range(count):
        n, (pt, gt) = int(torch.randint(0, 700, (1,), generator=gen)), types[k % 3 if k % 5 else 0]
        ps.append(torch.randn(n, generator=gen).to(pt).to(device))
        gs.append(torch.randn(n, generator=gen).to(gt).to(device))
    alone = [p.clone() for p in ps]
    state = _step(ps, gs, bits, device, step=3)
    for k, (p, g) in enumerate(zip(alone, gs)):
        st = _step([p], [g], bits, device, step=3, ordinals=[k])
        assert torch.equal(p, ps[k]) and all(torch.equal(a, b) for a, b in zip(st[0][0], state[k][0])), k


def check_adamw_flat(device, bits, ptype):
    """Tensors cut from flat buffers at odd places, moments and codes too: the same bits as for tensors of their own, and what lies
    between them is left as it was."""
    gen = torch.Generator().manual_seed(14)
    dt, sizes = NAMES[ptype], [5000, 2048, 3, 4099, 1]
    starts = [1 + sum(sizes[:k]) + 3 * k for k in range(len(sizes))]
    total = starts[-1] + sizes[-1] + 7
    flat = lambda t: torch.full((total,), 77, dtype=t, device=device)          # noqa: E731
    p, g, m, v = flat(dt), flat(dt), flat(torch.int8 if bits == 8 else torch.float32), flat(torch.uint8 if bits == 8 else torch.float32)
    cut = lambda t: [t[a:a + n] for a, n in zip(starts, sizes)]                # noqa: E731
    for q, h in zip(cut(p), cut(g)):
        q.copy_(torch.randn(len(q), generator=gen))
        h.copy_(torch.randn(len(h), generator=gen))
    for t in cut(m) + cut(v):
        t.zero_()
    own = [[t.clone() for t in cut(x)] for x in (p, g, m, v)]
    scales = [[torch.zeros(-(-n // 256), 2, device=device) for n in sizes] if bits == 8 else None for _ in range(2)]
    for step in (1, 2):
        for lists, s in (([cut(x) for x in (p, g, m, v)], scales[0]), (own, scales[1])):
            optim.adamw_step(*lists, s, step=step, lr=0.01, seed=3)
    for x, y in zip((p, m, v), (own[0], own[2], own[3])):
        assert all(torch.equal(a, b) for a, b in zip(cut(x), y))
        between = torch.ones(total, dtype=torch.bool, device=device)
        for a, n in zip(starts, sizes):
            between[a:a + n] = False
        assert (x[between] == 77).all()
    if bits == 8:
        for a, n, s in zip(starts, sizes, scales[0]):
            got, want = optim.adamw_moments(m[a:a + n], v[a:a + n], s), optim.adamw_moments(m[a:a + n].clone(), v[a:a + n].clone(), s)
            assert all(torch.equal(x, y) for x, y in zip(got, want))


def check_adamw_clock(device, bits):
    """Steps that read their number from device memory equal those that are given it."""
    import ctypes as C
    from mneslam_amd import _lib
    betas = (0.9, 0.99)
    offset = torch.zeros(1, dtype=torch.int32, device=device)
    table = torch.tensor([[1 - betas[0] ** t, 1 - betas[1] ** t] for t in range(1, 40)], dtype=torch.float64, device=device)
    clock = _lib.Clock()
    clock.step_offset, clock.bias_table, clock.n_table = offset.data_ptr(), table.data_ptr(), 39
    clock.beta1, clock.beta2 = betas
    gen = torch.Generator().manual_seed(4)
    g = torch.randn(777, generator=gen).to(device)
    p, q = torch.ones(777, device=device), torch.ones(777, device=device)
    sp, sq = None, None
    for k in range(4):
        sp = _step([p], [g], bits, device, step=5, state=sp, clock=clock)
        sq = _step([q], [g], bits, device, step=5 + k, state=sq)
        offset += 1
        assert torch.equal(p, q) and all(torch.equal(a, b) for a, b in zip(sp[0][0], sq[0][0])), k
    with pytest.raises(RuntimeError):
        _step([p], [g], bits, device, step=5, clock=clock, betas=(0.8, 0.99))
    return clock, offset, table


# ----------------------------------------------------------------------------------------------- routing: the rest of its contract
def check_routing_refusals(device):
    from mneslam_amd.routing import expert_combine, expert_dispatch, expert_sort
    ids = torch.zeros(6, 2, dtype=torch.int32, device=device)
    for bad, error in ((ids.float(), TypeError), (ids.to(torch.int16), TypeError), (ids.view(2, 3, 2), TypeError), (ids[:, :0], ValueError)):
        with pytest.raises(error):
            expert_sort(bad, 4)
    for experts in (0, -1, 4097):
        with pytest.raises(ValueError):
            expert_sort(ids, experts)
    plan = expert_sort(ids[:, 0], 4)
    assert plan.position.shape == (6, 1) and plan.n_tokens == 6 and plan.top_k == 1
    plan = expert_sort(ids, 4)
    x, y, w = torch.ones(6, 5, device=device), torch.ones(12, 5, device=device), torch.ones(6, 2, device=device)
    for f in (lambda: expert_dispatch(x[:5], plan), lambda: expert_dispatch(x[0], plan), lambda: expert_dispatch(x.view(6, 5, 1), plan),
              lambda: expert_combine(y[:11], plan), lambda: expert_combine(y, plan, w[:5]), lambda: expert_combine(y, plan, w.t()),
              lambda: expert_combine(y.view(12, 5, 1), plan), lambda: expert_combine(y, plan, w[:, :1]), lambda: expert_dispatch(x.to_sparse(), plan)):
        with pytest.raises(ValueError):
            f()
    for f in (lambda: expert_dispatch(x.double(), plan), lambda: expert_dispatch(x.int(), plan), lambda: expert_combine(y.double(), plan),
              lambda: expert_combine(y, plan, w.double()), lambda: expert_dispatch(None, plan)):
        with pytest.raises(TypeError):
            f()
    if device != "cpu":
        for f in (lambda: expert_sort(ids.cpu(), 4), lambda: expert_dispatch(x.cpu(), plan), lambda: expert_combine(y, plan, w.cpu())):
            with pytest.raises(ValueError):
                f()
    from mneslam_amd.routing import ExpertPlan
    wrong = ExpertPlan(plan.order.long(), plan.position.long(), plan.offsets)
    for f in (lambda: expert_dispatch(x, wrong), lambda: expert_combine(y, wrong)):
        with pytest.raises(TypeError):
            f()
    with pytest.raises(ValueError):
        expert_dispatch(x, ExpertPlan(plan.order, plan.position.t().contiguous().t(), plan.offsets))
    # a plan's entry that is no row is none (nothing is read or written outside)
    broken = ExpertPlan(plan.order, plan.position.clone(), plan.offsets)
    broken.position[2, 1], broken.position[3, 0] = 12, 2 ** 31 - 1
    got = expert_combine(y, broken, w)
    assert torch.equal(got[2:4], torch.ones(2, 5, device=device)) and expert_dispatch(x, broken).shape == (12, 5)
    # differentiable once
    a = x.clone().requires_grad_(True)
    out = expert_dispatch(a, plan)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(out.sum(), a, create_graph=True)
    b = y.clone().requires_grad_(True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(expert_combine(b, plan, w).sum(), b, create_graph=True)
    # what the backward pass reads must not have changed
    v = w.clone().requires_grad_(True)
    out = expert_combine(y, plan, v * 1)
    y.add_(1)
    with pytest.raises(RuntimeError):
        out.sum().backward()


def check_combine_keeps_what_it_needs(device):
    """Rows may be written again where their values are no part of a gradient."""
    from mneslam_amd.routing import expert_combine, expert_sort
    plan = expert_sort(torch.tensor([[1, 0], [1, -1]], device=device), 2)
    for w in (None, torch.tensor([[0.5, 2.0], [4.0, 1.0]], device=device)):
        a = torch.ones(4, 3, device=device, requires_grad=True)
        y = a * 1.0
        out = expert_combine(y, plan, w)
        y.zero_()
        out.sum().backward()
        want = torch.zeros(4, 3)
        for t, j in ((0, 0), (0, 1), (1, 0)):
            want[int(plan.position[t, j])] = 1.0 if w is None else float(w[t, j])
        assert torch.equal(a.grad.cpu(), want)
    w = torch.ones(2, 2, device=device, requires_grad=True)
    y = torch.ones(4, 3, device=device)
    out = expert_combine(y, plan, w)
    y.zero_()
    with pytest.raises(RuntimeError, match="inplace"):
        out.sum().backward()


def check_routing_views(device):
    """Gradients that are broadcast, tokens that are, no weights, a plan used again, rows of another layout."""
    from mneslam_amd.routing import expert_combine, expert_dispatch, expert_sort
    ids = torch.tensor([[2, 2], [0, -1], [1, 2], [-1, -1]], device=device)
    plan = expert_sort(ids.t().contiguous().t(), 3)
    one = torch.arange(1.0, 4.0, device=device, requires_grad=True)
    x = one.expand(4, 3)
    rows = expert_dispatch(x, plan)
    live = int(plan.live)
    assert live == 5 and torch.equal(rows[:live], one.detach().expand(5, 3)) and not rows[live:].any()
    rows.sum().backward()                                   # the gradient of a sum is one number broadcast over all rows
    assert torch.equal(one.grad, torch.full((3,), 5.0, device=device))
    y = torch.arange(8.0 * 3, device=device).view(3, 8).t().requires_grad_(True)          # columns next to each other
    out = expert_combine(y, plan)
    out.sum().backward()
    want = torch.zeros(4, 3, device=device)
    for t in range(4):
        for j in range(2):
            if ids[t, j] >= 0:
                want[t] += y.detach()[int(plan.position[t, j])]
    assert torch.equal(out, want)
    assert torch.equal(y.grad, (torch.arange(8, device=device) < live).float()[:, None].expand(8, 3))
    # a value of its own for each token and choice, against differences (the outputs are linear in each: any step is exact up to rounding)
    w = torch.rand(4, 2, device=device, requires_grad=True)
    yd = torch.rand(8, 3, device=device)
    probe = torch.rand(4, 3, device=device)
    (expert_combine(yd, plan, w) * probe).sum().backward()
    for t in range(4):
        for j in range(2):
            up = w.detach().clone()
            up[t, j] += 1.0
            diff = ((expert_combine(yd, plan, up) - expert_combine(yd, plan, w.detach())).double() * probe.double()).sum()
            assert abs(float(diff) - float(w.grad[t, j])) <= 64 * EPS32
    for experts in (2000, 2001, 4096):
        assert expert_sort(torch.zeros(0, 2, dtype=torch.int64, device=device), experts).offsets.tolist() == [0] * (experts + 1)
    empty = expert_sort(torch.zeros(0, 2, dtype=torch.int64, device=device), 3)
    assert empty.offsets.tolist() == [0, 0, 0, 0] and expert_dispatch(torch.zeros(0, 5, device=device), empty).shape == (0, 5)
    assert expert_combine(torch.zeros(0, 5, device=device), empty).shape == (0, 5)


# ------------------------------------------------------------------------------------------- tensors whose memory is not their values
def _lazily_negated(t):
    """``t`` as a view whose memory holds -t; t of one column (or one element) also as torch's public calls make it."""
    if t.is_floating_point() and t.dtype == torch.float32 and t.stride(-1) == 1 and t.shape[-1] == 1:
        view = torch.complex(torch.zeros_like(t), -t).conj().imag
    else:
        view = torch._neg_view(-t)
    assert view.is_neg() and torch.equal(view, t)
    return view


def check_negated_rows(device, dtype, width):
    """A lazily negated input of routing counts as its values: ids, tokens, rows, weights and the gradients that come in."""
    from mneslam_amd.routing import ExpertPlan, expert_combine, expert_dispatch, expert_sort
    gen = torch.Generator().manual_seed(41)
    n, k, e = 9, 2, 3
    dt = NAMES[dtype]
    ids = torch.randint(0, e, (n, k), generator=gen).to(device)
    x, y, w, gx, gy = (torch.randn(s, generator=gen).to(t).to(device) for s, t in
                       (((n, width), dt), ((n * k, width), dt), ((n, k), torch.float32), ((n * k, width), dt), ((n, width), dt)))
    plan = expert_sort(ids, e)
    again = expert_sort(_lazily_negated(ids), e)
    assert torch.equal(plan.position, again.position) and torch.equal(plan.order, again.order)
    results = []
    for seen in (lambda t: t, _lazily_negated):
        a, b, c = (seen(t).detach().requires_grad_(True) for t in (x, y, w))
        xs, out = expert_dispatch(a, plan), expert_combine(b, plan, c)
        results.append([xs, out, *torch.autograd.grad((xs, out), (a, b, c), (seen(gx), seen(gy)))])
    for plain, negated in zip(*results):
        assert torch.equal(plain, negated)
    wrong = ExpertPlan(plan.order, torch._neg_view(plan.position), plan.offsets)
    for f in (lambda: expert_dispatch(x, wrong), lambda: expert_combine(y, wrong)):
        with pytest.raises(ValueError, match="negated"):
            f()


def check_negated_adamw(device, bits):
    """A lazily negated gradient counts as its values; what is written in place must not be such a view."""
    for n in (1, 300):
        gen = torch.Generator().manual_seed(42)
        g = torch.randn(n, generator=gen).to(device)
        ps = [torch.ones(n, device=device) for _ in range(2)]
        states = [_step([p], [h], bits, device)[0] for p, h in zip(ps, (g, _lazily_negated(g)))]
        assert torch.equal(*ps) and (n == 1 or not torch.equal(ps[0], torch.ones_like(ps[0])))
        for a, b in zip(*(s[0] for s in states)):
            assert torch.equal(a, b)
        p, (lists, scales) = ps[0], states[0]
        before = p.clone()
        written = [[p], [lists[0]], [lists[1]]] + ([[scales]] if bits == 8 else [])
        for k in range(len(written)):
            args = [[torch._neg_view(t[0])] if i == k else t for i, t in enumerate(written)]
            with pytest.raises(ValueError, match="negated"):
                optim.adamw_step(args[0], [g], args[1], args[2], args[3] if bits == 8 else None, step=2, lr=0.1)
        with pytest.raises(ValueError, match="negated"):
            optim.adamw_step([p], [_lazily_negated(g)], [lists[0]], [lists[1]], [scales] if bits == 8 else None, step=2, lr=0.1, zero_grad=True)
        assert torch.equal(p, before)
        if bits == 8:
            want = optim.adamw_moments(*lists, scales)
            got = optim.adamw_moments(_lazily_negated(lists[0]), lists[1], _lazily_negated(scales))
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def check_not_traced(device):
    """A tracer cannot see what these calls compute: they are refused under one, and do nothing; modes that only watch are let through."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils.flop_counter import FlopCounterMode
    from mneslam_amd.routing import expert_combine, expert_dispatch, expert_sort
    ids = torch.tensor([[0, 1], [1, -1], [2, 0]], device=device)
    plan = expert_sort(ids, 3)
    x, y = torch.arange(15.0, device=device).view(3, 5), torch.arange(30.0, device=device).view(6, 5)
    p, m, v = torch.ones(5, device=device), torch.zeros(5, device=device), torch.zeros(5, device=device)
    c, d, s = torch.ones(5, device=device, dtype=torch.int8), torch.ones(5, device=device, dtype=torch.uint8), torch.ones(1, 2, device=device)
    calls = [(lambda t: expert_dispatch(t * 2, plan), x), (lambda t: expert_combine(t * 2, plan), y), (lambda t: expert_sort(t + 0, 3).position, ids),
             (lambda t: optim.adamw_step([p], [t * 2], [m], [v], step=1, lr=0.1) or p * 1, torch.ones(5, device=device)),
             (lambda t: optim.adamw_moments(c, d, t * 1)[0], s)]
    leaf = x.clone().requires_grad_(True)
    out = expert_dispatch(leaf, plan)
    calls.append((lambda t: torch.autograd.grad(out, leaf, t * 1, retain_graph=True)[0], torch.ones(6, 5, device=device)))
    for k, (f, arg) in enumerate(calls):
        with pytest.raises(RuntimeError, match="traced|Cannot insert a Tensor that requires grad"):      # (the latter: torch's own)
            torch.jit.trace(f, arg, check_trace=False)
        for mode, pre in (("real", False), ("real", True), ("fake", False), ("symbolic", False)):
            with pytest.raises((RuntimeError, TypeError), match="traced|classes"):
                make_fx(f, tracing_mode=mode, pre_dispatch=pre)(arg)
        with pytest.raises((RuntimeError, TypeError), match="traced|classes"):
            with FakeTensorMode(allow_non_fake_inputs=True):
                f(arg)
    assert (p == 1).all() and not m.any() and not v.any()
    with FlopCounterMode(display=False):
        got = [f(arg) for f, arg in calls[:3]]
    assert all(torch.equal(a, f(arg)) for a, (f, arg) in zip(got, calls))
    assert torch.equal(calls[5][0](calls[5][1]), torch.tensor([2.0, 1.0, 2.0], device=device)[:, None].expand(3, 5))

    class Own(torch.Tensor):                                        # a class with operations of its own
        @classmethod
        def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
            return NotImplemented
    own = torch.Tensor._make_subclass(Own, x)
    for f in (lambda: expert_dispatch(own, plan), lambda: optim.adamw_step([p], [torch.Tensor._make_subclass(Own, m)], [m], [v], step=1, lr=0.1)):
        with pytest.raises(TypeError, match="classes"):
            f()


def check_zeros_without_memory(device):
    """Zeros that torch keeps without memory (as forward-mode differentiation makes them) are zeros; they cannot be written."""
    from mneslam_amd.routing import ExpertPlan, expert_combine, expert_dispatch, expert_sort
    zeros = lambda *shape, **kw: torch._efficientzerotensor(shape, device=device, **kw)         # noqa: E731
    plan = expert_sort(torch.tensor([[0], [1], [0]], device=device), 2)
    assert torch.equal(expert_dispatch(zeros(3, 4), plan), torch.zeros(3, 4, device=device))
    assert torch.equal(expert_combine(torch.ones(3, 2, device=device), plan, zeros(3, 1)), torch.zeros(3, 2, device=device))
    assert torch.equal(expert_combine(zeros(3, 2), plan), torch.zeros(3, 2, device=device))
    assert expert_sort(zeros(3, 1, dtype=torch.int64), 2).offsets.tolist() == [0, 3, 3]
    with pytest.raises(ValueError):
        expert_dispatch(torch.ones(3, 4, device=device), ExpertPlan(plan.order, zeros(3, 1, dtype=torch.int32), plan.offsets))
    p, m, v = torch.ones(3, device=device), torch.ones(3, device=device), torch.ones(3, device=device)
    for lists in (([zeros(3)], [p], [m], [v]), ([p], [m.clone()], [zeros(3)], [v]), ([p], [m.clone()], [m], [zeros(3)])):
        with pytest.raises(ValueError):
            optim.adamw_step(*lists, step=1, lr=0.1)
    q = [t.clone() for t in (p, m, v)]
    optim.adamw_step([p], [zeros(3)], [m], [v], step=1, lr=0.1)
    optim.adamw_step(q[:1], [torch.zeros(3, device=device)], q[1:2], q[2:], step=1, lr=0.1)
    assert all(torch.equal(a, b) for a, b in zip((p, m, v), q))


def check_rows_copied_once(device):
    """Rows whose elements do not lie next to each other are copied once, the others never."""
    from torch.utils._python_dispatch import TorchDispatchMode
    from mneslam_amd.routing import expert_combine, expert_dispatch, expert_sort

    class Copies(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.count = getattr(self, "count", 0) + (func in (torch.ops.aten.clone.default, torch.ops.aten.copy_.default))
            return func(*args, **(kwargs or {}))

    plan = expert_sort(torch.tensor([[0, 1], [1, 0]], device=device), 2)
    for f, n in ((lambda t: expert_dispatch(t, plan), 2), (lambda t: expert_combine(t, plan), 4)):
        t = torch.arange(3.0 * n, device=device).view(n, 3)
        for given, want in ((t, 0), (t.t().contiguous().t(), 1)):
            with Copies() as seen:
                got = f(given)
            assert torch.equal(got, f(t)) and seen.count == want


def check_infinite_rows(device, dtype):
    """A row with one infinite element: the gradient of its weight is infinite wherever the element is, the others are what they are."""
    from mneslam_amd.routing import expert_combine, expert_sort
    dt = NAMES[dtype]
    for width in (1, 3, 4, 5, 8, 9, 13, 21):
        for k in (1, 2, 3):
            plan = expert_sort(torch.zeros(width, k, dtype=torch.int32, device=device), 1)          # token t's element t is the infinite one
            y = torch.ones(width * k, width, device=device, dtype=dt)
            y[plan.position[:, 0].long(), torch.arange(width, device=device)] = float("inf")
            w = torch.ones(width, k, device=device, requires_grad=True)
            (dw,) = torch.autograd.grad(expert_combine(y, plan, w), w, torch.ones(width, width, device=device, dtype=dt))
            want = torch.full((width, k), float(width))
            want[:, 0] = float("inf")
            assert torch.equal(dw.cpu(), want), (width, k)
            # ... and of the incoming gradient's element
            g = torch.ones(width, width, device=device, dtype=dt)
            g.fill_diagonal_(float("inf"))
            (dw,) = torch.autograd.grad(expert_combine(torch.ones_like(y), plan, w), w, g)
            assert torch.isposinf(dw).all(), (width, k)


def check_adamw_tiny_eps(device, ptype, bits):
    """An eps below fp32's normal range: what has no gradient stays where it is, and the others step by lr."""
    for eps in (1e-37, 1e-38, 1e-40, 1e-44):
        p, g = torch.ones(600, device=device, dtype=NAMES[ptype]), torch.zeros(600, device=device, dtype=NAMES[ptype])
        g[300:] = 0.5
        _step([p], [g], bits, device, eps=eps, lr=0.25)
        assert (p[:300] == 1).all() and (p[300:] == 0.75).all(), eps


def check_adamw8_quotient(device):
    """The update of a float32 parameter is one rounded quotient also with 8-bit moments: with beta = 0, lr = 1 and g = 1 nothing else of
    the step rounds, and p = -1 / (1 + eps)."""
    for j in range(1, 60):
        eps = float(np.float32(j / 61))
        p, g = torch.zeros(300, device=device), torch.ones(300, device=device)
        _step([p], [g], 8, device, betas=(0.0, 0.0), lr=1.0, eps=eps)
        want = -np.float32(1) / (np.float32(1) + np.float32(eps))
        assert (p.cpu().numpy() == want).all(), (j, float(p[0]), float(want))


# ------------------------------------------------------------------------------------------ the fp32 sums beside half-precision planes
class _RenderLike(torch.autograd.Function):
    """What the render node does for a half-precision plane: the fp32 gradient beside, its rounding to autograd."""

    @staticmethod
    def forward(ctx, p, g32):
        ctx.p, ctx.g32 = p, g32
        return p.float().sum()

    @staticmethod
    def backward(ctx, g):
        from mneslam_amd import plane_sums
        plane_sums.add(ctx.p, ctx.g32 * g)
        return (ctx.g32 * g).half(), None


def check_plane_gradients(device):
    """FusedAdamW takes a half-precision plane's gradient in fp32 while ``.grad`` is its rounding, and ``.grad`` itself wherever that is
    another: clipped, added to by another node, dropped and filled again, asked for without being accumulated."""
    tiny = torch.tensor([1e-9, -3e-9, 0.3, 2.0 ** -12 * 1.0003], device=device)        # two of them round to zero in fp16
    render = lambda p, s=1.0: _RenderLike.apply(p, tiny * s)                           # noqa: E731

    def moved(grads, **kw):
        """Where a zero parameter goes with beta = 0 after the gradients that ``grads(p)`` leaves: the moment is the gradient."""
        p = torch.nn.Parameter(torch.zeros(4, device=device, dtype=torch.float16))
        opt = optim.FusedAdamW([p], betas=(0.0, 0.0), weight_decay=0.0)
        grads(p, opt)
        opt.step(**kw)
        return opt.moments(p)[0], p, opt

    g, p, opt = moved(lambda p, _: render(p).backward())
    assert torch.equal(g, tiny)                                                        # not rounded
    opt.step()
    assert torch.equal(opt.moments(p)[0], tiny)

    def clipped(p, _):
        render(p).backward()
        torch.nn.utils.clip_grad_norm_([p], 1e-3)
    g, p, _ = moved(clipped)
    assert torch.equal(g, p.grad.float()) and float(g.norm()) < 1.01e-3
    assert torch.equal(moved(lambda p, _: (render(p).backward(), p.grad.neg_()))[0], -tiny.half().float())
    assert torch.equal(moved(lambda p, _: (render(p).backward(), setattr(p, "grad", p.grad * 4)))[0], 4 * tiny.half().float())

    more = torch.tensor([0.0, 1.0, 1.0, 0.0], device=device)                           # another source, in the same pass and in its own
    want = torch.where(more == 0, tiny, (tiny.half() + more.half()).float())
    assert torch.equal(moved(lambda p, _: (render(p) + (p * more.half()).sum()).backward())[0], want)
    assert torch.equal(moved(lambda p, _: (render(p).backward(), (p * more.half()).sum().backward()))[0], want)
    assert torch.equal(moved(lambda p, _: ((p * more.half()).sum().backward(), render(p).backward()))[0], want)

    def refilled(p, _):
        render(p).backward()
        p.grad = None
        (p * torch.zeros_like(p)).sum().backward()
    assert not moved(refilled)[0].any()                                                # the old sum is nobody's

    def dropped(p, _):
        render(p, 7.0).backward()
        p.grad = None
        render(p).backward()
    assert torch.equal(moved(dropped)[0], tiny)                                        # nor is it added to

    def asked(p, _):
        torch.autograd.grad(render(p, 5.0), p)
        render(p).backward()
    assert torch.equal(moved(asked)[0], tiny)

    def asked_after(p, _):
        render(p).backward()
        torch.autograd.grad(render(p, 5.0), p)
    assert torch.equal(moved(asked_after)[0], tiny.half().float())

    # added up over two passes and in one, cleared by the step, by the optimizer and by somebody else
    twice = torch.where((tiny.half() * 2) == (tiny * 2).half(), tiny * 2, (tiny.half() * 2).float())
    assert torch.equal(moved(lambda p, _: (render(p).backward(), render(p).backward()))[0], twice)
    assert torch.equal(moved(lambda p, _: (render(p) + render(p)).backward())[0], twice)
    for clear in (lambda p, opt: opt.step(zero_grad=True), lambda p, opt: opt.zero_grad(), lambda p, opt: opt.zero_grad(set_to_none=False),
                  lambda p, opt: setattr(p, "grad", None)):
        def cleared(p, opt):
            render(p, 3.0).backward()
            clear(p, opt)
            assert p.grad is None or not p.grad.any()
            render(p).backward()
        assert torch.equal(moved(cleared)[0], tiny)

    def cleared_beside(p, _):
        render(p, 3.0).backward()
        p.grad.zero_()
        render(p).backward()
    assert torch.equal(moved(cleared_beside)[0], tiny.half().float())


def check_plane_gradients_rendered(device):
    """The same with the render node itself: FusedAdamW's first moments of the planes are the fp32 sums, or what clipping left of ``.grad``."""
    import parity_cases as pc
    from helpers import load_golden
    from mneslam_amd import configs, slam_glue
    g = load_golden("fwd_onegrid")
    for clip in (False, True):
        cfg = configs.small_test_config(**pc.FWD_CASES["fwd_onegrid"])
        m = pc.model_from_golden(g, cfg, device).train()
        for lst in m.all_planes:
            for k in range(len(lst)):
                lst[k] = lst[k].half()
        opt = slam_glue.create_optimizer(m, cfg, optimizer_cls=optim.FusedAdamW)
        rays_o, rays_d, rgb, d, U = pc.to_dev(pc.fixture_inputs(g), device)
        losses = m._render(rays_o, rays_d, rgb, d, u=U)[-1]
        slam_glue.get_loss_from_ret(cfg, {k: losses[i] for i, k in enumerate(pc.LOSS_KEYS)}, is_co_sdf=False).backward()
        planes = [p for lst in m.all_planes for p in lst]
        sums = [p.grad32.clone() for p in planes]
        assert all(torch.equal(s.half(), p.grad) for s, p in zip(sums, planes)) and any(s.any() for s in sums)
        if clip:
            torch.nn.utils.clip_grad_value_(planes, 1e-6)
        opt.step()
        for s, p in zip(sums, planes):
            want = _as_param(p.grad.float() if clip else s, p)
            m1 = opt.moments(p)[0]
            assert (m1 - 0.1 * want).abs().max() <= 2 * EPS32 * 0.1 * want.abs().max()


class _FlatMap:
    """A map that answers one value everywhere."""

    def __init__(self, box, value):
        self.bounding_box, self.value = torch.tensor(box, dtype=torch.float64), value

    def query_color_sdf(self, points):
        return torch.full((len(points), 4), self.value, device=points.device)


def check_agent_maps_have_no_seam(device):
    """Three boxes and more over one place: the answer is continuous where one map takes another's place among the deepest."""
    from mneslam_amd.model.agent_maps import AgentMaps
    wide = [[-4.0, 4.0], [-4.0, 4.0]]
    three = [_FlatMap([[-5.0, 5.0], *wide], 0.0), _FlatMap([[-3.0, 2.0], *wide], 1.0), _FlatMap([[-2.0, 3.0], *wide], -1.0)]
    four = three + [_FlatMap([[-4.0, 2.5], [-4.5, 5.0], [-3.0, 3.0]], 3.0)]
    for maps, tops in ((three, (2, 3)), (four, (2, 3, 4))):
        for top in tops:
            union = AgentMaps(maps, top=top)
            # along lines through the place, away from where top + 1 maps are equally deep at once
            x = torch.linspace(-4.5, 4.5, 9001, dtype=torch.float64, device=device)
            for y, z in ((0.3, -0.2), (-1.1, 0.7)):
                p = torch.stack([x, torch.full_like(x, y), torch.full_like(x, z)], 1)
                got = union.query_sdf(p).double()
                # a depth changes by at most the step, 1e-3; the weights' sum is the depth of the deepest map above that of the one left
                # out, at the least
                depth = torch.stack([torch.minimum(p - m.bounding_box[:, 0].to(device), m.bounding_box[:, 1].to(device) - p).amin(1) for m in maps], 1)
                ranked = depth.clamp(min=0).sort(1, descending=True).values
                margin = ranked[:, 0] - (ranked[:, top] if top < len(maps) else 0.0)
                clear = torch.minimum(margin[1:], margin[:-1])
                jump = (got[1:] - got[:-1]).abs()
                # (a quotient of sums of `top` weights, each changing by 2e-3 at most, of values that are 4 apart at most; fp32; the 1e-6
                # share of a box that a map keeps at its edge)
                assert (jump <= 4 * 2 * top * 2e-3 / clear.clamp(min=1e-9) + 1e-5 / clear.clamp(min=1e-9) + 1e-5).all(), (top, float(jump.max()))
    union = AgentMaps(three)
    at = lambda v: float(union.query_sdf(torch.tensor([[v, 0.0, 0.0]], device=device)))          # noqa: E731
    assert abs(at(-1e-3)) < 1e-2 and abs(at(1e-3)) < 1e-2
    ids, w = union.route(torch.tensor([[1.0, 0.0, 0.0], [4.9, 0.0, 0.0], [2.5, 0.0, 0.0]], device=device))
    # depths 4, 1, 2 (0.1 and none; 2.5, none and 0.5): the third is left out at depth 1
    assert ids.tolist() == [[0, 2], [0, -1], [0, 2]] and torch.allclose(w.cpu(), torch.tensor([[0.75, 0.25], [1.0, 0.0], [2.5 / 3, 0.5 / 3]]), atol=1e-5)


# --------------------------------------------------------------------------------------------------- FusedAdamW: loaded states
def _stepped(p, **kw):
    opt = optim.FusedAdamW([p], **kw)
    p.grad = torch.ones_like(p)
    opt.step()
    return opt


def check_fused_adamw_loads_all_or_nothing(device):
    """A saved state that does not fit is refused, and the optimizer goes on as if nothing had been asked."""
    shape = (6, 5, 3, 4)
    p = torch.nn.Parameter(torch.ones(shape, device=device))
    good = {bits: _stepped(p, lr=0.5, state_bits=bits).state_dict() for bits in (8, 32)}

    def changed(bits, **kw):
        saved = {"param_groups": good[bits]["param_groups"], "state": {0: {**good[bits]["state"][0], **kw}}}
        return {**saved, "state": {0: {k: v for k, v in saved["state"][0].items() if v is not None}}}

    st = good[8]["state"][0]
    other_order = st["exp_avg"].contiguous(memory_format=torch.channels_last)
    bad = [changed(8, exp_avg=other_order, exp_avg_sq=other_order.to(torch.uint8)), changed(8, scales=st["scales"][:1]), changed(8, scales=None),
           changed(8, scales=st["scales"].to(torch.int32)), changed(8, exp_avg_sq=st["exp_avg"]), changed(8, exp_avg=st["exp_avg"].float()),
           changed(32, exp_avg=torch.ones(4, device=device)), changed(32, exp_avg_sq=torch.ones(1, 5, 3, 4, device=device)), changed(32, exp_avg=None),
           changed(32, step=None), changed(32, exp_avg=1.0)]
    for saved in bad:
        for bits in (8, 32):
            q = torch.nn.Parameter(torch.ones(shape, device=device))
            opt = _stepped(q, lr=0.25, state_bits=bits)
            before = {k: v.clone() if torch.is_tensor(v) else v for k, v in opt.state[q].items()}
            with pytest.raises(ValueError):
                opt.load_state_dict(saved)
            assert opt.param_groups[0]["lr"] == 0.25 and opt.param_groups[0]["state_bits"] == bits
            for k, v in before.items():
                assert torch.equal(opt.state[q][k], v) and opt.state[q][k].dtype == v.dtype if torch.is_tensor(v) else opt.state[q][k] == v
            opt.step()
    for bits in (8, 32):                                  # what fits is loaded, also through a hook that changes it
        q = torch.nn.Parameter(torch.ones(shape, device=device))
        opt = optim.FusedAdamW([q])
        hook = opt.register_load_state_dict_pre_hook(lambda _, sd: {**sd, "state": {0: {**sd["state"][0], "step": 7}}})
        opt.load_state_dict(good[bits])
        hook.remove()
        assert opt.state[q]["step"] == 7 and torch.equal(opt.state[q]["exp_avg"], good[bits]["state"][0]["exp_avg"])
        opt.load_state_dict(good[bits])
        assert opt.state[q]["step"] == 1
    empty = optim.FusedAdamW([torch.nn.Parameter(torch.zeros(0, 3, device=device))])
    empty.load_state_dict(empty.state_dict())


def check_fused_adamw_loads_no_other_decay(device):
    """States of optimizers that go on by another rule are refused, those that go on by the same are loaded."""
    def other(cls, **kw):
        p = torch.nn.Parameter(torch.ones(4))
        opt = cls([p], lr=0.5, **kw)
        p.grad = torch.ones_like(p)
        if cls is not optim.FusedAdam:
            opt.step()
        return opt.state_dict()

    for cls, kw in ((torch.optim.Adam, dict(weight_decay=0.1)), (torch.optim.NAdam, {}), (torch.optim.RAdam, {}), (torch.optim.Adamax, {}), (torch.optim.Adagrad, {}),
                    (torch.optim.SGD, dict(momentum=0.9)), (optim.FusedAdam, dict(weight_decay=1e-6)), (torch.optim.AdamW, dict(amsgrad=True))):
        opt = optim.FusedAdamW([torch.nn.Parameter(torch.ones(4, device=device))], lr=0.25)
        with pytest.raises(ValueError):
            opt.load_state_dict(other(cls, **kw))
        assert opt.param_groups[0]["lr"] == 0.25 and not opt.state, cls
    for cls, kw in ((torch.optim.Adam, {}), (torch.optim.AdamW, dict(weight_decay=0.1)), (torch.optim.AdamW, {}), (optim.FusedAdam, {}), (optim.FusedAdamW, {})):
        p = torch.nn.Parameter(torch.ones(4, device=device))
        opt = optim.FusedAdamW([p], lr=0.25)
        saved = other(cls, **kw) if cls is not optim.FusedAdamW else optim.FusedAdamW([torch.nn.Parameter(torch.ones(4))], lr=0.5).state_dict()
        opt.load_state_dict(saved)
        assert opt.param_groups[0]["lr"] == 0.5 and opt.param_groups[0]["weight_decay"] == saved["param_groups"][0]["weight_decay"]
        p.grad = torch.ones_like(p)
        opt.step()
        assert opt.state[p]["step"] == (2 if saved["state"] else 1)
        opt.param_groups[0]["weight_decay"] = 0.3                  # from here on the decay is this optimizer's
        again = optim.FusedAdamW([torch.nn.Parameter(torch.ones(4, device=device))])
        again.load_state_dict(opt.state_dict())
        assert again.param_groups[0]["weight_decay"] == 0.3


def check_fused_adamw_keeps_its_bits(device):
    """A state of torch.optim.AdamW says nothing of 8-bit moments: an optimizer made with them stays one, and refuses moments in 32 bits
    where it cannot go on from them."""
    p = torch.nn.Parameter(torch.ones(300))
    ref = torch.optim.AdamW([p], lr=0.5)
    fresh = ref.state_dict()
    p.grad = torch.ones_like(p)
    ref.step()
    q = torch.nn.Parameter(torch.ones(300, device=device))
    opt = optim.FusedAdamW([q], lr=0.25, state_bits=8, seed=6)
    with pytest.raises(ValueError, match="state_bits"):
        opt.load_state_dict(ref.state_dict())
    assert opt.param_groups[0]["lr"] == 0.25 and not opt.state
    opt.load_state_dict(fresh)                                            # no step taken: nothing to go on from
    assert opt.param_groups[0]["lr"] == 0.5 and opt.param_groups[0]["state_bits"] == 8 and opt.param_groups[0]["seed"] == 6
    q.grad = torch.ones_like(q)
    opt.step()
    assert opt.state[q]["exp_avg"].dtype == torch.int8
    saved = opt.state_dict()                                              # ... and what says so decides
    other = optim.FusedAdamW([torch.nn.Parameter(torch.ones(300, device=device))], state_bits=32, seed=1)
    other.load_state_dict(saved)
    assert other.param_groups[0]["state_bits"] == 8 and other.param_groups[0]["seed"] == 6
    mixed = {**saved, "param_groups": [{**saved["param_groups"][0], "state_bits": 32}]}
    with pytest.raises(ValueError, match="state_bits"):
        other.load_state_dict(mixed)
    with pytest.raises(ValueError):                                       # another number of groups: torch's own refusal
        other.load_state_dict({**saved, "param_groups": saved["param_groups"] * 2})


def check_fused_adamw_steps_all_or_nothing(device):
    """A step that is refused for one group has changed none; a gradient laid out otherwise is cleared like the others."""
    from mneslam_amd import _lib
    make = lambda *shape: torch.nn.Parameter(torch.ones(shape, device=device))                 # noqa: E731

    def refused(error, last, grad, bits=32, **kw):
        first, second = make(300), make(20)
        opt = optim.FusedAdamW([{"params": [first]}, {"params": [second], "lr": 0.5, "betas": (0.9, 0.99)}, {"params": [last]}], state_bits=bits)
        for p in (first, second):
            p.grad = torch.ones_like(p)
        opt.step()
        last.grad = grad
        before = [t.detach().clone() for p in (first, second) for t in (p, p.grad, *opt.moments(p))]
        with pytest.raises(error):
            opt.step(**kw)
        assert all(torch.equal(a, b) for a, b in zip(before, [t for p in (first, second) for t in (p, p.grad, *opt.moments(p))]))
        assert opt.state[first]["step"] == opt.state[second]["step"] == 1
        last.grad = None
        opt.step()
        assert opt.state[first]["step"] == 2 and not torch.equal(first, before[0])

    for bits in (8, 32):
        refused(RuntimeError, make(5), torch.ones(5, device=device).to_sparse(), bits)
        double = torch.nn.Parameter(torch.ones(5, device=device, dtype=torch.float64))
        refused(TypeError, double, torch.ones(5, device=device, dtype=torch.float64), bits)
        refused(ValueError, make(4, 5), torch.ones(1, 1, device=device).expand(4, 5), bits, zero_grad=True)
        refused(ValueError, torch.nn.Parameter(torch.ones(1, device=device).expand(5)), torch.ones(5, device=device), bits)
    offset, table = torch.zeros(1, dtype=torch.int32, device=device), torch.ones(9, 2, dtype=torch.float64, device=device)
    clock = _lib.Clock()
    clock.step_offset, clock.bias_table, clock.n_table, clock.beta1, clock.beta2 = offset.data_ptr(), table.data_ptr(), 9, 0.9, 0.999
    refused(RuntimeError, make(5), torch.ones(5, device=device), clock=clock)                   # (the second group has other betas)

    for bits in (8, 32):
        gen = torch.Generator().manual_seed(51)
        p, q = make(6, 7), make(6, 7)
        g = torch.randn(6, 7, generator=gen).to(device)
        opt = optim.FusedAdamW([p, q], state_bits=bits)
        p.grad, q.grad = g.clone(), g.t().contiguous().t()
        seen = q.grad
        opt.step(zero_grad=True)
        assert not p.grad.any() and q.grad is seen and not seen.any()
        want = optim.FusedAdamW([r := make(6, 7), s := make(6, 7)], state_bits=bits)
        r.grad, s.grad = g.clone(), g.clone()
        want.step()
        assert torch.equal(p, r) and torch.equal(q, s)
    p = torch.ones(300, device=device)
    scales = torch.zeros(5, device=device)[1:].view(2, 2)                                     # not at a multiple of 8 bytes
    with pytest.raises(ValueError, match="scales"):
        optim.adamw_step([p], [p.clone()], [p.to(torch.int8)], [p.to(torch.uint8)], [scales], step=1, lr=0.1)


def check_adamw_gradient_in_written_memory(device):
    """A gradient that lies over what the step writes would be read half before and half after: refused, unless it is a tensor's own
    memory element for element."""
    flat = torch.arange(1000.0, device=device)
    p, q = flat[:300], flat[300:600]
    for bits in (8, 32):
        states = [_state_for(t, bits, device) for t in (p, q)]
        before = flat.clone()
        m = states[0][0][0]
        for grads in ([flat[1:301], q.clone()], [flat[600:900], flat[450:750]], [q, q.clone()], [q, p], [flat[299:599], q.clone()]) + \
                (([m.new_ones(300), m],) if bits == 32 else ()):
            with pytest.raises(ValueError, match="overlap"):
                _step([p, q], grads, bits, device, state=states)
        assert torch.equal(flat, before) and not m.any()
        _step([p, q], [flat[600:900], flat[650:950]], bits, device, state=states)            # beside it, and shared
        assert torch.equal(flat[600:], before[600:]) and not torch.equal(p, before[:300])
    p, g = torch.ones(300, device=device), torch.ones(300, device=device)
    _step([p], [p], 32, device)
    _step([g], [g.clone()], 32, device)
    assert torch.equal(p, g)


def check_adamw_outdates_what_it_writes(device):
    """What autograd has saved of anything that a step writes is out of date: parameters, moments, scales, gradients that it clears."""
    for bits in (8, 32):
        p, g = torch.ones(300, device=device), torch.ones(300, device=device)
        (m, v), s = state = _state_for(p, bits, device)
        written = [t for t in (p, m, v, s) if t is not None]
        old = [t._version for t in written + [g]]
        _step([p], [g], bits, device, state=[state])
        assert all(t._version > n for t, n in zip(written, old)) and g._version == old[-1]
        w = torch.ones(300, device=device, requires_grad=True)
        products = [(w * t) for t in [g] + [t for t in written if t.is_floating_point() and t.numel() == 300]]
        _step([p], [g], bits, device, step=2, state=[state], zero_grad=True)
        for out in products:
            with pytest.raises(RuntimeError, match="inplace"):
                out.sum().backward()
        with torch.inference_mode():
            q, h = torch.ones(5, device=device), torch.ones(5, device=device)
            _step([q], [h], bits, device, zero_grad=True)
            assert (q < 1).all() and not h.any()


def check_plan_tensors_are_apart(device):
    """A plan's tensors are memory of their own: writing into one touches no other, in value or in autograd's eyes, and no workspace stays."""
    from mneslam_amd.routing import expert_combine, expert_dispatch, expert_sort
    for n, k, e in ((4, 2, 3), (3000, 2, 3), (5000, 1, 2500), (0, 2, 3)):
        ids = torch.zeros(n, k, dtype=torch.int32, device=device)
        plan = expert_sort(ids, e)
        for t in (plan.order, plan.position, plan.offsets):
            assert t.untyped_storage().nbytes() == 4 * t.numel() and t.is_contiguous()
        x = torch.ones(n, 2, device=device, requires_grad=True)
        out = expert_combine(expert_dispatch(x, plan), plan)
        plan.order.fill_(-1)
        out.sum().backward()
        assert (x.grad == k).all() and plan.offsets.tolist() == [0] + [n * k] * e and plan.position.reshape(-1).tolist() == list(range(n * k))


def check_adamw8_follows_32(device):
    """A hundred steps with 8-bit moments go where 32-bit ones go.  The gradient is constant, so a step is lr, and every |m| and sqrt(v) of a
    block lies between half its largest and that:
    a code step of m is (2 c + 1) / c^2 of it, c >= 89: at most 2.3 %; a dither's deviation is at most half of that, and the running mean
    with beta 0.9 holds 0.9 / sqrt(1 - 0.81) = 2.1 times one step's: 2.4 %.  Of sqrt(v): c >= 180, 0.56 %, and with beta 0.99 at most 7.1
    times: 4.0 %.  One step is off by 4.7 % of lr (one deviation), the sum of a hundred by no more than that of a hundred lr: five
    deviations are 24 %.  On average over n elements only the squares stay: (4.0 %)^2 from dividing by sqrt(v), and 0.0056^2 / 0.01 / 2
    from v's mean, 0.32 % together; and 5 * 4.7 % / sqrt(n)."""
    n, steps, lr = 256 * 64, 100, 2.0 ** -8
    gen = torch.Generator().manual_seed(61)
    g = ((0.5 + 0.5 * torch.rand(n, generator=gen)) * torch.where(torch.rand(n, generator=gen) < 0.5, -1.0, 1.0)).to(device)
    ends = []
    for bits in (8, 32):
        p, state = torch.zeros(n, device=device), None
        for step in range(1, steps + 1):
            state = _step([p], [g], bits, device, step=step, state=state, lr=lr)
        ends.append((p * -torch.sign(g)).double() / (steps * lr))
    assert (ends[1] - 1).abs().max() < 1e-5
    assert (ends[0] - 1).abs().max() < 0.24
    assert abs(float(ends[0].mean()) - 1) < 0.0032 + 5 * 0.047 / n ** 0.5


def check_fused_adamw_loads_no_scales_with_32_bits(device):
    """Scales beside 32-bit moments would be taken for codes' by ``moments``: refused."""
    p = torch.nn.Parameter(torch.ones(300, device=device))
    saved = _stepped(p).state_dict()
    saved = {**saved, "state": {0: {**saved["state"][0], "scales": torch.ones(2, 2)}}}
    opt = _stepped(torch.nn.Parameter(torch.ones(300, device=device)))
    with pytest.raises(ValueError, match="scales"):
        opt.load_state_dict(saved)
    assert "scales" not in opt.state[opt.param_groups[0]["params"][0]]
