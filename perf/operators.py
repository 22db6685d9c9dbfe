"""The operators of a model made of several expert maps, as cases that can be timed and compared.

``adamw``   one AdamW step over many tensors at once, moments in 32 bits or in 8 (blocks of 256 elements with two scales)
``route``   a batch of points or tokens sorted by expert, dealt to the experts' rows and blended back with weights, as it is
            served (``grad`` false) and as it is trained (``grad`` true: the gradients of rows, tokens and weights as well)

``run`` computes them in plain torch operations where ``own`` is false, and through mneslam_amd where it is true.
"""
import itertools
import math

import torch

own = False

DEV = "cuda"
BLOCK = 256                      # elements that share the two scales of an 8-bit state
GOLD, MIX1, MIX2 = 0x9E3779B1, 0x7FEB352D, 0x846CA68B
LR, BETAS, EPS, DECAY, SEED = 0.005, (0.9, 0.99), 1e-8, 0.01, 20
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    adamw, route = {"op": "adamw"}, {"op": "route"}
    return [
        # the four weight matrices of a 2 x 32 decoder: the optimizer call of every mapping iteration, all latency
        {**adamw, "name": "adamw decoder", "bits": 32, "param": "float32", "grads": "float32", "tensors": 4, "elements": 6208},
        {**adamw, "name": "adamw8 decoder", "bits": 8, "param": "float32", "grads": "float32", "tensors": 4, "elements": 6208},
        # the planes of one indoor map: 38.4 million values in twelve tensors, a few of them holding most
        {**adamw, "name": "adamw planes", "bits": 32, "param": "float32", "grads": "float32", "tensors": 12, "elements": 38400000},
        {**adamw, "name": "adamw8 planes", "bits": 8, "param": "float32", "grads": "float32", "tensors": 12, "elements": 38400000},
        # many experts' matrices in 16 bits: hundreds of odd sizes in one call
        {**adamw, "name": "adamw experts", "bits": 32, "param": "bfloat16", "grads": "bfloat16", "tensors": 256, "elements": 67000000},
        {**adamw, "name": "adamw8 experts", "bits": 8, "param": "bfloat16", "grads": "bfloat16", "tensors": 256, "elements": 67000000},
        # one token between two steps of serving
        {**route, "name": "route one token", "grad": False, "tokens": 1, "top": 2, "experts": 8, "dim": 1024, "out": 1024, "type": "bfloat16", "padded": 0.0},
        # the points of one iteration (2150 rays of 128 samples) dealt to eight agents' maps, (r, g, b, sdf) coming back
        {**route, "name": "route points", "grad": False, "tokens": 275200, "top": 2, "experts": 8, "dim": 3, "out": 4, "type": "float32", "padded": 0.1},
        # the largest served batch
        {**route, "name": "route batch", "grad": False, "tokens": 131071, "top": 4, "experts": 64, "dim": 2048, "out": 2048, "type": "bfloat16", "padded": 0.0},
        # training: the features of the samples with one expert each, odd rows
        {**route, "name": "route features grad", "grad": True, "tokens": 275200, "top": 1, "experts": 1000, "dim": 65, "out": 65, "type": "float32", "padded": 0.05},
        # training: rows of a wide layer
        {**route, "name": "route rows grad", "grad": True, "tokens": 16384, "top": 2, "experts": 64, "dim": 1024, "out": 1024, "type": "bfloat16", "padded": 0.02},
        # training: a small ragged batch with many choices
        {**route, "name": "route ragged grad", "grad": True, "tokens": 777, "top": 8, "experts": 129, "dim": 320, "out": 320, "type": "float16", "padded": 0.3},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.45:
        param = rng.choice(["float32", "bfloat16", "float16"])
        tensors = _log(rng, 1, 300)
        return {"op": "adamw", "bits": rng.choice([8, 32]), "param": param, "grads": rng.choice([param, "float32"]),
                "tensors": tensors, "elements": tensors * 8 + _log(rng, 100, 38000000)}
    top, grad, kind = rng.randint(1, 8), rng.random() < 0.5, rng.choice(["float32", "bfloat16", "float16"])
    dim = _log(rng, 1, 2048)
    if rng.random() < 0.5:
        dim = -(-dim // 8) * 8                              # half of the widths are whole vectors, half are as they come
    rows = max(top, min(1 << 20, (1 << 27) // dim))         # rows * dim stays below the largest listed case's
    tokens = _log(rng, 1, rows // top)
    return {"op": "route", "grad": grad, "tokens": tokens, "top": top, "experts": _log(rng, 1, 4096), "dim": dim,
            "out": dim if grad else rng.choice([dim, max(1, dim // 2)]), "type": kind, "padded": rng.choice([0.0, 0.1, 0.5])}


def _sizes(case):
    """Element counts of the tensors: shares fall off geometrically for a dozen tensors, and vary around their mean for many."""
    k, n = case["tensors"], case["elements"]
    if case["tensors"] == 4 and n == 6208:
        return [2016, 96, 3584, 512]                        # w_col0, w_col1, w_sdf0, w_sdf1
    share = [0.7 ** i for i in range(k)] if k <= 16 else [1.0 + 0.5 * math.sin(2.4 * i) for i in range(k)]
    got = [max(1, int(n * s / sum(share))) for s in share]
    got[0] += max(0, n - sum(got))
    return got


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (_prepare_adamw if case["op"] == "adamw" else _prepare_route)(case, g)


def _prepare_adamw(case, g):
    """Parameters, gradients and moments, each kind in one buffer that the tensors are cut from at multiples of 256."""
    sizes = _sizes(case)
    blocks = [-(-n // BLOCK) for n in sizes]
    starts = [BLOCK * b for b in itertools.accumulate([0] + blocks[:-1])]
    total = BLOCK * sum(blocks)
    ordinal = torch.arange(len(sizes), device=DEV).repeat_interleave(torch.tensor(blocks, device=DEV))    # the tensor of a block
    block = torch.arange(total // BLOCK, device=DEV) - torch.tensor(starts, device=DEV)[ordinal] // BLOCK  # its number in there
    live = (block[:, None] * BLOCK + torch.arange(BLOCK, device=DEV) < torch.tensor(sizes, device=DEV)[ordinal][:, None]).reshape(-1)
    randn = lambda: torch.randn(total, generator=g, device=DEV)          # noqa: E731
    rand = lambda: torch.rand(total, generator=g, device=DEV)            # noqa: E731
    size = torch.exp(2.0 * torch.randn(total // BLOCK, generator=g, device=DEV)).repeat_interleave(BLOCK) * 1e-3
    grad = randn() * size * (rand() > 0.3)                               # a third of a map's cells is hit by no sample
    s = {"case": case, "sizes": sizes, "starts": starts, "step": 100,
         "p": (0.1 * randn() * live).to(TYPES[case["param"]]), "g": (grad * live).to(TYPES[case["grads"]])}
    if case["bits"] == 32:
        s["m"], s["v"] = 0.3 * randn() * size * live, torch.square(size * (0.2 + rand())) * live
    else:
        s["m"] = (randn() * 40).clamp(-127, 127).to(torch.int8) * live
        s["v"] = (1 + 254 * rand()).to(torch.uint8) * live
        scale = size[::BLOCK]
        s["scales"] = torch.stack([scale / 16129, 2 * scale / 65025], 1).contiguous()
    cut = lambda t: [t[a:a + n] for a, n in zip(starts, sizes)]          # noqa: E731
    s["params"], s["grads"], s["exp_avg"], s["exp_avg_sq"] = cut(s["p"]), cut(s["g"]), cut(s["m"]), cut(s["v"])
    if case["bits"] == 8:
        s["scale"] = [s["scales"][a // BLOCK:a // BLOCK + -(-n // BLOCK)] for a, n in zip(starts, sizes)]
        s["ordinal"], s["block"] = ordinal, block
    return s


def _prepare_route(case, g):
    n, k, e, t = case["tokens"], case["top"], case["experts"], TYPES[case["type"]]
    popular = torch.rand(e, generator=g, device=DEV) ** 3 + 1e-3          # some experts take many rows, some next to none
    edges = torch.cumsum(popular, 0)
    ids = torch.searchsorted(edges, torch.rand(n, k, generator=g, device=DEV) * edges[-1]).clamp(max=e - 1)
    ids = torch.where(torch.rand(n, k, generator=g, device=DEV) < case["padded"], -1, ids)
    s = {"case": case, "ids": ids.to(torch.int32), "x": torch.randn(n, case["dim"], generator=g, device=DEV).to(t),
         "y": torch.randn(n * k, case["out"], generator=g, device=DEV).to(t),
         "w": torch.softmax(torch.randn(n, k, generator=g, device=DEV), 1)}
    if case["grad"]:
        s["dxs"] = torch.randn(n * k, case["dim"], generator=g, device=DEV).to(t)
        s["dout"] = torch.randn(n, case["out"], generator=g, device=DEV).to(t)
        for name in ("x", "y", "w"):
            s[name].requires_grad_(True)
    return s


def run(s):
    if own:
        return _own_adamw(s) if s["case"]["op"] == "adamw" else _own_route(s)
    return _plain_adamw(s) if s["case"]["op"] == "adamw" else _plain_route(s)


def _own_adamw(s):
    from mneslam_amd.optim import adamw_moments, adamw_step
    s["step"] += 1
    adamw_step(s["params"], s["grads"], s["exp_avg"], s["exp_avg_sq"], s.get("scale"), step=s["step"], lr=LR, betas=BETAS,
               eps=EPS, weight_decay=DECAY, seed=SEED)
    if s["case"]["bits"] == 32:
        return {"p": s["p"], "m": s["m"], "v": s["v"]}
    m, v = adamw_moments(s["m"], s["v"], s["scales"])
    return {"p": s["p"], "m": m, "v": v}


def _own_route(s):
    from mneslam_amd.routing import expert_combine, expert_dispatch, expert_sort
    plan = expert_sort(s["ids"], s["case"]["experts"])
    xs = expert_dispatch(s["x"], plan)
    out = expert_combine(s["y"], plan, s["w"])
    got = {"order": plan.order, "position": plan.position, "offsets": plan.offsets, "xs": xs, "out": out}
    if s["case"]["grad"]:
        got["dx"], got["dy"], got["dw"] = torch.autograd.grad((xs, out), (s["x"], s["y"], s["w"]), (s["dxs"], s["dout"]))
    return got


def _constants(step, beta1, beta2):
    return LR / (1.0 - beta1 ** step), math.sqrt(1.0 - beta2 ** step), 1.0 - LR * DECAY


def _root(x):
    """The square root rounded once: what is next to a border of the 8-bit codes has to fall on its own side."""
    return torch.sqrt(x.double()).float()


def _plain_adamw(s):
    s["step"] += 1
    (b1, b2), bits = BETAS, s["case"]["bits"]
    size, root_bc2, decay = _constants(s["step"], b1, b2)
    g = s["g"].float()
    if bits == 32:
        m, v = s["m"], s["v"]
    else:
        m, r = _plain_values(s["m"], s["v"], s["scales"])
        v = r * r
    m = m * b1 + g * (1.0 - b1)
    v = v * b2 + (g * g) * (1.0 - b2)
    r = _root(v)
    s["p"].copy_(s["p"].float() * decay - size * (m / (r / root_bc2 + EPS)))
    if bits == 32:
        s["m"].copy_(m)
        s["v"].copy_(v)
        return {"p": s["p"], "m": s["m"], "v": s["v"]}
    um, ur = _dither(s["ordinal"], s["block"], s["step"])
    m, r = m.reshape(-1, BLOCK), r.reshape(-1, BLOCK)
    mc, ms = _encode(m.abs(), um, 16129.0, 127, 2.0 ** -100)
    rc, rs = _encode(r, ur, 65025.0, 255, 0.0)
    rc = torch.where((rc == 0) & (r > 0) & torch.isfinite(rs)[:, None], 1, rc)
    s["m"].copy_((torch.sign(torch.nan_to_num(m)) * mc).to(torch.int8).reshape(-1))
    s["v"].copy_(rc.to(torch.uint8).reshape(-1))
    s["scales"].copy_(torch.stack([ms, rs], 1))
    m, r = _plain_values(s["m"], s["v"], s["scales"])
    return {"p": s["p"], "m": m, "v": r * r}


def _plain_values(mc, rc, scales):
    """What the codes stand for: the first moment, and the square root of the second."""
    scale = scales.repeat_interleave(BLOCK, 0)
    mc, rc = mc.float(), rc.float()
    return mc * mc.abs() * scale[:, 0], rc * rc * scale[:, 1]


def _encode(x, u, top, most, least):
    """Codes c with c^2 standing for x * top / max(x), rounded up with the dither's probability, and the scale of each block."""
    big = x.max(1).values
    fine = torch.isfinite(x).all(1)
    zero = big <= least
    scale = torch.where(fine, torch.where(zero, 0.0, (big.double() / top).float()), math.nan)
    y = x * torch.where(fine & ~zero, (top / big.double()).float(), 0.0)[:, None]
    y = torch.where(fine[:, None], y, 0.0)
    c = torch.floor(torch.sqrt(y.double())).float()
    c = c + (u * (2.0 * c + 1.0) < y - c * c)
    return c.clamp(max=most), scale


def _mix(h):
    h = (h ^ (h >> 16)) * MIX1 & 0xFFFFFFFF
    h = (h ^ (h >> 15)) * MIX2 & 0xFFFFFFFF
    return h ^ (h >> 16)


def _dither(ordinal, block, step):
    """Two 16-bit dithers an element, from the seed, the tensor's place in the list, the step, the block and the element."""
    key = _mix((SEED + ordinal * GOLD) & 0xFFFFFFFF)
    key = _mix(((key + step * GOLD) & 0xFFFFFFFF) ^ _mix(block & 0xFFFFFFFF))
    h = (key[:, None] + torch.arange(BLOCK, device=block.device) * GOLD) & 0xFFFFFFFF
    h = (h ^ (h >> 16)) * MIX1 & 0xFFFFFFFF
    h = h ^ (h >> 15)
    return (h & 0xFFFF).float() / 65536.0, (h >> 16).float() / 65536.0


def _plain_sort(ids, experts):
    flat = ids.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < experts), flat, experts)
    order = torch.argsort(key, stable=True)
    offsets = torch.searchsorted(key[order], torch.arange(experts + 1, device=ids.device))
    rows = torch.arange(flat.numel(), device=ids.device)
    position = torch.empty_like(order)
    position[order] = rows
    live = rows < offsets[-1]
    order = torch.where(live, order, -1)
    position = torch.where(key < experts, position, -1).reshape(ids.shape)
    return order.int(), position.int(), offsets.int(), live


def _take(rows, position):
    """The rows of each token's slots in 32 bits, [tokens, top, width]; zeros where a slot has no expert."""
    return torch.where((position >= 0)[..., None], rows[position.clamp(min=0).long()].float(), 0.0)


def _plain_route(s):
    k, w, t = s["case"]["top"], s["w"].detach(), TYPES[s["case"]["type"]]
    x, y = s["x"].detach(), s["y"].detach()
    order, position, offsets, live = _plain_sort(s["ids"], s["case"]["experts"])
    slot = order.clamp(min=0).long()
    xs = torch.where(live[:, None], x[slot // k], 0.0).to(t)
    ys = _take(y, position)
    got = {"order": order, "position": position, "offsets": offsets, "xs": xs, "out": (ys * w[..., None]).sum(1).to(t)}
    if s["case"]["grad"]:
        dout = s["dout"].float()
        got["dx"] = _take(s["dxs"], position).sum(1).to(t)
        got["dy"] = torch.where(live[:, None], dout[slot // k] * w.reshape(-1)[slot][:, None], 0.0).to(t)
        got["dw"] = (ys * dout[:, None]).sum(2)
    return got


def work(case):
    if case["op"] == "adamw":
        n, sp, sg = sum(_sizes(case)), TYPES[case["param"]].itemsize, TYPES[case["grads"]].itemsize
        # the step itself, and with 8-bit moments their values in 32 bits, which are asked for behind it
        state = 16 if case["bits"] == 32 else 4 + 16 / BLOCK + 8
        return {"bytes": n * (2 * sp + sg + state), "flops": 14 * n}
    n, k, d, o, e = case["tokens"], case["top"], case["dim"], case["out"], TYPES[case["type"]].itemsize
    slots = n * k
    taken = slots * (1 - case["padded"])
    size = slots * 12 + 4 * case["experts"] + (n + slots) * d * e + (taken + n) * o * e + slots * 4
    flops = 2 * taken * o
    if case["grad"]:
        size += (taken + n) * d * e + (n + taken + slots) * o * e + 4 * slots
        flops += taken * (d + 3 * o)
    return {"bytes": size, "flops": flops}


def exact(case, seed):
    """In 64 bits. The moments that are held in 8 bits have no value of this kind: which of two neighbouring codes is taken is
    decided by IEEE 32-bit arithmetic next to a border, and that is part of what the operator is."""
    s = prepare(case, seed)
    if case["op"] == "adamw":
        (b1, b2), step = BETAS, s["step"] + 1
        size, root_bc2, decay = _constants(step, b1, b2)
        g, p, m, v = s["g"].double(), s["p"].double(), s["m"].double(), s["v"].double()
        if case["bits"] == 8:
            per_block = lambda i: s["scales"][:, i:i + 1].double().expand(-1, BLOCK).reshape(-1)      # noqa: E731
            m, v = torch.sign(m) * torch.square(m) * per_block(0), torch.square(torch.square(v) * per_block(1))
        m, v = torch.lerp(g, m, b1), torch.lerp(torch.square(g), v, b2)
        p = p * decay - size * m / (v.sqrt() / root_bc2 + EPS)
        return {"p": p, "m": m, "v": v} if case["bits"] == 32 else {"p": p, "m": None, "v": None}
    n, k, e = case["tokens"], case["top"], case["experts"]
    ids, w = s["ids"].reshape(-1).cpu(), s["w"].detach().double()
    slots = torch.nonzero((ids >= 0) & (ids < e)).reshape(-1)
    slots = slots[torch.sort(ids[slots], stable=True).indices].to(DEV)                # slot of each live row
    live = slots.numel()
    token = slots // k
    at = torch.arange(live, device=DEV)

    def rows(width, values):
        full = torch.zeros(n * k, width, dtype=torch.float64, device=DEV)
        full[:live] = values
        return full

    x, y = s["x"].detach().double(), s["y"].detach().double()
    share = w.reshape(-1)[slots][:, None]
    got = {"order": None, "position": None, "offsets": None, "xs": rows(case["dim"], x[token]),
           "out": torch.zeros(n, case["out"], dtype=torch.float64, device=DEV).index_add_(0, token, share * y[at])}
    if case["grad"]:
        dout = s["dout"].double()[token]
        got["dx"] = torch.zeros_like(x).index_add_(0, token, s["dxs"][at].double())
        got["dy"] = rows(case["out"], share * dout)
        got["dw"] = torch.zeros(n * k, dtype=torch.float64, device=DEV).index_put_((slots,), (dout * y[at]).sum(1)).reshape(n, k)
    return got
