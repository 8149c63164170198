"""The optimiser and table operators as users call them, as cases that can be timed and compared with their plain forms.

A case is a dict of plain values; its "kind" says which operator a pass goes through:

  adamw   AdamW.step(): one step over many tensors, moments in 32 or in 8 bits, with clipping by the global norm or without
  norm    grad_norm(): the global norm of many gradients and the factor that clips them
  look    lookup(): rows (or columns) of a table by index, scaled
  grad    lookup_backward(): the gradient of a table from the gradient of its looked-up entries, ordered within the call
          or by an order that the program keeps
  plan    lookup_plan(): the order of the entries by their index, and where each index begins

Tensors of an optimiser lie in one flat buffer per kind, as in a program that exchanges them between ranks: packed one
behind the other, or each from a multiple of 256 elements. "sizes" names the tensors: the net's, a point cloud's, or a
generic list of so many tensors with sizes spread over a geometric range.
"""
import math

import torch

own = False

BENCH_NET = "16,32,64,64"       # the benchmark's net: four levels
DEFAULT_NET = "32,32,32,32,32"  # MultiScaleUnet2dParams' own: five levels of 32
BLOCK = 256                     # elements that share a scale in 8 bits
BETAS, EPS, DECAY, LR = (0.9, 0.999), 1e-8, 1e-2, 1e-3
SEED = 12345                    # of the optimiser's rounding
DTYPES = dict(f32=torch.float32, bf16=torch.bfloat16, f16=torch.float16)
BYTES = dict(f32=4, bf16=2, f16=2, none=0)


def _adamw(sizes, *, bits=32, weights="f32", grads="f32", copy="none", clip=0.0, packed=False):
    return dict(kind="adamw", sizes=sizes, bits=bits, weights=weights, grads=grads, copy=copy, clip=clip, packed=packed)


def _norm(sizes, *, grads="f32", clip=1.0, packed=False):
    return dict(kind="norm", sizes=sizes, grads=grads, clip=clip, packed=packed)


def _table(kind, *, layout, texels, points, channels=1, dtype="f32", skew=1.0, outside=0.0, index="i32", kept=False):
    return dict(kind=kind, layout=layout, texels=texels, points=points, channels=channels, dtype=dtype, skew=skew,
                outside=outside, index=index, kept=kept)


def listed():
    return [
        # the benchmark's net in a training step: 18 small tensors, clipped; launches and host time
        dict(name="adamw_net_clip", **_adamw("net:" + BENCH_NET, clip=1.0)),
        # position, size, descriptors and confidence of the benchmark's 6M points
        dict(name="adamw_points_6M", **_adamw("points:6000000:4")),
        # the same cloud with its moments in 8 bits
        dict(name="adamw_points_6M_8bit", **_adamw("points:6000000:4", bits=8)),
        # a larger net: 40 tensors of 257 to 400k elements packed into flat buffers, bfloat16 gradients, a bfloat16 copy
        dict(name="adamw_packed_8bit_bf16", **_adamw("spread:40:257:400003", bits=8, grads="bf16", copy="bf16", clip=1.0,
                                                    packed=True)),
        # the default net's gradients before a step of any optimiser
        dict(name="norm_net", **_norm("net:" + DEFAULT_NET)),
        # all gradients of the benchmark's cloud
        dict(name="norm_points_6M", **_norm("points:6000000:4")),
        # token embeddings in bfloat16: a batch of 8191 tokens, frequent ones first, some of it padding
        dict(name="look_tokens_bf16", **_table("look", layout="rows", texels=50_000, points=8191, channels=1024, dtype="bf16",
                                               skew=3.0, outside=0.05, index="i64")),
        # descriptors shared by four points each, points in no order
        dict(name="look_6M_shared", **_table("look", layout="columns", texels=1_500_000, points=6_000_000, channels=4)),
        # the gradient of the token embeddings, ordered within the call
        dict(name="grad_tokens_bf16", **_table("grad", layout="rows", texels=50_000, points=8191, channels=1024, dtype="bf16",
                                               skew=3.0, outside=0.05, index="i64")),
        # the gradient of the shared descriptors; the points' texels stay the same, so their order is kept
        dict(name="grad_6M_shared_kept", **_table("grad", layout="columns", texels=1_500_000, points=6_000_000, channels=4,
                                                  kept=True)),
        # the order of a small object's points
        dict(name="plan_20k", **_table("plan", layout="columns", texels=5_000, points=20_000)),
        # the order of the benchmark's points, each with a texel of its own on average
        dict(name="plan_6M", **_table("plan", layout="columns", texels=6_000_000, points=6_000_000)),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_sizes(rng, most):
    kind = rng.choice(("net", "points", "spread", "spread"))
    if kind == "net":
        levels = rng.randint(2, 6)
        return "net:" + ",".join(str(rng.choice((16, 24, 32, 48, 64))) for _ in range(levels))
    if kind == "points":
        channels = rng.choice((3, 4, 6, 8, 16))
        return "points:%d:%d" % (_log_int(rng, 1000, most // (6 + channels)), channels)
    largest = _log_int(rng, 300, most // 20)
    return "spread:%d:%d:%d" % (rng.randint(1, 60), _log_int(rng, 1, 256), largest)


def draw(rng):
    kind = rng.choice(("adamw", "adamw", "norm", "look", "grad", "grad", "plan"))
    if kind == "adamw":
        return _adamw(_draw_sizes(rng, 45_000_000), bits=rng.choice((32, 8)), weights=rng.choice(("f32", "f32", "bf16", "f16")),
                      grads=rng.choice(("f32", "bf16", "f16")), copy=rng.choice(("none", "bf16", "f16")),
                      clip=rng.choice((0.0, 0.5, 1.0)), packed=rng.random() < 0.5)
    if kind == "norm":
        return _norm(_draw_sizes(rng, 60_000_000), grads=rng.choice(("f32", "bf16", "f16")), clip=rng.choice((0.1, 1.0, 10.0)),
                     packed=rng.random() < 0.5)
    skew, outside = rng.choice((1.0, 1.0, 2.0, 4.0)), rng.choice((0.0, 0.0, 0.1))
    index = rng.choice(("i32", "i64"))
    if kind == "plan":
        return _table("plan", layout="columns", texels=_log_int(rng, 1, 6_000_000), points=_log_int(rng, 1, 6_000_000),
                      skew=skew, outside=outside, index=index)
    layout, dtype = rng.choice(("columns", "rows")), rng.choice(("f32", "bf16", "f16"))
    channels = rng.choice((1, 3, 4, 6, 8, 16)) if layout == "columns" else _log_int(rng, 1, 2048)
    most = min(6_000_000 if layout == "columns" else 2_000_000, 24_000_000 // channels)
    return _table(kind, layout=layout, texels=_log_int(rng, 1, most), points=_log_int(rng, 1, most), channels=channels, dtype=dtype,
                  skew=skew, outside=outside, index=index, kept=kind == "grad" and rng.random() < 0.5)


# ---- sizes ----

def tensor_sizes(sizes):
    """Elements of each tensor that "sizes" names."""
    kind, *rest = sizes.split(":")
    if kind == "points":
        n, c = int(rest[0]), int(rest[1])
        return [4 * n, n, c * n, n]
    if kind == "spread":
        count, lo, hi = (int(v) for v in rest)
        ratio = (hi / lo) ** (1.0 / max(count - 1, 1))
        return [max(1, int(lo * ratio ** i)) for i in range(count)]
    filters, c, got = [int(f) for f in rest[0].split(",")], 4, []
    for i, f in enumerate(filters):
        last = i == len(filters) - 1
        cin = c if last else c + filters[i + 1]
        cout = f - (c if i == 0 and not last else 2 * c)
        got += [cout * cin * 9, cout, cout * cin * 9, cout]
    return got + [3 * filters[0], 3]


def _offsets(sizes, packed):
    at, got = 0, []
    for n in sizes:
        got.append(at)
        at += n if packed else -(-n // BLOCK) * BLOCK
    return got, at


# ---- inputs ----

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _moments(case, seed, total, blocks):
    """Moments as a run of some hundred steps leaves them."""
    g = _generator(seed * 7 + 1)
    if case["bits"] == 32:
        m = torch.randn(total, device="cuda", generator=g) * 0.003
        return dict(m=m, v=(torch.randn(total, device="cuda", generator=g) * 0.01).square_())
    m = (torch.randn(total, device="cuda", generator=g) * 60).to(torch.float8_e4m3fn)
    v = (torch.randn(total, device="cuda", generator=g).square_() * 3000).clamp_(2.0 ** -16, 57344.0).to(torch.float8_e5m2)
    ms = torch.exp2(torch.randint(-16, -13, (blocks,), device="cuda", generator=g).float())
    vs = torch.exp2(torch.randint(-26, -22, (blocks,), device="cuda", generator=g).float())
    return dict(m=m, v=v, ms=ms, vs=vs)


def _prepare_optimiser(case, seed):
    sizes = tensor_sizes(case["sizes"])
    at, total = _offsets(sizes, case["packed"])
    g = _generator(seed)
    grads = torch.randn(total, device="cuda", generator=g).mul_(0.01)
    real = torch.zeros(total, device="cuda", dtype=torch.bool)
    for o, n in zip(at, sizes):
        real[o:o + n] = True
    grads = grads.mul_(real).to(DTYPES[case["grads"]])
    s = dict(case=case, sizes=sizes, at=at, grads=grads)
    if case["kind"] == "norm":
        if own:
            s["list"] = [grads[o:o + n] for o, n in zip(at, sizes)]
        return s
    s["w"] = torch.randn(total, device="cuda", generator=g).mul_(0.05).mul_(real).to(DTYPES[case["weights"]])
    if case["copy"] != "none":
        s["copy"] = s["w"].to(DTYPES[case["copy"]])
    blocks_of = [-(-n // BLOCK) for n in sizes]
    s.update(_moments(case, seed, total, sum(blocks_of)))
    for k in ("m", "v"):
        # (what lies between two tensors belongs to none: zeros, as the padding of a flat buffer is)
        if case["bits"] == 32:
            s[k].mul_(real)
        else:
            s[k].view(torch.uint8).mul_(real)
    s["steps"] = torch.full((len(sizes),), 100 + seed % 50, dtype=torch.int32, device="cuda")
    if case["bits"] == 8 and case["packed"]:
        # place of each element when every tensor begins at a multiple of a block
        wide, _ = _offsets(sizes, False)
        s["place"] = torch.cat([torch.arange(w, w + n, device="cuda") for w, n in zip(wide, sizes)])
    if own:
        from trips_amd.adamw import AdamW
        params = []
        for o, n in zip(at, sizes):
            p = torch.nn.Parameter(s["w"][o:o + n])
            p.grad = grads[o:o + n] if grads.dtype == p.dtype else None
            params.append(p)
        opt = AdamW(params, lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, state_bits=case["bits"], min_8bit_size=0,
                    max_grad_norm=case["clip"], seed=SEED)
        b = 0
        for i, (p, o, n) in enumerate(zip(params, at, sizes)):
            st = dict(step=s["steps"][i], first_moment=s["m"][o:o + n], second_moment=s["v"][o:o + n])
            if case["bits"] == 8:
                st.update(first_scale=s["ms"][b:b + blocks_of[i]], second_scale=s["vs"][b:b + blocks_of[i]])
            b += blocks_of[i]
            opt.state[p] = st
            if case["copy"] != "none":
                opt.set_copy(p, s["copy"][o:o + n])
        s["opt"] = opt
        # gradients of another type than their weights are handed over
        s["handed"] = None if grads.dtype == s["w"].dtype else {p: grads[o:o + n] for p, o, n in zip(params, at, sizes)}
    return s


def _prepare_table(case, seed):
    g = _generator(seed)
    n, t, c, dt = case["points"], case["texels"], case["channels"], DTYPES[case["dtype"]]
    # frequent indexes first: a power of a uniform number
    u = torch.rand(n, device="cuda", generator=g, dtype=torch.float64).pow_(case["skew"])
    index = (u * t).to(torch.int64).clamp_(0, t - 1)
    if case["outside"] > 0:
        index[torch.rand(n, device="cuda", generator=g) < case["outside"]] = -1  # padding
    index = index.to(torch.int32 if case["index"] == "i32" else torch.int64)
    s = dict(case=case, index=index, scale=math.sqrt(c))
    if case["kind"] == "look":
        shape = (c, t) if case["layout"] == "columns" else (t, c)
        s["table"] = torch.randn(shape, device="cuda", generator=g).to(dt)
    elif case["kind"] == "grad":
        shape = (c, n) if case["layout"] == "columns" else (n, c)
        s["grad"] = torch.randn(shape, device="cuda", generator=g).to(dt)
        if own:
            from trips_amd.lookup import lookup_plan
            s["plan"] = lookup_plan(index, t) if case["kept"] else None
    return s


def prepare(case, seed):
    return _prepare_optimiser(case, seed) if case["kind"] in ("adamw", "norm") else _prepare_table(case, seed)


# ---- plain forms ----

def _norm_and_factor(grads, clip):
    norm = grads.double().square().sum().sqrt()
    factor = (clip / (norm + 1e-6)).clamp(max=1.0) if clip > 0 else torch.ones_like(norm)
    factor = torch.where(torch.isfinite(norm), factor, torch.full_like(norm, math.nan))
    return torch.stack([norm, factor]).float()


def _mix(x):
    """32 well-mixed bits of 32 (held in int64)."""
    x = x ^ (x >> 16)
    x = (x * 0x9E3779B9) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0xB504F333) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _round_to_8bit(y, u, mantissa, low, top):
    """|y| on the grid of an 8-bit float with so many mantissa bits, lowest exponent and largest value: up where the
    part below the grid and u together reach one step."""
    exponent = torch.frexp(y)[1] - 1
    step = torch.exp2((exponent.clamp(min=low) - mantissa).double())
    return ((y / step + u).floor() * step).clamp(max=top)


def _scale_exponent(top_of_block, top):
    """Smallest k with top_of_block <= top 2^k."""
    k = torch.frexp(top_of_block / top)
    k = torch.where(k[0] == 0.5, k[1] - 1, k[1])
    return torch.where(top_of_block > 0, k, torch.full_like(k, -118)).clamp(-118, 111)


def _adamw_plain(s):
    case, (b1, b2) = s["case"], BETAS
    both = _norm_and_factor(s["grads"], case["clip"]) if case["clip"] > 0 else None
    s["steps"] += 1
    t = s["steps"][0].double()
    rate, root = LR / (1 - b1 ** t), (1 - b2 ** t).sqrt()
    if case["bits"] == 32:
        g = s["grads"].float()
        if both is not None:
            g = g * both[1]
        m, v = s["m"], s["v"]
        m.mul_(b1).add_(g * (1 - b1))
        v.mul_(b2).add_(g * g * (1 - b2))
        new = s["w"].float() * (1 - LR * DECAY) - rate.float() * m / (v.sqrt() / root.float() + EPS)
    else:
        g = s["grads"].double()
        if both is not None:
            g = g * both[1].double()
        place = s.get("place")
        blocks = s["ms"].shape[0]

        def spread(x):  # a value of each block to the block's elements
            x = x.double().repeat_interleave(BLOCK)
            return x if place is None else x[place]

        def highest(x):
            if place is None:
                return x.view(blocks, BLOCK).amax(1)
            wide = torch.zeros(blocks * BLOCK, dtype=x.dtype, device=x.device)
            wide[place] = x
            return wide.view(blocks, BLOCK).amax(1)

        m = s["m"].double() * spread(s["ms"]) * b1 + g * (1 - b1)
        v = s["v"].double() * spread(s["vs"]) * b2 + g * g * (1 - b2)
        new = s["w"].double() * (1 - LR * DECAY) - rate * m / (v.sqrt() / root + EPS)
        at = torch.arange(blocks * BLOCK, device=g.device) if place is None else place
        bits = _mix(at ^ _mix((SEED + s["steps"][0].to(torch.int64) * 0x9E3779B9) & 0xFFFFFFFF))
        km, kv = _scale_exponent(highest(m.abs()), 448.0), _scale_exponent(highest(v), 57344.0)
        y = _round_to_8bit(m.abs() * torch.exp2(-spread(km)), ((bits & 0xFFFF).double() + 0.5) / 65536, 3, -6, 448.0)
        s["m"].copy_(torch.copysign(y, m).float())
        y = _round_to_8bit(v * torch.exp2(-spread(kv)), ((bits >> 16).double() + 0.5) / 65536, 2, -14, 57344.0)
        s["v"].copy_(torch.where(v > 0, y.clamp(min=2.0 ** -16), y).float())
        s["ms"].copy_(torch.exp2(km.float()))
        s["vs"].copy_(torch.exp2(kv.float()))
    s["w"].copy_(new)
    if "copy" in s:
        s["copy"].copy_(new)
    return _adamw_outputs(s, both)


def _adamw_outputs(s, both):
    got = {k: s[k] for k in ("w", "copy", "m", "v", "ms", "vs", "steps") if k in s}
    if both is not None:
        got["norm"] = both
    return got


def _look_plain(s):
    rows = s["case"]["layout"] == "rows"
    index = s["index"].long()
    inside = (index >= 0) & (index < s["case"]["texels"])
    index = torch.where(inside, index, torch.zeros_like(index))
    if rows:
        out = s["table"][index].float() * s["scale"] * inside[:, None]
    else:
        out = s["table"][:, index].float() * s["scale"] * inside
    return out.to(s["table"].dtype)


def _grad_plain(s):
    rows, t = s["case"]["layout"] == "rows", s["case"]["texels"]
    index = s["index"].long()
    inside = (index >= 0) & (index < t)
    index = torch.where(inside, index, torch.full_like(index, t))  # one entry more, for what is outside
    g = s["grad"].float()
    if rows:
        total = torch.zeros(t + 1, g.shape[1], device=g.device).index_add_(0, index, g)[:t]
    else:
        total = torch.zeros(g.shape[0], t + 1, device=g.device).index_add_(1, index, g)[:, :t]
    return (total * s["scale"]).to(s["grad"].dtype)


def _plan_plain(s):
    t = s["case"]["texels"]
    index = s["index"].long()
    key = torch.where((index >= 0) & (index < t), index, torch.full_like(index, t))
    key, order = torch.sort(key, stable=True)
    starts = torch.searchsorted(key, torch.arange(t + 1, device=key.device))
    return dict(order=order.to(torch.int32), starts=starts.to(torch.int32))


def _run_own(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "adamw":
        s["opt"].step(grads=s["handed"])
        return _adamw_outputs(s, s["opt"].grad_norm if case["clip"] > 0 else None)
    if kind == "norm":
        from trips_amd.adamw import grad_norm
        return grad_norm(s["list"], max_norm=case["clip"])
    from trips_amd import lookup as table
    layout = table.ROWS if case["layout"] == "rows" else table.COLUMNS
    if kind == "look":
        return table.lookup(s["table"], s["index"], scale=s["scale"], layout=layout)
    if kind == "grad":
        return table.lookup_backward(s["grad"], s["index"], case["texels"], scale=s["scale"], layout=layout, plan=s["plan"])
    plan = table.lookup_plan(s["index"], case["texels"])
    return dict(order=plan.order, starts=plan.starts)


def run(state):
    if own:
        return _run_own(state)
    kind = state["case"]["kind"]
    if kind == "norm":
        return _norm_and_factor(state["grads"], state["case"]["clip"])
    return dict(adamw=_adamw_plain, look=_look_plain, grad=_grad_plain, plan=_plan_plain)[kind](state)


def work(case):
    kind = case["kind"]
    if kind in ("adamw", "norm"):
        n = sum(tensor_sizes(case["sizes"]))
        if kind == "norm":
            return dict(bytes=n * BYTES[case["grads"]] + 8, flops=2 * n)
        blocks = sum(-(-k // BLOCK) for k in tensor_sizes(case["sizes"]))
        moments = 16 * n if case["bits"] == 32 else 4 * n + 16 * blocks
        # (a step that is clipped reads the gradients twice: the factor depends on all of them)
        grads = n * BYTES[case["grads"]] * (2 if case["clip"] > 0 else 1)
        return dict(bytes=n * (2 * BYTES[case["weights"]] + BYTES[case["copy"]]) + grads + moments, flops=14 * n)
    n, t, c, size = case["points"], case["texels"], case["channels"], BYTES[case["dtype"]]
    index = n * (4 if case["index"] == "i32" else 8)
    if kind == "plan":
        return dict(bytes=index + 4 * n + 4 * (t + 1), flops=n)
    if kind == "look":
        return dict(bytes=index + (min(n, t) + n) * c * size, flops=n * c)
    return dict(bytes=(4 * (n + t + 1) if case["kept"] else index) + (n + t) * c * size, flops=n * c)


# ---- the definitions in 64 bits ----

def _exact_8bit(y, u, dtype):
    """y >= 0 between its two neighbours among the values of an 8-bit float type."""
    every = torch.arange(256, dtype=torch.uint8, device=y.device).view(dtype).double()
    values = torch.unique(every[torch.isfinite(every) & (every >= 0)])
    low = (torch.searchsorted(values, y, right=True) - 1).clamp(0, values.numel() - 1)
    high = (low + 1).clamp(max=values.numel() - 1)
    part = (y - values[low]) / torch.where(high > low, values[high] - values[low], torch.ones_like(y))
    return torch.where(part.clamp(max=1.0) + u >= 1, values[high], values[low])


def _exact_adamw(s):
    case, got = s["case"], {}
    (b1, b2), t = BETAS, int(s["steps"][0]) + 1
    g, w = s["grads"].double(), s["w"].double()
    factor = 1.0
    if case["clip"] > 0:
        norm = math.sqrt(float((g ** 2).sum()))
        factor = min(1.0, case["clip"] / (norm + 1e-6))
        got["norm"] = torch.tensor([norm, factor], dtype=torch.float64)
        factor = float(torch.tensor(factor, dtype=torch.float32)) if case["bits"] == 8 else factor
    g = g * factor
    m, v = s["m"].double(), s["v"].double()
    wide, blocks = None, 0
    if case["bits"] == 8:
        blocks = s["ms"].numel()
        at, _ = _offsets(s["sizes"], False)
        wide = torch.cat([torch.arange(n, device=g.device) + o for n, o in zip(s["sizes"], at)]) if case["packed"] \
            else torch.arange(g.numel(), device=g.device)
        block_of = torch.div(wide, BLOCK, rounding_mode="floor")
        m, v = m * s["ms"].double()[block_of], v * s["vs"].double()[block_of]
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g ** 2
    ahead, spread = m / (1 - b1 ** t), torch.sqrt(v / (1 - b2 ** t))
    w = w - LR * DECAY * w - LR * ahead / (spread + EPS)
    got.update(w=w, steps=None)
    if "copy" in s:
        got["copy"] = w
    if case["bits"] == 32:
        got.update(m=m, v=v)
        return got
    word = ((SEED + t * 0x9E3779B9) & 0xFFFFFFFF)
    for shift, factor_ in ((16, 0x9E3779B9), (15, 0xB504F333)):
        word = ((word ^ (word >> shift)) * factor_) & 0xFFFFFFFF
    bits = wide ^ (word ^ (word >> 16))
    for shift, factor_ in ((16, 0x9E3779B9), (15, 0xB504F333)):
        bits = ((bits ^ (bits >> shift)) * factor_) & 0xFFFFFFFF
    bits = bits ^ (bits >> 16)
    for x, part, dtype, name, scale in ((m, bits % 65536, torch.float8_e4m3fn, "m", "ms"), (v, bits // 65536, torch.float8_e5m2, "v", "vs")):
        most = torch.finfo(dtype).max
        high = torch.zeros(blocks, dtype=torch.float64, device=x.device).scatter_reduce_(0, block_of, x.abs(), "amax")
        k = torch.ceil(torch.log2(high.clamp(min=1e-300) / most))
        k = torch.where(high > most * 2.0 ** k, k + 1, torch.where(high <= most * 2.0 ** (k - 1), k - 1, k)).clamp(-118, 111)
        y = _exact_8bit(x.abs() / 2.0 ** k[block_of], (part.double() + 0.5) / 65536, dtype)
        if name == "v":
            y = torch.where((x > 0) & (y == 0), torch.full_like(y, 2.0 ** -16), y)
        got[name], got[scale] = y * torch.sign(x), 2.0 ** k
    return got


def exact(case, seed):
    kind = case["kind"]
    if kind == "plan":
        return None  # whole numbers
    s = _prepare_optimiser(case, seed) if kind in ("adamw", "norm") else _prepare_table(case, seed)
    if kind == "adamw":
        return _exact_adamw(s)
    if kind == "norm":
        norm = math.sqrt(float((s["grads"].double() ** 2).sum()))
        return torch.tensor([norm, min(1.0, case["clip"] / (norm + 1e-6))], dtype=torch.float64)
    t, index = case["texels"], s["index"].long()
    valid = ((index >= 0) & (index < t)).nonzero()[:, 0]
    dim = 0 if case["layout"] == "rows" else 1
    if kind == "look":
        n = index.numel()
        shape = (n, case["channels"]) if dim == 0 else (case["channels"], n)
        out = torch.zeros(shape, dtype=torch.float64, device=index.device)
        return out.index_copy_(dim, valid, torch.index_select(s["table"], dim, index[valid]).double() * s["scale"])
    g = torch.index_select(s["grad"], dim, valid).double() * s["scale"]
    shape = (t, case["channels"]) if dim == 0 else (case["channels"], t)
    return torch.zeros(shape, dtype=torch.float64, device=index.device).index_add_(dim, index[valid], g)
