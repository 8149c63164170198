"""A table's softmax cross entropy and dropout as users call them, as cases that can be timed and compared with their plain forms.

A case is a dict of plain values; its "kind" says which operator a pass goes through:

  score    table_cross_entropy() without gradients: what each row loses on its target among all entries of a table
  train    the same with the gradients of the rows and of the table
  drop     dropout() without gradients, with a residual that it is added to or without
  regrad   dropout() with the gradient of what went in

Dropout's words come from Philox-4x32-10: the key is the seed, the counter the number of the block of eight elements, the call
and the step; each of the four words holds the 16 bits of two elements, the lower half first. An element is dropped where its
16 bits are below round(65536 p).
"""
import math

import torch

own = False

SEED = 0x1234_5678_9ABC_DEF0
DTYPES = dict(f32=torch.float32, bf16=torch.bfloat16, f16=torch.float16)
BYTES = dict(f32=4, bf16=2, f16=2)


def _loss(kind, *, tokens, entries, channels, dtype="bf16", reduction="mean", scale=1.0, padding=0.0, index="i64"):
    return dict(kind=kind, tokens=tokens, entries=entries, channels=channels, dtype=dtype, reduction=reduction, scale=scale,
                padding=padding, index=index)


def _drop(kind, *, rows, channels, dtype="bf16", p=0.1, residual=False):
    return dict(kind=kind, rows=rows, channels=channels, dtype=dtype, p=p, residual=residual)


def listed():
    return [
        # one token of an answer, scored against all embeddings: the table is read once
        dict(name="score_1_token", **_loss("score", tokens=1, entries=50_000, channels=1024, reduction="none")),
        # a prompt whose tokens are scored
        dict(name="score_2047_tokens", **_loss("score", tokens=2047, entries=50_000, channels=1024, reduction="none")),
        # 20k points of 16 channels among 150 labels
        dict(name="score_20k_points_f32", **_loss("score", tokens=20_000, entries=150, channels=16, dtype="f32", index="i32")),
        # a batch of 8191 tokens, some of it padding: the embeddings' other end
        dict(name="train_tokens_bf16", **_loss("train", tokens=8191, entries=50_000, channels=1024, padding=0.05)),
        # few tokens of a large table with wide rows
        dict(name="train_large_table_bf16", **_loss("train", tokens=2048, entries=250_007, channels=2048)),
        # half precision, weights of the tokens' losses given
        dict(name="train_weighted_f16", **_loss("train", tokens=3000, entries=32_000, channels=768, dtype="f16",
                                                reduction="none", scale=0.7)),
        # single precision, a smaller table
        dict(name="train_f32", **_loss("train", tokens=1023, entries=20_000, channels=384, dtype="f32", index="i32")),
        # a few points: launches and host time
        dict(name="train_25_rows_f32", **_loss("train", tokens=25, entries=5000, channels=64, dtype="f32", index="i32")),
        # 32 rows of an answer's batch
        dict(name="drop_32_rows", **_drop("drop", rows=32, channels=1024)),
        # a block's output added to what runs past it
        dict(name="drop_tokens_residual", **_drop("drop", rows=8191, channels=1024, residual=True)),
        # descriptors of the benchmark's 6M points, forward and backward
        dict(name="regrad_6M_points_f32", **_drop("regrad", rows=6_000_000, channels=4, dtype="f32", p=0.25)),
        # a wide layer of the batch, an odd number of elements in a row
        dict(name="regrad_wide_bf16", **_drop("regrad", rows=8191, channels=4097, residual=True)),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("score", "train", "train", "drop", "regrad"))
    dtype = rng.choice(("f32", "bf16", "bf16", "f16"))
    if kind in ("drop", "regrad"):
        channels = _log_int(rng, 1, 8192)
        return _drop(kind, rows=_log_int(rng, 1, max(1, min(6_000_000, 30_000_000 // channels))), channels=channels, dtype=dtype,
                     p=rng.choice((0.0, 0.05, 0.1, 0.25, 0.5, 0.9)), residual=rng.random() < 0.5)
    most = 1e12 if dtype != "f32" else 2e10
    tokens, entries = _log_int(rng, 1, 16_384), _log_int(rng, 2, 262_144)
    entries = min(entries, 500_000_000 // tokens)
    channels = min(_log_int(rng, 4, 4096), max(4, int(most / tokens / entries)))
    if rng.random() < 0.5:
        channels = -(-channels // 8) * 8
    return _loss(kind, tokens=tokens, entries=entries, channels=channels, dtype=dtype, reduction=rng.choice(("none", "sum", "mean")),
                 scale=rng.choice((1.0, 1.0, 0.7)), padding=rng.choice((0.0, 0.0, 0.1, 0.5)), index=rng.choice(("i32", "i64")))


# ---- inputs ----

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _prepare_loss(case, seed):
    g = _generator(seed)
    n, t, c, dt = case["tokens"], case["entries"], case["channels"], DTYPES[case["dtype"]]
    # frequent entries first; logits some units wide, a row's own entry ahead of most, as a trained model has them
    target = (torch.rand(n, device="cuda", generator=g, dtype=torch.float64).pow_(3.0) * t).to(torch.int64).clamp_(0, t - 1)
    table = torch.randn(t, c, device="cuda", generator=g).mul_(2.0 / math.sqrt(c))
    rows = torch.randn(n, c, device="cuda", generator=g).add_(table[target], alpha=1.5)
    if case["padding"] > 0:
        target[torch.rand(n, device="cuda", generator=g) < case["padding"]] = -1
    s = dict(case=case, rows=rows.to(dt), table=table.to(dt), target=target.to(torch.int32 if case["index"] == "i32" else torch.int64))
    if case["kind"] == "train":
        shape = (n,) if case["reduction"] == "none" else ()
        s["grad"] = torch.rand(shape, device="cuda", generator=g) + 0.5  # what follows the loss: weights of the tokens, a factor
        if own:
            s["rows"].requires_grad_()
            s["table"].requires_grad_()
    return s


def _prepare_drop(case, seed):
    g = _generator(seed)
    shape, dt = (case["rows"], case["channels"]), DTYPES[case["dtype"]]
    s = dict(case=case, call=seed % 1000, step=torch.full((), 100 + seed % 50, device="cuda", dtype=torch.int32))
    s["x"] = torch.randn(shape, device="cuda", generator=g).to(dt)
    s["residual"] = torch.randn(shape, device="cuda", generator=g).to(dt) if case["residual"] else None
    if case["kind"] == "regrad":
        s["grad"] = torch.randn(shape, device="cuda", generator=g).to(dt)
        if own:
            s["x"].requires_grad_()
    return s


def prepare(case, seed):
    return _prepare_drop(case, seed) if case["kind"] in ("drop", "regrad") else _prepare_loss(case, seed)


# ---- plain forms ----

def _loss_plain(s):
    case = s["case"]
    x, w, target = s["rows"].float(), s["table"].float(), s["target"].long()
    inside = (target >= 0) & (target < case["entries"])
    own_entry = torch.where(inside, target, torch.zeros_like(target))[:, None]
    logits = (x @ w.t()).mul_(case["scale"])
    top = logits.amax(1, keepdim=True)
    own_logit = logits.gather(1, own_entry)
    e = logits.sub_(top).exp_()
    total = e.sum(1, keepdim=True)
    losses = torch.where(inside, (top + total.log() - own_logit)[:, 0], torch.zeros_like(top[:, 0]))
    count = inside.sum().clamp(min=1)
    loss = losses if case["reduction"] == "none" else losses.sum() if case["reduction"] == "sum" else losses.sum() / count
    if case["kind"] == "score":
        return loss
    g = s["grad"] / count if case["reduction"] == "mean" else s["grad"]
    d = e.div_(total)
    d.scatter_add_(1, own_entry, torch.full_like(own_logit, -1.0))
    d.mul_((torch.where(inside, g, torch.zeros_like(losses)) * case["scale"])[:, None])
    dt = s["rows"].dtype
    return dict(loss=loss, d_rows=(d @ w).to(dt), d_table=(d.t() @ x).to(dt))


def _product(a, b):
    """The two 32-bit halves (high, low) of a * b, for a of 32 bits held in int64 and a number b of 32 bits."""
    low, high = (a & 0xFFFF) * b, (a >> 16) * b
    low = low + ((high & 0xFFFF) << 16)
    return (high >> 16) + (low >> 32), low & 0xFFFFFFFF


def _words(n, call, step, device):
    """16 bits for each of n elements."""
    block = torch.arange(-(-n // 8), device=device, dtype=torch.int64)
    c = [block & 0xFFFFFFFF, block >> 32, torch.full_like(block, call), step.to(torch.int64).expand(block.shape) & 0xFFFFFFFF]
    k0, k1 = SEED & 0xFFFFFFFF, SEED >> 32
    for _ in range(10):
        h0, l0 = _product(c[0], 0xD2511F53)
        h1, l1 = _product(c[2], 0xCD9E8D57)
        c = [h1 ^ c[1] ^ k0, l1, h0 ^ c[3] ^ k1, l0]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return torch.stack([half for word in c for half in (word & 0xFFFF, word >> 16)], 1).reshape(-1)[:n]


def _drop_plain(s):
    case = s["case"]
    border = round(65536 * case["p"])
    keep = (_words(s["x"].numel(), s["call"], s["step"], s["x"].device) >= border).view(s["x"].shape)
    factor = 65536 / (65536 - border)

    def through(t):
        t = t.float() * factor
        return torch.where(keep, t, torch.zeros_like(t))
    out = through(s["x"])
    if case["residual"]:
        out = out + s["residual"].float()
    out = out.to(s["x"].dtype)
    if case["kind"] == "drop":
        return out
    return dict(out=out, d_x=through(s["grad"]).to(s["x"].dtype))


def _run_own(s):
    case = s["case"]
    if case["kind"] in ("score", "train"):
        from trips_amd.table_loss import table_cross_entropy
        loss = table_cross_entropy(s["rows"], s["table"], s["target"], scale=case["scale"], reduction=case["reduction"])
        if case["kind"] == "score":
            return loss
        d_rows, d_table = torch.autograd.grad(loss, (s["rows"], s["table"]), s["grad"])
        return dict(loss=loss.detach(), d_rows=d_rows, d_table=d_table)
    from trips_amd.dropout import dropout
    out = dropout(s["x"], case["p"], SEED, call=s["call"], step=s["step"], residual=s["residual"])
    if case["kind"] == "drop":
        return out
    d_x, = torch.autograd.grad(out, (s["x"],), s["grad"])
    return dict(out=out.detach(), d_x=d_x)


def run(state):
    if own:
        return _run_own(state)
    return (_drop_plain if state["case"]["kind"] in ("drop", "regrad") else _loss_plain)(state)


def work(case):
    size = BYTES[case["dtype"]]
    if case["kind"] in ("drop", "regrad"):
        n = case["rows"] * case["channels"]
        tensors = 2 + case["residual"] + (2 if case["kind"] == "regrad" else 0)
        return dict(bytes=tensors * n * size, flops=(2 if case["kind"] == "regrad" else 1) * n)
    n, t, c = case["tokens"], case["entries"], case["channels"]
    counted = max(1, round(n * (1 - case["padding"])))
    losses = 4 * (n if case["reduction"] == "none" else 1)
    bytes_ = n * (4 if case["index"] == "i32" else 8) + losses + (counted + t) * c * size
    if case["kind"] == "score":
        return dict(bytes=bytes_, flops=2 * counted * t * c)
    # (the logits, the product with the table and the product with the rows)
    return dict(bytes=bytes_ + losses + (n + t) * c * size, flops=6 * counted * t * c)


# ---- the definitions in 64 bits ----

def _exact_loss(case, seed):
    s = _prepare_loss(case, seed)
    n, t, c = case["tokens"], case["entries"], case["channels"]
    x, w, target = s["rows"].detach().double(), s["table"].detach().double(), s["target"].long()
    counted = ((target >= 0) & (target < t)).nonzero()[:, 0]
    losses = torch.zeros(n, dtype=torch.float64, device=x.device)
    train = case["kind"] == "train"
    d_rows, d_table = torch.zeros_like(x), torch.zeros_like(w) if train else None
    if train:
        g = s["grad"].double().expand(n) / (max(1, counted.numel()) if case["reduction"] == "mean" else 1)
    for part in counted.split(max(1, 200_000_000 // t)):
        logits = case["scale"] * (x[part] @ w.t())
        logp = torch.log_softmax(logits, 1)
        at = torch.arange(part.numel(), device=x.device)
        losses[part] = -logp[at, target[part]]
        if train:
            d = logp.exp_()
            d[at, target[part]] -= 1
            d *= (case["scale"] * g[part])[:, None]
            d_rows[part] = d @ w
            d_table += d.t() @ x[part]
    loss = losses if case["reduction"] == "none" else losses.sum()
    if case["reduction"] == "mean":
        loss = loss / max(1, counted.numel())
    return dict(loss=loss, d_rows=d_rows, d_table=d_table) if train else loss


def _exact_drop(case, seed):
    s = _prepare_drop(case, seed)
    border, n = round(65536 * case["p"]), s["x"].numel()
    # the generator again, with products of 64 bits that wrap around
    m0, m1 = 0xD2511F53, 0xCD9E8D57
    a = torch.arange((n + 7) // 8, device="cuda", dtype=torch.int64)
    b, mask = a >> 32, 0xFFFFFFFF
    a, c, d = a & mask, torch.full_like(a, s["call"]), torch.full_like(a, int(s["step"]))
    for r in range(10):
        k0, k1 = (SEED + r * 0x9E3779B9) & mask, ((SEED >> 32) + r * 0xBB67AE85) & mask
        p, q = a * m0, c * m1
        a, b, c, d = ((q >> 32) & mask) ^ b ^ k0, q & mask, ((p >> 32) & mask) ^ d ^ k1, p & mask
    words = torch.empty(a.numel(), 8, dtype=torch.int64, device="cuda")
    for i, v in enumerate((a, b, c, d)):
        words[:, 2 * i], words[:, 2 * i + 1] = v % 65536, v // 65536
    kept = (words.reshape(-1)[:n] >= border).view(s["x"].shape).double() * (65536.0 / (65536 - border))
    out = s["x"].detach().double() * kept
    if case["residual"]:
        out = out + s["residual"].double()
    return dict(out=out, d_x=s["grad"].double() * kept) if case["kind"] == "regrad" else out


def exact(case, seed):
    return _exact_drop(case, seed) if case["kind"] in ("drop", "regrad") else _exact_loss(case, seed)
