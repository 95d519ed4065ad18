"""Cases of the language-model products: linear_cross_entropy and matrix_mul_w4.

Two operators stand next to matrix_mul:

* ``linear_cross_entropy``: the output projection of a language model fused with its loss,
  softmax cross entropy over the vocabulary, and the loss's gradients by the hidden states
  and by the projection's weight.  The [tokens, vocabulary] logits are never kept.
* ``matrix_mul_w4``: x @ W.T with W held as 4-bit codes with one scale (and, if asked, one
  zero point) per group of consecutive inputs: W[n, k] = (code[n, k] - zero) * scale.

``run`` computes either one in plain torch operations in 32 bits (own = False) or through
this package's entry points (own = True).
"""
import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
IGNORE = -100

# Largest listed costs, which drawn cases stay below.
MAX_CE = 8192 * 131072 * 4096
MAX_W4 = 2048 * 8192 * 8192
MAX_W4_WEIGHT = 28672 * 8192


def _ce(name, tokens, vocab, dim, dtype, ignored, reduction, grad):
    c = {"op": "ce", "tokens": tokens, "vocab": vocab, "dim": dim, "dtype": dtype, "ignored": ignored,
         "reduction": reduction, "grad": grad}
    return {"name": name, **c} if name else c


def _w4(name, rows, n, k, group, dtype, zeros, bias):
    c = {"op": "w4", "rows": rows, "n": n, "k": k, "group": group, "dtype": dtype, "zeros": zeros, "bias": bias}
    return {"name": name, **c} if name else c


def listed():
    return [
        # A few candidate tokens scored under a small model: latency and one read of the weight.
        _ce("ce_score_16", 16, 32000, 1024, "bf16", 0.0, "none", False),
        # Evaluation of a text, token by token: the forward pass alone.
        _ce("ce_score_4096", 4096, 65536, 2048, "bf16", 0.0, "none", False),
        # A training micro-batch of a small model, with some padding.
        _ce("ce_train_512", 512, 32000, 1024, "bf16", 0.1, "mean", True),
        # Odd sizes in every direction: rows that are not 16-byte aligned, ragged tiles.
        _ce("ce_train_ragged_f16", 1001, 30011, 777, "f16", 0.1, "mean", True),
        # Fine-tuning on answers only: most tokens are prompt and have no target.
        _ce("ce_train_masked", 4096, 50000, 2048, "bf16", 0.6, "sum", True),
        # float32 training, the type of the package's other products.
        _ce("ce_train_f32", 2048, 32000, 1024, "f32", 0.1, "mean", True),
        # Pretraining of a large model: one long sequence, a large vocabulary.
        _ce("ce_train_8192", 8192, 131072, 4096, "bf16", 0.05, "mean", True),
        # Decoding one token: an attention projection and the widest feed-forward product.
        _w4("w4_1_square", 1, 4096, 4096, 128, "bf16", False, False),
        _w4("w4_1_wide", 1, 28672, 8192, 128, "bf16", True, False),
        # Decoding a batch of sequences.
        _w4("w4_8", 8, 8192, 8192, 64, "f16", True, True),
        # The package's odd product (1000 x 3001 x 777) with its weight in 4 bits, float32 activations.
        _w4("w4_ragged_f32", 5, 777, 3001, 32, "f32", True, True),
        # A prompt: the same weights with many rows at once.
        _w4("w4_prompt", 2048, 8192, 8192, 128, "bf16", True, False),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    if rng.random() < 0.5:
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        tokens, vocab, dim = _log(rng, 1, 8192), _log(rng, 1000, 131072), _log(rng, 64, 4096)
        if rng.random() < 0.5:  # weights come with aligned rows as often as not
            vocab, dim = (vocab + 63) // 64 * 64, (dim + 63) // 64 * 64
        return _ce(None, tokens, vocab, dim, dtype, rng.choice([0.0, 0.1, 0.5, 0.9]),
                   rng.choice(["mean", "sum", "none"]), rng.random() < 0.7)
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    n, k = _log(rng, 64, 28672), _log(rng, 64, 28672)
    if rng.random() < 0.5:
        n, k = (n + 63) // 64 * 64, (k + 127) // 128 * 128
    if n * k > MAX_W4_WEIGHT:
        n = MAX_W4_WEIGHT // k
    rows = _log(rng, 1, 64) if rng.random() < 0.6 else _log(rng, 64, 4096)
    rows = max(1, min(rows, MAX_W4 // (n * k)))
    return _w4(None, rows, n, k, rng.choice([32, 64, 128]), dtype, rng.random() < 0.5, rng.random() < 0.3)


def _ce_inputs(case, seed):
    """Hidden states of unit scale that lean towards their target's row, as in a model that
    has learnt something (the target's logit stands out of the others' spread of about 1);
    targets are more often low indices (frequent tokens); some have no target."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    t, v, d = case["tokens"], case["vocab"], case["dim"]
    dt = DTYPES[case["dtype"]]
    w = torch.randn(v, d, device=DEV, generator=g, dtype=torch.float32).mul_(d ** -0.5)
    target = (torch.rand(t, device=DEV, generator=g).pow(2) * v).long().clamp_(max=v - 1)
    lean = 4.0 * torch.rand(t, 1, device=DEV, generator=g)
    x = (torch.randn(t, d, device=DEV, generator=g) + lean * w[target]).to(dt)
    w = w.to(dt)
    if case["ignored"] > 0:
        skip = torch.rand(t, device=DEV, generator=g) < case["ignored"]
        skip[0] = False  # a batch has a target
        target[skip] = IGNORE
    go = torch.rand(t, device=DEV, generator=g) + 0.5 if case["reduction"] == "none" else None
    return x, w, target, go


def _w4_inputs(case, seed):
    """Codes, scales and zero points as a quantiser leaves them: codes around the middle of
    the range, zero points near 8, scales that bring the weights to about k ** -0.5."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    m, n, k = case["rows"], case["n"], case["k"]
    dt = DTYPES[case["dtype"]]
    groups = -(-k // case["group"])
    codes = (torch.randn(n, k, device=DEV, generator=g) * 3 + 8).round_().clamp_(0, 15).to(torch.uint8)
    scales = ((torch.rand(n, groups, device=DEV, generator=g) + 0.5) * (k ** -0.5 / 3)).to(dt)
    zeros = None
    if case["zeros"]:
        zeros = torch.randint(6, 11, (n, groups), device=DEV, generator=g, dtype=torch.uint8)
    x = torch.randn(m, k, device=DEV, generator=g).to(dt)
    bias = torch.randn(n, device=DEV, generator=g).to(dt) if case["bias"] else None
    return x, codes, scales, zeros, bias


def prepare(case, seed):
    if case["op"] == "ce":
        x, w, target, go = _ce_inputs(case, seed)
        if case["grad"]:
            x.requires_grad_(True)
            w.requires_grad_(True)
        return {"case": case, "x": x, "w": w, "target": target, "go": go}
    x, codes, scales, zeros, bias = _w4_inputs(case, seed)
    state = {"case": case, "x": x, "bias": bias}
    if own:
        from tilec_b200 import ext
        state["weight"] = ext.pack_w4(codes, scales, zeros, group_size=case["group"])
    else:
        if case["k"] % 2:
            codes = torch.nn.functional.pad(codes, (0, 1))
        state["packed"] = codes[:, 0::2] | codes[:, 1::2] << 4  # two codes a byte, the even one low
        state["scales"], state["zeros"] = scales, zeros
    return state


def _run_ce_own(s):
    from tilec_b200 import ext
    loss = ext.linear_cross_entropy(s["x"], s["w"], s["target"], ignore_index=IGNORE,
                                    reduction=s["case"]["reduction"])
    if not s["case"]["grad"]:
        return loss
    return (loss.detach(), *torch.autograd.grad(loss, (s["x"], s["w"]), s["go"]))


def _run_ce_plain(s):
    x, w, target, go = s["x"].detach().float(), s["w"].detach().float(), s["target"], s["go"]
    reduction = s["case"]["reduction"]
    valid = target != IGNORE
    idx = torch.where(valid, target, 0)
    logits = x @ w.t()
    top = logits.amax(1, keepdim=True)
    e = torch.exp(logits - top)
    z = e.sum(1, keepdim=True)
    loss = torch.log(z[:, 0]) + top[:, 0] - logits.gather(1, idx[:, None])[:, 0]
    loss = torch.where(valid, loss, 0.0)
    count = valid.sum()
    if reduction == "sum":
        loss = loss.sum()
    elif reduction == "mean":
        loss = (loss.double().sum() / count).float()
    if not s["case"]["grad"]:
        return loss
    r = valid.float() if go is None else valid * go
    if reduction == "mean":
        r = r / count
    p = e.div_(z)
    p[torch.arange(len(idx), device=p.device), idx] -= 1
    p *= r[:, None]
    return loss, (p @ w).to(s["x"].dtype), (p.t() @ x).to(s["w"].dtype)


def _run_w4_own(s):
    from tilec_b200 import ext
    return ext.matrix_mul_w4(s["x"], s["weight"], bias=s["bias"])


def _run_w4_plain(s):
    case, x, packed = s["case"], s["x"], s["packed"]
    n, k, group = case["n"], case["k"], case["group"]
    codes = torch.stack((packed & 15, packed >> 4), 2).view(n, -1)[:, :k].float()
    scales = s["scales"].float().repeat_interleave(group, 1)[:, :k]
    zeros = 8.0 if s["zeros"] is None else s["zeros"].float().repeat_interleave(group, 1)[:, :k]
    y = x.float() @ ((codes - zeros) * scales).t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(x.dtype)


def run(state):
    if state["case"]["op"] == "ce":
        return _run_ce_own(state) if own else _run_ce_plain(state)
    return _run_w4_own(state) if own else _run_w4_plain(state)


def work(case):
    b = SIZE[case["dtype"]]
    if case["op"] == "ce":
        t, v, d = case["tokens"], case["vocab"], case["dim"]
        live = t * (1.0 - case["ignored"])  # tokens with a target
        bytes_ = (live * d + v * d) * b + t * 8
        if not case["grad"]:
            return {"bytes": bytes_ + (t if case["reduction"] == "none" else 1) * 4, "flops": 2.0 * live * v * d}
        return {"bytes": bytes_ + (t * d + v * d) * b + 4, "flops": 6.0 * live * v * d}
    m, n, k = case["rows"], case["n"], case["k"]
    groups = -(-k // case["group"])
    bytes_ = n * k / 2 + n * groups * (b + (0.5 if case["zeros"] else 0)) + (m * k + m * n) * b
    return {"bytes": bytes_ + (n * b if case["bias"] else 0), "flops": 2.0 * m * n * k}


def _exact_ce(case, seed):
    """By the definition, a block of tokens at a time: loss_t = log sum_v exp(x_t.w_v) - x_t.w_y,
    d loss_t / d logit_v = softmax_v - [v = y]."""
    x, w, target, go = _ce_inputs(case, seed)
    x64, w64 = x.double(), w.double()
    t = case["tokens"]
    live = target.ne(IGNORE)
    weight = torch.ones(t, device=DEV, dtype=torch.float64) if go is None else go.double()
    if case["reduction"] == "mean":
        weight = weight / live.sum().double()
    losses = torch.zeros(t, device=DEV, dtype=torch.float64)
    dx, dw = torch.zeros_like(x64), torch.zeros_like(w64)
    rows = live.nonzero()[:, 0]
    for at in range(0, len(rows), 1024):
        r = rows[at:at + 1024]
        logp = torch.log_softmax(x64[r] @ w64.T, dim=1)
        y = target[r, None]
        losses[r] = -logp.gather(1, y)[:, 0]
        if case["grad"]:
            q = logp.exp_()
            q.scatter_add_(1, y, torch.full_like(y, -1, dtype=torch.float64))
            q.mul_(weight[r, None])
            dx[r] = q @ w64
            dw.addmm_(q.T, x64[r])
    if case["reduction"] != "none":
        losses = losses.sum() / (live.sum() if case["reduction"] == "mean" else 1)
    return (losses, dx, dw) if case["grad"] else losses


def _exact_w4(case, seed):
    x, codes, scales, zeros, bias = _w4_inputs(case, seed)
    n, k, group = case["n"], case["k"], case["group"]
    y = torch.zeros(case["rows"], n, device=DEV, dtype=torch.float64)
    for g in range(scales.shape[1]):  # group by group: scale * (x . code - zero * sum x)
        sl = slice(g * group, min(k, (g + 1) * group))
        xg = x[:, sl].double()
        zero = 8.0 if zeros is None else zeros[:, g].double()
        y += (xg @ codes[:, sl].double().T - xg.sum(1, keepdim=True) * zero) * scales[:, g].double()
    return y if bias is None else y + bias.double()


def exact(case, seed):
    return _exact_ce(case, seed) if case["op"] == "ce" else _exact_w4(case, seed)
