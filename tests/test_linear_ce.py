"""linear_cross_entropy: refusals (CPU) and numerics against the definition in 64 bits (GPU).

Tolerances, u = half a unit in the last place relative to the value (2^-8 bf16, 2^-11 fp16,
2^-24 fp32), of errors measured against the fp64 definition on the same (rounded) inputs:

* logits: fp32 sums of exact products (16-bit types) or of 3xTF32 products (fp32: 3 * 2^-20
  = 2.9e-6 relative per product, random in sign); 2e-6 of ||x|| ||w|| covers either.
* loss: one logit's error e = 1e-5 + 2e-6 max||x|| max||w|| absolute, 1e-5 relative.
* gradients, relative Frobenius error: the logits' gradient is rounded to the dtype (u),
  the sum is rounded once more (u), and the softmax carries the logits' errors (2e): each
  element's error relative to sum |terms|.  The terms' roundings are independent, so the
  Frobenius error stays below 2u * ||terms|| / ||sum||, and the sums here (random signs, no
  cancellation by design) keep that ratio near 1: 2.5u + 2e + 2e-5.
"""
import math

import pytest
import torch

from tilec_b200 import TilecError, ext

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
U = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}
IGNORE = -100


def _make(t, v, d, dtype, seed=0, ignored=0.2, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    w = (torch.randn(v, d, generator=g) * d ** -0.5).to(DT[dtype])
    target = torch.randint(0, v, (t,), generator=g)
    x = (torch.randn(t, d, generator=g) + 2.0 * torch.rand(t, 1, generator=g) * w.float()[target]).to(DT[dtype])
    if ignored:
        target[torch.rand(t, generator=g) < ignored] = IGNORE
        if t:
            target[0] = int(torch.randint(0, v, (1,), generator=g))
    return x.to(device), w.to(device), target.to(device)


def _definition(x, w, target, reduction, ignore=IGNORE, go=None):
    """Loss, dx and dw in 64 bits on the CPU; rows without a target are left out."""
    x, w, target = x.detach().cpu().double(), w.detach().cpu().double(), target.cpu()
    live = (target != ignore).nonzero()[:, 0]
    logits = x[live] @ w.t()
    lse = torch.logsumexp(logits, 1)
    y = target[live]
    loss = torch.zeros(len(target), dtype=torch.float64)
    loss[live] = lse - logits[torch.arange(len(live)), y]
    p = torch.exp(logits - lse[:, None])
    p[torch.arange(len(live)), y] -= 1
    r = torch.ones(len(live), dtype=torch.float64)
    if reduction == "mean":
        r = r / max(len(live), 1)
    if go is not None:
        r = r * (go.cpu().double().reshape(-1)[live] if reduction == "none" else go.cpu().double())
    p = p * r[:, None]
    dx = torch.zeros_like(x)
    dx[live] = p @ w
    dw = p.t() @ x[live]
    if reduction == "sum":
        loss = loss.sum()
    elif reduction == "mean":
        loss = loss.sum() / len(live) if len(live) else torch.tensor(float("nan"))
    return loss, dx, dw


def _rel(a, b):
    a, b = a.detach().cpu().double(), b.double()
    n = b.norm().item()
    return (a - b).norm().item() / n if n else a.norm().item()


def _check(x, w, target, dtype, reduction="mean", go=None, ignore=IGNORE):
    x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss = ext.linear_cross_entropy(x, w, target, ignore_index=ignore, reduction=reduction)
    assert loss.dtype == torch.float32 and loss.shape == (target.shape if reduction == "none" else ())
    if go is None:
        go = torch.ones_like(loss)
    dx, dw = torch.autograd.grad(loss, (x, w), go)
    want, wdx, wdw = _definition(x, w, target, reduction, ignore, go)
    scale = max(1, int((target != ignore).sum())) if reduction == "sum" else 1
    e = 1e-5 + 2e-6 * (x.double().norm(dim=1).max() * w.double().norm(dim=1).max()).item()
    torch.testing.assert_close(loss.detach().cpu().double(), want, rtol=1e-5, atol=e * scale, check_dtype=False)
    tol = 2.5 * U[dtype] + 2 * e + 2e-5
    assert dx.dtype == x.dtype and dw.dtype == w.dtype
    for got, ref in ((dx, wdx), (dw, wdw)):
        assert torch.isfinite(got).all()
        # An fp16 result below 2^-14 is a multiple of 2^-24: it is off by up to 2^-25, whatever
        # its size, and ||errors|| by up to 2^-25 sqrt(elements).
        sub = 2.0 ** -25 * math.sqrt(ref.numel()) / max(ref.norm().item(), 1e-30) if dtype == "f16" else 0.0
        assert _rel(got, ref) <= tol + sub, f"{_rel(got, ref):.3e} > {tol:.3e} + {sub:.3e}"
    assert (dx[target == ignore] == 0).all()
    ext.check_device()


# ---------------------------------------------------------------- refusals (no GPU needed)
def test_refusals():
    x, w, y = torch.randn(4, 8), torch.randn(16, 8), torch.zeros(4, dtype=torch.int64)
    call = ext.linear_cross_entropy
    with pytest.raises(ValueError, match="reduction"):
        call(x, w, y, reduction="average")
    with pytest.raises(ValueError, match="don't match"):
        call(x, torch.randn(16, 7), y)
    with pytest.raises(ValueError, match="don't match"):
        call(x, torch.randn(16), y)
    with pytest.raises(TypeError, match="share"):
        call(x, w.bfloat16(), y)
    with pytest.raises(TypeError, match="share"):
        call(x.double(), w.double(), y)
    with pytest.raises(TypeError, match="int64"):
        call(x, w, y.int())
    with pytest.raises(ValueError, match="target has shape"):
        call(x, w, y[:3])
    with pytest.raises(ValueError, match="empty"):
        call(x, torch.randn(0, 8), y)
    with pytest.raises(ValueError, match="CUDA"):
        call(x, w, y)


def test_abi_refusals():
    from tilec_b200 import _native
    lib = _native.load()
    ok = dict(dtype=2, T=4, V=16, D=8, ldx=8, ldw=8)

    def forward(x=256, w=256, y=256, loss=256, stats=256, reduction=2, **kw):
        a = {**ok, **kw}
        return lib.tilec_linear_ce_forward(x, w, y, a["dtype"], a["T"], a["V"], a["D"], a["ldx"], a["ldw"], -100,
                                           reduction, loss, stats, None, 0, None)

    for bad in (dict(dtype=3), dict(dtype=-1), dict(T=-1), dict(V=0), dict(D=0), dict(ldx=7), dict(ldw=7),
                dict(x=None), dict(w=None), dict(y=None), dict(loss=None), dict(stats=None), dict(reduction=3),
                dict(x=257), dict(w=257), dict(dtype=0, x=258)):
        assert forward(**bad) == 1, bad
    assert forward(T=1 << 31) == 7
    back = lib.tilec_linear_ce_backward
    assert back(256, 256, 256, 2, 4, 16, 8, 8, 8, -100, 2, None, 256, 256, 256, None, 0, None) == 1
    assert back(256, 256, 256, 2, 4, 16, 8, 8, 8, -100, 2, 256, None, 256, 256, None, 0, None) == 1
    assert back(256, 256, 256, 2, 4, 16, 8, 8, 8, -100, 2, 256, 256, None, None, None, 0, None) == 0
    assert back(256, 256, 256, 2, 4, 16, 8, 8, 8, -100, 2, 256, 256, 264, 256, None, 0, None) == 1
    assert back(256, 256, 256, 2, 4, 16, 8, 8, 8, -100, 2, 256, 256, 256, 264, None, 0, None) == 1
    assert lib.tilec_linear_ce_workspace_bytes(None, None, 3, 4, 16, 8, 8, 8, 2, 0) == 0


def test_abi_refuses_pointers_off_their_elements():
    from tilec_b200 import _native
    lib = _native.load()

    def forward(y=256, loss=256, stats=256):
        return lib.tilec_linear_ce_forward(256, 256, y, 2, 4, 16, 8, 8, 8, -100, 2, loss, stats, None, 0, None)

    def backward(y=256, stats=256, grad=256):
        return lib.tilec_linear_ce_backward(256, 256, y, 2, 4, 16, 8, 8, 8, -100, 2, stats, grad, 256, 256, None, 0,
                                            None)

    for bad in (dict(y=260), dict(loss=258), dict(stats=260)):
        assert forward(**bad) == 1, bad
    for bad in (dict(y=260), dict(stats=260), dict(grad=258)):
        assert backward(**bad) == 1, bad


# ---------------------------------------------------------------- numerics
gpu = pytest.mark.gpu

# (tokens, vocabulary, width): one token, one class, odd and ragged sizes, one and several
# tiles either way, few tokens with a long sum, many tokens with a small vocabulary.
SHAPES = [(1, 1, 1), (1, 7, 8), (1, 1000, 64), (3, 257, 33), (17, 300, 72), (255, 513, 64), (256, 256, 256),
          (257, 1025, 130), (300, 5000, 96), (64, 9000, 128), (700, 40, 64), (1100, 130, 520)]


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("shape", SHAPES)
def test_matches_definition(shape, dtype):
    _check(*_make(*shape, dtype), dtype)


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_reductions_and_gradients_of_the_loss(reduction, dtype):
    x, w, y = _make(333, 1111, 104, dtype, seed=1)
    go = torch.tensor(3.7, device="cuda") if reduction != "none" else None
    if reduction == "none":
        g = torch.Generator().manual_seed(2)
        go = (torch.randn(333, generator=g) * torch.logspace(-2, 2, 333)).cuda()
    _check(x, w, y, dtype, reduction, go)


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("go", [1e-7, 1e5])
def test_small_and_large_loss_gradients(go, dtype):
    """fp16 gradients of the mean are far below 1: the probabilities must not be scaled down
    before they are summed.  (fp16 results reach neither 1e-7 / 200 nor 1e5: smaller steps.)"""
    if dtype == "f16":
        go = 1e-2 if go < 1 else 200.0
    x, w, y = _make(200, 600, 64, dtype, seed=3)
    _check(x, w, y, dtype, "mean", torch.tensor(go, device="cuda"))


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_no_target_at_all(reduction, dtype):
    x, w, y = _make(70, 300, 40, dtype)
    y.fill_(IGNORE)
    x.requires_grad_(True), w.requires_grad_(True)
    loss = ext.linear_cross_entropy(x, w, y, reduction=reduction)
    if reduction == "mean":
        assert torch.isnan(loss)
    else:
        assert (loss == 0).all()
    dx, dw = torch.autograd.grad(loss, (x, w), torch.ones_like(loss))
    assert (dx == 0).all() and (dw == 0).all()


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_ignored_rows_never_matter(dtype):
    """NaN and infinities in rows without a target reach neither loss nor gradients."""
    x, w, y = _make(600, 700, 72, dtype, ignored=0.6)
    dirty = x.clone()
    dirty[y == IGNORE] = float("nan")
    dirty[(y == IGNORE).nonzero()[::2, 0]] = float("inf")
    res = []
    for xx in (x, dirty):
        xx = xx.requires_grad_(True)
        ww = w.clone().requires_grad_(True)
        loss = ext.linear_cross_entropy(xx, ww, y)
        res.append((loss.detach(), *torch.autograd.grad(loss, (xx, ww))))
    for a, b in zip(*res):
        assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_ignore_index_can_be_a_class(dtype):
    x, w, y = _make(100, 50, 32, dtype, ignored=0)
    _check(x, w, y, dtype, "mean", ignore=int(y[3]))


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_bad_targets_are_nan_and_reported(dtype):
    x, w, y = _make(300, 200, 64, dtype, ignored=0.1)
    good = ext.linear_cross_entropy(x, w, y, reduction="none")
    y2 = y.clone()
    y2[5], y2[280] = 200, -3
    x.requires_grad_(True)
    loss = ext.linear_cross_entropy(x, w, y2, reduction="none")
    bad = torch.zeros(300, dtype=torch.bool, device="cuda")
    bad[5] = bad[280] = True
    assert torch.isnan(loss[bad]).all() and torch.equal(loss[~bad], good[~bad])
    (dx,) = torch.autograd.grad(loss.sum(), (x,))
    assert torch.isnan(dx[bad]).all() and torch.isfinite(dx[~bad]).all()
    with pytest.raises(TilecError, match="BAD_INDEX"):
        ext.check_device()
    ext.check_device()


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_large_and_infinite_logits(dtype):
    x, w, y = _make(40, 300, 64, dtype, ignored=0)
    _check(x * 30, w, y, dtype, "none")   # logits of some hundreds: a confident softmax
    x2 = x.clone()
    x2[7, 3] = float("inf")
    loss = ext.linear_cross_entropy(x2, w, y, reduction="none")
    ok = torch.arange(40, device="cuda") != 7
    assert torch.isnan(loss[7]) or torch.isinf(loss[7])
    assert torch.equal(loss[ok], ext.linear_cross_entropy(x, w, y, reduction="none")[ok])


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_certain_target_has_a_tiny_loss(dtype):
    """The target's logit is the maximum by 12: the loss is 3.9e-4 and keeps its digits."""
    w = torch.eye(64).to(DT[dtype]).cuda()
    y = torch.arange(64, device="cuda")
    x = w * 12
    loss = ext.linear_cross_entropy(x, w, y, reduction="none")
    want = math.log1p(63 * math.exp(-12.0))
    # s = 1 + 63 small terms in fp32: at most 63 roundings of half a unit of 1, 2^-24 each
    assert ((loss.double() - want).abs() <= 64 * 2.0 ** -24).all()


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_strides_shapes_and_frozen_inputs(dtype):
    x, w, y = _make(2 * 37, 400, 48, dtype)
    base = ext.linear_cross_entropy(x, w, y, reduction="none")

    def same(got, ref):
        # The fp32 product picks its kernel by alignment, so two layouts may differ by twice
        # one call's error; 16-bit operands go through one kernel.
        if dtype != "f32":
            return torch.equal(got, ref)
        e = 1e-5 + 2e-6 * (x.norm(dim=1).max() * w.norm(dim=1).max()).item()
        return torch.allclose(got, ref, rtol=2e-5, atol=2 * e)

    # leading dimensions
    out = ext.linear_cross_entropy(x.view(2, 37, 48), w, y.view(2, 37), reduction="none")
    assert out.shape == (2, 37) and torch.equal(out.view(-1), base)
    # row views of wider tensors, one of them off a 16-byte boundary, and column views
    for off in (0, 1, 8):
        wide_x = torch.full((74, 72), float("nan"), dtype=x.dtype, device="cuda")
        wide_w = torch.full((400, 72), float("nan"), dtype=x.dtype, device="cuda")
        wide_x[:, off:off + 48], wide_w[:, off:off + 48] = x, w
        a = wide_x[:, off:off + 48].requires_grad_(True)
        b = wide_w[:, off:off + 48].requires_grad_(True)
        assert same(ext.linear_cross_entropy(a, b, y, reduction="none"), base)
        _check(a, b, y, dtype)
    assert same(ext.linear_cross_entropy(x.t().contiguous().t(), w.t().contiguous().t(), y, reduction="none"), base)
    # every other target of a longer tensor
    yy = torch.stack((y, y), 1)[:, 0]
    assert torch.equal(ext.linear_cross_entropy(x, w, yy, reduction="none"), base)
    # one of the operands frozen
    xg, wg = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    dx, dw = torch.autograd.grad(ext.linear_cross_entropy(xg, wg, y), (xg, wg))
    assert torch.equal(torch.autograd.grad(ext.linear_cross_entropy(xg, w, y), xg)[0], dx)
    assert torch.equal(torch.autograd.grad(ext.linear_cross_entropy(x, wg, y), wg)[0], dw)
    # a broadcast row: its gradient is the sum over tokens
    row = x[:1].clone().requires_grad_(True)
    (drow,) = torch.autograd.grad(ext.linear_cross_entropy(row.expand(74, 48), w, y, reduction="sum"), row)
    _, full, _ = _definition(x[:1].expand(74, 48), w, y, "sum")
    assert _rel(drow, full.sum(0, keepdim=True)) <= 4 * U[dtype] + 3e-5


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_no_tokens(dtype):
    x, w, y = _make(0, 50, 32, dtype, ignored=0)
    x.requires_grad_(True), w.requires_grad_(True)
    assert ext.linear_cross_entropy(x, w, y, reduction="none").shape == (0,)
    assert ext.linear_cross_entropy(x, w, y, reduction="sum") == 0
    loss = ext.linear_cross_entropy(x, w, y)
    assert torch.isnan(loss)
    dx, dw = torch.autograd.grad(loss, (x, w))
    assert dx.shape == (0, 32) and (dw == 0).all()


@gpu
def test_gradient_against_differences():
    """fp32: (L(x + h d) - L(x - h d)) / 2h against the gradient, along random directions.
    The loss is good to about 1e-6, so with h = 0.05 the quotient is good to 2e-5 plus the
    third-order term h^2 |L'''| / 6 (|L'''| along a unit direction of logits is below 1)."""
    x, w, y = _make(50, 120, 32, "f32", seed=5)
    x.requires_grad_(True), w.requires_grad_(True)
    dx, dw = torch.autograd.grad(ext.linear_cross_entropy(x, w, y), (x, w))
    g = torch.Generator(device="cuda").manual_seed(6)
    h = 0.05
    for t, grad in ((x, dx), (w, dw)):
        d = torch.randn(t.shape, device="cuda", generator=g)
        d /= d.norm()
        with torch.no_grad():
            args = [(t + s * h * d if u is t else u) for s in (1, -1) for u in (x, w)]
            up = ext.linear_cross_entropy(args[0], args[1], y).double()
            down = ext.linear_cross_entropy(args[2], args[3], y).double()
        assert abs(((up - down) / (2 * h) - (grad * d).sum().double()).item()) <= 2e-5 + h * h


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_several_pieces_of_the_vocabulary(dtype):
    """More tokens than a piece of the whole vocabulary has room for: dx adds up over pieces."""
    t, v, d = (40000, 9000, 40) if dtype == "bf16" else (20000, 9000, 24)
    x, w, y = _make(t, v, d, dtype, ignored=0.5)
    xg, wg = x.requires_grad_(True), w.requires_grad_(True)
    loss = ext.linear_cross_entropy(xg, wg, y)
    dx, dw = torch.autograd.grad(loss, (xg, wg))
    x64, w64 = x.detach().double(), w.detach().double()
    live = y != IGNORE
    dw64 = torch.zeros_like(w64)
    want = 0.0
    n = int(live.sum())
    for r in live.nonzero()[:, 0].split(4000):
        logp = torch.log_softmax(x64[r] @ w64.t(), 1)
        want += -logp.gather(1, y[r, None]).sum().item() / n
        p = logp.exp()
        p[torch.arange(len(r)), y[r]] -= 1
        p /= n
        dw64 += p.t() @ x64[r]
        if int(r[0]) == int(live.nonzero()[0, 0]):
            assert _rel(dx[r], (p @ w64).cpu()) <= 2.5 * U[dtype] + 3e-5
    assert abs(loss.item() - want) <= 1e-5 * want
    assert _rel(dw, dw64.cpu()) <= 2.5 * U[dtype] + 3e-5


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_repeats_equal_and_streams(dtype):
    """Two calls give the same bits; calls on two streams at once do not disturb each other."""
    sets = [_make(500, 3000, 128, dtype, seed=s) for s in (7, 8)]

    def call(x, w, y):
        x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        loss = ext.linear_cross_entropy(x, w, y)
        return (loss.detach(), *torch.autograd.grad(loss, (x, w)))

    want = [call(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(call(*sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for res in got[i]:
            for a, b in zip(res, want[i]):
                assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_captured_training_step(dtype):
    """Forward and backward captured into two graphs, replayed on new data, on two streams."""
    def step(x, w, y):
        x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        loss = ext.linear_cross_entropy(x, w, y)
        return (loss.detach(), *torch.autograd.grad(loss, (x, w)))

    graphs = []
    for seed in (1, 2):
        bufs = _make(300, 1500, 64, dtype, seed=seed)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(*bufs)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(*bufs)
        graphs.append((g, bufs, out))
    fresh = [_make(300, 1500, 64, dtype, seed=s, ignored=0.7) for s in (11, 12)]
    want = [step(*f) for f in fresh]
    for (_, bufs, _), f in zip(graphs, fresh):
        for b, src in zip(bufs, f):
            b.copy_(src)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for (g, _, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for (_, _, out), ref in zip(graphs, want):
        for a, b in zip(out, ref):
            assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_gave_up_is_nan_and_the_context_works(dtype):
    """Every bounded wait cut to 1 ns: the loss and gradients that were not finished are NaN,
    the status word says so, and the next call with the limit restored is right."""
    from tilec_b200 import _native
    x, w, y = _make(600, 2000, 1024, dtype, ignored=0.1)
    x.requires_grad_(True), w.requires_grad_(True)

    def step():
        loss = ext.linear_cross_entropy(x, w, y)
        return (loss.detach(), *torch.autograd.grad(loss, (x, w)))

    good = step()
    ext.check_device()
    lib = _native.load()
    _native.check(lib.tilec_mm_set_wait_limit(1, None), "set_wait_limit")
    try:
        bad = step()
        torch.cuda.synchronize()
        with pytest.raises(TilecError, match="TIMEOUT"):
            ext.check_device()
    finally:
        _native.check(lib.tilec_mm_set_wait_limit(0, None), "set_wait_limit")
    for b, g in zip(bad, good):
        assert torch.isnan(b).any() or torch.equal(b, g)
    assert any(torch.isnan(b).any() for b in bad)
    for again, g in zip(step(), good):
        assert torch.equal(again, g)
    ext.check_device()


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("reduction", ["sum", "mean"])
@pytest.mark.parametrize("shape", [(1100, 130, 520), (2048, 1000, 1024), (5000, 300, 77)])
def test_no_target_where_the_sums_over_tokens_are_cut(shape, reduction, dtype):
    """No token has a target and dW's sum over tokens is cut into slices: its slices are empty and
    its factor, 1 / 0 for the mean, is not a number to multiply them by.  Gradients are zeros."""
    x, w, y = _make(*shape, dtype)
    y.fill_(IGNORE)
    x.requires_grad_(True), w.requires_grad_(True)
    loss = ext.linear_cross_entropy(x, w, y, reduction=reduction)
    assert torch.isnan(loss) if reduction == "mean" else loss == 0
    for go in (1.0, float("inf")):
        dx, dw = torch.autograd.grad(loss, (x, w), torch.full_like(loss, go), retain_graph=True)
        assert (dx == 0).all() and (dw == 0).all()
    # the same sizes with one token left
    y[len(y) // 2] = 3
    _check(x, w, y, dtype, reduction)


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("go", [1e-45, 1e-40, 5e-39, 1.2e-38, 1e-30])
def test_vanishing_gradients_of_the_loss(go, dtype):
    """Per-token gradients down to fp32's smallest number, zeros among them: nothing infinite or
    NaN on the way, and no gradient above what the definition has.  An element of dx (dW) is at
    most 2 go max|w| (2 go T max|x|) in magnitude; rounding adds one smallest step of the type."""
    x, w, y = _make(64, 500, 64, dtype)
    x.requires_grad_(True), w.requires_grad_(True)
    loss = ext.linear_cross_entropy(x, w, y, reduction="none")
    g = torch.full_like(loss, go)
    g[::3] = 0
    dx, dw = torch.autograd.grad(loss, (x, w), g)
    step = {"bf16": 2.0 ** -133, "f16": 2.0 ** -24, "f32": 2.0 ** -149}[dtype]
    assert (dx.double().abs() <= 2.1 * go * w.double().abs().max() + step).all()
    assert (dw.double().abs() <= 2.1 * go * 64 * x.double().abs().max() + step).all()
    assert (dx[::3] == 0).all()
    if dtype == "f16":
        assert (dx == 0).all() and (dw == 0).all()


@gpu
@pytest.mark.parametrize("first", [True, False])
def test_selection_table_and_workspace(first, monkeypatch):
    """The fp32 form runs the products that the selection table selects: the first call installs the
    table, and a later table whose plans take more room changes the workspace with them."""
    from tilec_b200 import _native, select
    x, w, y = _make(300, 700, 4096, "f32")
    split = [[0, 40, 0, 40, 0, 40, _native.VARIANTS["3xtf32"], 16]]
    small = [[0, 40, 0, 40, 0, 40, _native.VARIANTS["simt"], 0]]
    try:
        if first:
            select.install(small)
            monkeypatch.setattr(select, "_installed", False)
            monkeypatch.setattr(select, "load_table", lambda path=None: split)
            monkeypatch.setattr(ext, "_installed", False)
            a = ext.linear_cross_entropy(x, w, y)       # installs `split`
            assert select._installed
            ext.matrix_mul(x[:, :64].contiguous(), x[:64, :64].contiguous())
            assert torch.equal(ext.linear_cross_entropy(x, w, y), a)
        else:
            select.install(small)
            _check(x, w, y, "f32")
        select.install(split)
        _check(x, w, y, "f32")
        select.install(small)
        _check(x, w, y, "f32")
    finally:
        monkeypatch.undo()
        select.install(select.load_table())


@pytest.mark.parametrize("grad", [False, True])
def test_refuses_forward_mode_tangents(grad):
    """There is no forward-mode derivative: a tangent is refused, not dropped."""
    fw = torch.autograd.forward_ad
    x, w, y = torch.randn(4, 8), torch.randn(16, 8), torch.zeros(4, dtype=torch.int64)
    if grad:
        x.requires_grad_(True)
    with fw.dual_level():
        for a, b in ((fw.make_dual(x, torch.ones_like(x)), w), (x, fw.make_dual(w, torch.ones_like(w)))):
            for guard in (torch.enable_grad, torch.no_grad):
                with guard(), pytest.raises(ValueError, match="forward-mode"):
                    ext.linear_cross_entropy(a, b, y)
        with pytest.raises(ValueError, match="CUDA"):   # no tangent: on to the next check
            ext.linear_cross_entropy(x, w, y)


@gpu
@pytest.mark.parametrize("t,v,d,dtype,ignored,reduction", [
    (1001, 3011, 777, "f16", 0.1, "mean"),      # odd everywhere, dW in slices or padded rows
    (1001, 3011, 777, "bf16", 0.97, "none"),
    (4096, 5000, 512, "bf16", 0.6, "sum"),      # most tokens have no target: few live rows of many
    (4096, 5000, 512, "f16", 0.999, "mean"),
    (2048, 300, 264, "bf16", 0.5, "mean"),      # long sums over tokens
    (300, 20000, 136, "f16", 0.3, "sum"),       # long sums over the vocabulary
    (2048, 9001, 100, "f32", 0.6, "mean")])
def test_masked_and_ragged_training(t, v, d, dtype, ignored, reduction):
    x, w, y = _make(t, v, d, dtype, seed=t + v, ignored=ignored)
    go = None
    if reduction == "none":
        go = (torch.rand(t, generator=torch.Generator().manual_seed(4)) + 0.5).cuda()
    _check(x, w, y, dtype, reduction, go)


@gpu
@pytest.mark.parametrize("dtype,t,d", [("bf16", 40000, 41), ("f16", 40000, 41), ("f32", 20000, 25)])
def test_several_pieces_of_an_odd_width(dtype, t, d):
    """Pieces of the vocabulary with gradients whose rows are no whole 16-byte pieces; every other
    row frozen out by ignore_index, dx and dW asked for apart give what they give together."""
    v = 9000
    x, w, y = _make(t, v, d, dtype, ignored=0.5)
    xg, wg = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    loss = ext.linear_cross_entropy(xg, wg, y)
    dx, dw = torch.autograd.grad(loss, (xg, wg))
    live = (y != IGNORE).nonzero()[:, 0]
    n, w64 = len(live), w.double()
    dw64, dx64 = torch.zeros_like(w64), torch.zeros(t, d, dtype=torch.float64, device="cuda")
    for r in live.split(4000):
        p = torch.softmax(x[r].double() @ w64.t(), 1)
        p[torch.arange(len(r)), y[r]] -= 1
        p /= n
        dw64 += p.t() @ x[r].double()
        dx64[r] = p @ w64
    # fp16: gradients are of the order of 1 / n, some below 2^-14, where a step is 2^-24 whatever their size
    for got, ref in ((dx, dx64), (dw, dw64)):
        sub = 2.0 ** -25 * math.sqrt(ref.numel()) / ref.norm().item() if dtype == "f16" else 0.0
        assert _rel(got, ref.cpu()) <= 2.5 * U[dtype] + 3e-5 + sub
    assert (dx[y == IGNORE] == 0).all()
    assert torch.equal(torch.autograd.grad(ext.linear_cross_entropy(xg, w, y), xg)[0], dx)
    assert torch.equal(torch.autograd.grad(ext.linear_cross_entropy(x, wg, y), wg)[0], dw)
