"""4-bit weights: packing, quantising and refusals (CPU), matrix_mul_w4 against 64 bits (GPU).

Element-wise bounds, u = half a unit in the last place (2^-8 bf16, 2^-11 fp16, 2^-24 fp32) and
S = sum_k |x (code - zero) scale|:

* up to 8 rows: x is rounded to a whole number of steps of 2^-29 of its 128-k block's largest
  magnitude, far below what follows; group sums are exact, the at most 64 blocks' (in up to 24
  parts) and four digits' sums are added in fp32, (64 + 4) * 2^-24 S for the upper digit, which
  holds all but 2^-7 of S: below 2^-17.8 S at worst, and the roundings are independent: 2^-18 S
  is held to; then one rounding, u |y|.
  Three to eight rows of 16-bit x: products of codes and x are exact; a 128-k block adds 8
  groups of 16 products to an accumulator, each sum truncated at worst (16 * 2^-23 S), and the
  at most 64 blocks are added in fp32 (64 * 2^-24 S), the scale's product rounds once: below
  2^-18 S.
* more rows: the weight is rounded to the type, u S more (fp32: the 3xTF32 product,
  3 * 2^-20 S); sums over K <= 8192 in the tensor cores' fp32 stay below 2^-14 S (K / 16 sums,
  each truncated by 2^-23).
* fp16 results below 2^-14 are multiples of 2^-24: 2^-25 absolute.
"""
import pytest
import torch

from tilec_b200 import ext

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
U = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}


def _make(m, n, k, group, dtype, zeros=True, bias=False, sdtype=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    groups = -(-k // group)
    codes = torch.randint(0, 16, (n, k), generator=g, dtype=torch.uint8)
    scales = ((torch.rand(n, groups, generator=g) + 0.1) * k ** -0.5 / 4).to(DT[sdtype or dtype])
    z = torch.randint(0, 16, (n, groups), generator=g, dtype=torch.uint8) if zeros else None
    x = torch.randn(m, k, generator=g).to(DT[dtype])
    b = torch.randn(n, generator=g).to(DT[dtype]) if bias else None
    return x, codes, scales, z, b


def _weight64(codes, scales, zeros, group):
    k = codes.shape[1]
    s = scales.double().repeat_interleave(group, 1)[:, :k]
    z = 8.0 if zeros is None else zeros.double().repeat_interleave(group, 1)[:, :k]
    return (codes.double() - z) * s


def _bound(x, w, y, dtype, rows):
    s = x.double().abs() @ w.abs().t()
    few = rows <= 8
    rel = 2.0 ** -18 if few else 2.0 ** -14 + (3 * 2.0 ** -20 if dtype == "f32" else U[dtype])
    return rel * s + 1.001 * U[dtype] * y.abs() + (2.0 ** -25 if dtype == "f16" else 0.0)


def _check(x, codes, scales, zeros, bias, group, dtype, call=None):
    w = _weight64(codes, scales, zeros, group)
    y = x.double() @ w.t()
    tol = _bound(x, w, y, dtype, len(x))
    if bias is not None:
        y = y + bias.double()
        tol = tol + U[dtype] * y.abs() + 2.0 ** -23 * bias.double().abs()
    weight = ext.pack_w4(codes, scales, zeros, group).to("cuda")
    got = (call or ext.matrix_mul_w4)(x.cuda(), weight, None if bias is None else bias.cuda())
    assert got.dtype == x.dtype and got.shape == y.shape
    err = (got.cpu().double() - y).abs()
    assert torch.isfinite(got).all()
    assert (err <= tol).all(), f"worst {(err / tol.clamp(min=1e-300)).max():.2f} of the bound"
    ext.check_device()


# ---------------------------------------------------------------- CPU
@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("n,k", [(1, 1), (5, 300), (3, 128), (16, 513)])
def test_pack_keeps_codes_and_values(n, k, group):
    _, codes, scales, zeros, _ = _make(1, n, k, group, "f32")
    w = ext.pack_w4(codes, scales, zeros, group)
    assert torch.equal(w.unpack(), codes)
    assert torch.equal(w.dequantize().double(), _weight64(codes, scales, zeros, group).float().double())
    assert torch.equal(w.scales(), scales) and torch.equal(w.zeros(), zeros)
    # the layout of include/tilec_mm.h, word by word
    blocks, per_block = -(-k // 128), max(1, 128 // group)
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        half = ext.pack_w4(codes, scales.to(dtype), zeros, group)
        assert torch.equal(half.scales(), scales.to(dtype)) and torch.equal(half.zeros(), zeros)
        assert (ext.pack_w4(codes, scales.to(dtype), None, group).zeros() == 8).all()
        wide = 2 if dtype == torch.float32 else 1
        assert half.data.shape == (-(-n // 16), blocks, 64 * per_block * wide + 1024)
        for row in range(n):
            for b in range(blocks):
                piece = half.data[row // 16, b]
                words = piece[:-1024].clone().view(torch.int32).view(16, per_block, wide)[row % 16]
                for i in range(per_block):
                    at = (b * 128 + i * (128 // per_block)) // group
                    if b * 128 + i * (128 // per_block) >= k:
                        continue
                    s = scales.to(dtype)[row, at:at + 1].contiguous()
                    bits = int(s.view(torch.int32) if wide == 2 else s.view(torch.int16).int() << 16)
                    z = int(zeros[row, at])
                    assert words[i].tolist() == ([z, bits] if wide == 2 else [z | bits])
                word = piece[-1024:].reshape(16, 16, 4)[row % 16].long()
                word = word[:, 0] | word[:, 1] << 8 | word[:, 2] << 16 | word[:, 3] << 24
                full = torch.nn.functional.pad(codes[row, b * 128:b * 128 + 128], (0, max(0, b * 128 + 128 - k)))
                e = torch.arange(128)
                j, t, i, odd = e // 32, e % 32 // 8, e % 8 // 2, e % 2
                assert torch.equal(word[4 * t + j] >> (4 * i + 16 * odd) & 15, full.long())


@pytest.mark.parametrize("symmetric", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("group", [32, 128])
def test_quantize_error_is_half_a_step(group, dtype, symmetric):
    g = torch.Generator().manual_seed(1)
    w = torch.randn(24, 300, generator=g).to(DT[dtype])
    w[3] = 0                       # a group of zeros
    w[4] = w[4].abs() + 1          # all positive: the range is widened to hold zero
    q = ext.quantize_w4(w, group, symmetric)
    step = q.scales().float().repeat_interleave(group, 1)[:, :300]
    err = (q.dequantize() - w.float()).abs()
    # the rounded scale spans 15 (7) steps short by up to 15 u (7 u) of a step at the ends,
    # and the zero point is rounded to a step
    slack = 15 * U[dtype] + 2.0 ** -20
    assert (err <= (0.5 + (0 if symmetric else 0.5) + slack) * step + 1e-30).all()
    assert (q.dequantize()[3] == 0).all()
    assert q.shape == (24, 300) and (q.zeros() == 8).all() >= symmetric


def test_refusals():
    c, s = torch.zeros(4, 64, dtype=torch.uint8), torch.ones(4, 2)
    for bad in (0, 16, 48, 96, 160, -128, 32.0):
        with pytest.raises(ValueError, match="group_size"):
            ext.pack_w4(c, s, group_size=bad)
        with pytest.raises(ValueError, match="group_size"):
            ext.quantize_w4(torch.ones(4, 64), bad)
    with pytest.raises(TypeError, match="uint8"):
        ext.pack_w4(c.int(), s, group_size=32)
    with pytest.raises(ValueError, match="scales have shape"):
        ext.pack_w4(c, s, group_size=64)
    with pytest.raises(TypeError, match="scales must be"):
        ext.pack_w4(c, s.double(), group_size=32)
    with pytest.raises(ValueError, match="zeros have shape"):
        ext.pack_w4(c, s, c[:, :1], group_size=32)
    with pytest.raises(TypeError, match="zeros must be"):
        ext.pack_w4(c, s, s, group_size=32)
    with pytest.raises(ValueError, match="0..15"):
        ext.pack_w4(c + 16, s, group_size=32)
    with pytest.raises(ValueError, match="K >= 1"):
        ext.pack_w4(c[:, :0], s, group_size=32)
    with pytest.raises(TypeError, match="weight must be"):
        ext.quantize_w4(torch.ones(4, 64, dtype=torch.float64))
    w = ext.pack_w4(c, s, group_size=32)
    x = torch.ones(2, 64)
    with pytest.raises(TypeError, match="W4Weight"):
        ext.matrix_mul_w4(x, c)
    with pytest.raises(ValueError, match="don't match"):
        ext.matrix_mul_w4(x[:, :63], w)
    with pytest.raises(TypeError, match="x must be"):
        ext.matrix_mul_w4(x.double(), w)
    with pytest.raises(ValueError, match="CUDA"):
        ext.matrix_mul_w4(x, w)


def test_abi_refusals():
    from tilec_b200 import _native
    lib = _native.load()
    ok = dict(x=256, dtype=2, M=2, ldx=64, weight=256, sdt=2, N=8, K=64, group=32, bias=None, out=256, ldo=8)

    def call(**kw):
        return lib.tilec_mm_w4(*{**ok, **kw}.values(), None, 0, None)

    for bad in (dict(dtype=3), dict(sdt=-1), dict(M=-1), dict(N=-1), dict(K=0), dict(ldx=63), dict(group=16),
                dict(group=0), dict(group=192), dict(x=None), dict(weight=None), dict(out=None),
                dict(ldo=7), dict(weight=264), dict(x=257), dict(out=257), dict(bias=257)):
        assert call(**bad) == 1, bad
    assert call(M=1 << 31) == 7
    assert call(M=0, x=None, out=None) == 0 and call(N=0, weight=None, ldo=0) == 0
    assert lib.tilec_mm_w4_workspace_bytes(None, 9, 2, 64, 2, 8, 64, 32, None, 8) == 0


def test_weight_fields_are_checked_and_read_only():
    """The kernels read data in place by shape, group_size and scale_dtype."""
    w = ext.pack_w4(torch.zeros(20, 300, dtype=torch.uint8), torch.ones(20, 5, dtype=torch.bfloat16), group_size=64)
    again = ext.W4Weight(w.shape, w.group_size, w.scale_dtype, w.data)
    assert torch.equal(again.unpack(), w.unpack()) and again.shape == (20, 300)
    for bad in (dict(shape=(33, 300)), dict(shape=(20, 400)), dict(shape=(-1, 300)), dict(shape=(20, 0)),
                dict(group_size=32), dict(group_size=48), dict(scale_dtype=torch.float32), dict(data=w.data[:1]),
                dict(data=w.data.transpose(0, 1).contiguous().transpose(0, 1)),
                dict(data=torch.zeros(w.data.numel() + 1, dtype=torch.uint8)[1:].view(w.data.shape))):
        with pytest.raises(ValueError, match="W4Weight"):
            ext.W4Weight(**{**dict(shape=w.shape, group_size=64, scale_dtype=w.scale_dtype, data=w.data), **bad})
    for bad in (dict(scale_dtype=torch.float64), dict(data=w.data.view(torch.int8))):
        with pytest.raises(TypeError, match="W4Weight"):
            ext.W4Weight(**{**dict(shape=w.shape, group_size=64, scale_dtype=w.scale_dtype, data=w.data), **bad})
    for name in ("shape", "group_size", "scale_dtype", "data"):
        with pytest.raises(AttributeError):
            setattr(w, name, getattr(w, name))
    assert ext.pack_w4(torch.zeros(0, 5, dtype=torch.uint8), torch.ones(0, 1)).shape == (0, 5)


def test_quantize_extremes():
    top = 0.9 * torch.finfo(torch.float32).max   # high - low is past the type's range, 8 steps are not
    w = torch.tensor([[top, -top, 0.0, top / 2], [0.0, 0.0, 0.0, 0.0], [1e-45, 0.0, 0.0, 0.0]])
    q = ext.quantize_w4(w, 32)
    step = top / 7.5
    assert torch.isfinite(q.scales()).all() and ((q.dequantize()[0].double() - w[0].double()).abs() <= step * 1.001).all()
    assert (q.dequantize()[1] == 0).all() and (q.dequantize()[2] <= 1e-44).all()
    for bad in (float("inf"), float("-inf"), float("nan")):
        with pytest.raises(ValueError, match="infinities"):
            ext.quantize_w4(torch.tensor([[1.0, bad]]))


# ---------------------------------------------------------------- GPU
gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("n,k", [(1, 1), (7, 31), (16, 128), (33, 300), (100, 1024), (130, 4100)])
def test_one_token(n, k, group, dtype):
    _check(*_make(1, n, k, group, dtype), group, dtype)


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("m", [2, 3, 8, 9, 10, 11, 16, 17, 32, 33, 65, 127, 128, 129, 257])
def test_rows(m, dtype):
    """Either side of each variant's row count, with bias, symmetric and with zero points."""
    for zeros, group, n, k in ((True, 32, 90, 640), (False, 128, 259, 1157)):
        _check(*_make(m, n, k, group, dtype, zeros=zeros, bias=True, seed=m), group, dtype)


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("sdtype", ["bf16", "f16", "f32"])
def test_scale_types(sdtype, dtype):
    for m in (1, 5, 40):
        _check(*_make(m, 70, 384, 64, dtype, sdtype=sdtype), 64, dtype)


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("m,n,k", [(1, 16, 8192), (5, 4096, 512), (1, 300, 8190), (40, 520, 8192), (20, 2500, 1000),
                                   (128, 130, 4000), (300, 700, 2048)])
def test_long_sums_and_many_tiles(m, n, k, dtype):
    _check(*_make(m, n, k, 128, dtype), 128, dtype)


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_exact_values(dtype):
    """Small whole numbers: every product and sum is exact, so the result is too."""
    g = torch.Generator().manual_seed(3)
    for m in (1, 6, 50):
        codes = torch.randint(0, 16, (75, 384), generator=g, dtype=torch.uint8)
        scales = torch.randint(1, 3, (75, 12), generator=g).to(DT[dtype])
        zeros = torch.randint(0, 16, (75, 12), generator=g, dtype=torch.uint8)
        x = torch.zeros(m, 384)
        x[:, torch.randperm(384, generator=g)[:8]] = torch.randint(-2, 3, (m, 8), generator=g).float()
        w = ext.pack_w4(codes, scales, zeros, 32).to("cuda")
        got = ext.matrix_mul_w4(x.to(DT[dtype]).cuda(), w).cpu().double()
        want = x.double() @ _weight64(codes, scales, zeros, 32).t()
        assert torch.equal(got, want.to(DT[dtype]).double())


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("m", [3, 40])
def test_strides_out_and_shapes(m, dtype):
    x, codes, scales, zeros, bias = _make(m, 200, 320, 64, dtype, bias=True)
    w = ext.pack_w4(codes, scales, zeros, 64).to("cuda")
    x, bias = x.cuda(), bias.cuda()
    base = ext.matrix_mul_w4(x, w, bias)
    for off in (0, 1, 8):   # row views, off a 16-byte boundary too; what lies beside them is NaN
        wide = torch.full((m, 400), float("nan"), dtype=x.dtype, device="cuda")
        wide[:, off:off + 320] = x
        got = ext.matrix_mul_w4(wide[:, off:off + 320], w, bias)
        if dtype == "f32" and m > 8:   # the fp32 product picks its kernel by alignment
            torch.testing.assert_close(got, base, rtol=1e-5, atol=1e-4)
        else:
            assert torch.equal(got, base)
    assert torch.equal(ext.matrix_mul_w4(x.t().contiguous().t(), w, bias), base)
    assert torch.equal(ext.matrix_mul_w4(x.view(1, m, 320), w, bias), base.view(1, m, 200))
    assert ext.matrix_mul_w4(x[0], w, bias).shape == (200,)
    for off in (0, 3):      # a wider out: its other columns stay as they were
        buf = torch.full((m, 260), 7.0, dtype=x.dtype, device="cuda")
        view = buf[:, off:off + 200]
        assert ext.matrix_mul_w4(x, w, bias, out=view) is view
        if dtype == "f32" and m > 8:
            torch.testing.assert_close(view, base, rtol=1e-5, atol=1e-4)
        else:
            assert torch.equal(view, base)
        assert (buf[:, :off] == 7).all() and (buf[:, off + 200:] == 7).all()
    odd = ext.pack_w4(codes[:197], scales[:197], zeros[:197], 64).to("cuda")   # N no multiple of 8, the stride one
    buf = torch.full((m, 256), 7.0, dtype=x.dtype, device="cuda")
    ext.matrix_mul_w4(x, odd, bias[:197], out=buf[:, :197])
    torch.testing.assert_close(buf[:, :197], base[:, :197], rtol=1e-5, atol=1e-4)
    assert (buf[:, 197:] == 7).all()
    for bad in (base.float() if dtype != "f32" else base.half(), base[:, :-1], base.t().contiguous().t(), base.cpu()):
        with pytest.raises(ValueError, match="out must"):
            ext.matrix_mul_w4(x, w, bias, out=bad)
    with pytest.raises(ValueError, match="bias must"):
        ext.matrix_mul_w4(x, w, bias[:-1])
    with pytest.raises(ValueError, match="not differentiable"):
        ext.matrix_mul_w4(x.clone().requires_grad_(True), w)
    with pytest.raises(ValueError, match="one CUDA device"):
        ext.matrix_mul_w4(x, w.to("cpu"))


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_empty(dtype):
    x, codes, scales, zeros, _ = _make(0, 20, 64, 32, dtype)
    w = ext.pack_w4(codes, scales, zeros, 32).to("cuda")
    assert ext.matrix_mul_w4(x.cuda(), w).shape == (0, 20)
    w = ext.pack_w4(codes[:0], scales[:0], zeros[:0], 32).to("cuda")
    assert ext.matrix_mul_w4(torch.ones(3, 64, dtype=DT[dtype], device="cuda"), w).shape == (3, 0)


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("m", [2, 9, 40])
def test_not_finite_values_stay_in_their_row(m, dtype):
    x, codes, scales, zeros, _ = _make(m, 150, 256, 64, dtype)
    w = ext.pack_w4(codes, scales, zeros, 64).to("cuda")
    x = x.cuda()
    base = ext.matrix_mul_w4(x, w)
    bad = x.clone()
    bad[0, 17], bad[1, 40] = float("inf"), float("nan")
    got = ext.matrix_mul_w4(bad, w)
    assert not torch.isfinite(got[0]).any() or (codes[:, 17] == zeros[:, 0]).any()
    value = codes[:, 17].int() - zeros[:, 0].int()
    assert torch.isnan(got[1]).all()
    assert (~torch.isfinite(got[0].cpu()))[value != 0].all()
    assert torch.equal(got[2:], base[2:])


@gpu
@pytest.mark.parametrize("m", [1, 40])
def test_streams_and_graphs(m):
    """Two graphs replayed at once on two streams with new inputs; repeats give the same bits."""
    sets = []
    for seed in (1, 2):
        x, codes, scales, zeros, _ = _make(m, 500, 3001, 32, "f32" if m == 1 else "bf16", seed=seed)
        w = ext.pack_w4(codes, scales, zeros, 32).to("cuda")
        x = x.cuda()
        ext.matrix_mul_w4(x, w)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = ext.matrix_mul_w4(x, w)
        sets.append((g, x, w, y))
    want = []
    for _, x, w, _ in sets:
        x.mul_(-0.5)
        want.append(ext.matrix_mul_w4(x, w))
        assert torch.equal(want[-1], ext.matrix_mul_w4(x, w))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(4):
        for (g, _, _, _), st in zip(sets, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for (_, _, _, y), ref in zip(sets, want):
        assert torch.equal(y, ref)


@gpu
def test_offsets_past_32_bits():
    """Codes of 2.2 GB: rows past 2^31 bytes are read from where they are."""
    n, k = 140000, 32768
    g = torch.Generator(device="cuda").manual_seed(5)
    data = torch.randint(0, 256, (n // 16, k // 128, 64 + 1024), device="cuda", generator=g, dtype=torch.uint8)
    words = torch.rand(n // 16, k // 128, 16, device="cuda", generator=g).half().view(torch.int16).int() << 16 | 8
    data[:, :, :64] = words.view(torch.uint8)
    w = ext.W4Weight((n, k), 128, torch.float16, data)
    x = torch.zeros(1, k, device="cuda", dtype=torch.float16)
    x[0, ::97] = 1.0
    got = ext.matrix_mul_w4(x, w)[0]
    for rows in (slice(0, 64), slice(n - 64, n)):
        part = ext.W4Weight((64, k), 128, torch.float16, data[rows.start // 16:rows.stop // 16])
        want = x.double() @ part.dequantize().double().t()
        assert ((got[rows].double() - want[0]).abs() <= 2.0 ** -10 * want[0].abs() + 2.0 ** -14 * 400).all()


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_train_quantise_serve(dtype):
    """The operators together: train a small head with linear_cross_entropy, quantise it, and
    serve its logits in 4 bits; they equal the dequantised head's, and the loss over them is
    the loss linear_cross_entropy gives for the dequantised head."""
    g = torch.Generator(device="cuda").manual_seed(9)
    v, d, t = 1000, 256, 24
    head = (torch.randn(v, d, device="cuda", generator=g) * d ** -0.5).to(DT[dtype]).requires_grad_(True)
    x = torch.randn(t, d, device="cuda", generator=g).to(DT[dtype])
    y = torch.randint(0, v, (t,), device="cuda", generator=g)
    for _ in range(3):
        loss = ext.linear_cross_entropy(x, head, y)
        loss.backward()
        with torch.no_grad():
            head -= head.grad
            head.grad = None
    q = ext.quantize_w4(head, 64)
    per_token = []
    with torch.no_grad():
        whole = ext.matrix_mul_w4(x, q)            # a batch at once (24 rows)
        for i in range(t):                          # and one token after another
            step = ext.matrix_mul_w4(x[i], q)
            per_token.append(step)
    w = q.dequantize().double()
    ref = x.double() @ w.t()
    bound = 2.0 ** -18 * (x.double().abs() @ w.abs().t()) + 1.001 * U[dtype] * ref.abs()
    # 24 rows at once: the weight is rounded to bf16, or (fp32) goes through the 3xTF32 product
    more = (2.0 ** -14 + (U[dtype] if dtype == "bf16" else 0)) * (x.double().abs() @ w.abs().t())
    assert ((whole.double() - ref).abs() <= bound + more).all()
    assert ((torch.stack(per_token).double() - ref).abs() <= bound).all()
    if dtype == "f32":
        got = ext.linear_cross_entropy(x, q.dequantize(), y, reduction="none").double()
        want = torch.logsumexp(ref, 1) - ref.gather(1, y[:, None])[:, 0]
        e = 1e-5 + 2e-6 * (x.double().norm(dim=1).max() * w.norm(dim=1).max()).item()
        assert ((got - want).abs() <= e + 1e-5 * want).all()


@gpu
@pytest.mark.parametrize("m,dtype", [(1, "bf16"), (5, "f32"), (4, "f16"), (64, "bf16"), (200, "f16"), (300, "bf16")])
def test_gave_up_is_nan_or_right_and_the_context_works(m, dtype, monkeypatch):
    """Every bounded wait cut to 1 ns: what a kernel did not finish is NaN (a few-row kernel may
    compute such outputs one by one instead), the status word says so, and the next call with
    the limit restored is right.  No fault, no endless wait."""
    from tilec_b200 import TilecError, _native
    x, codes, scales, zeros, _ = _make(m, 260, 2048, 64, dtype)
    w = ext.pack_w4(codes, scales, zeros, 64).to("cuda")
    x = x.cuda()
    good = ext.matrix_mul_w4(x, w)
    out = torch.full_like(good, 12345.0)
    ext.check_device()
    lib = _native.load()
    _native.check(lib.tilec_mm_set_wait_limit(1, None), "set_wait_limit")
    try:
        ext.matrix_mul_w4(x, w, out=out)
        torch.cuda.synchronize()
        gave_up = False
        try:
            ext.check_device()
        except TilecError as e:
            assert "TIMEOUT" in str(e)
            gave_up = True
    finally:
        _native.check(lib.tilec_mm_set_wait_limit(0, None), "set_wait_limit")
    nan = torch.isnan(out)
    assert gave_up or not nan.any()
    w64 = _weight64(codes, scales, zeros, 64).cuda()
    err = (out.double() - x.double() @ w64.t()).abs()
    assert (err[~nan] <= _bound(x.cpu(), w64.cpu(), good.cpu().double(), dtype, m).cuda()[~nan] * 2).all()
    assert torch.equal(ext.matrix_mul_w4(x, w), good)
    ext.check_device()


@gpu
def test_workspace_follows_each_operand_alignment():
    """x 240 bytes into its storage, out on a 16-byte boundary or off it: each call's workspace
    is sized for its own operands."""
    x, codes, scales, zeros, _ = _make(300, 64, 256, 128, "bf16")
    weight = ext.pack_w4(codes, scales, zeros).to("cuda")
    xs = torch.zeros(300 * 256 + 120, dtype=torch.bfloat16, device="cuda")[120:].view(300, 256).copy_(x)
    room = torch.empty(300 * 64 + 8, dtype=torch.bfloat16, device="cuda")
    ref = ext.matrix_mul_w4(xs, weight)
    for at in (0, 1, 3, 8):
        out = room[at:at + 300 * 64].view(300, 64)
        assert torch.equal(ext.matrix_mul_w4(xs, weight, out=out), ref)
    with pytest.raises(ValueError, match="requires a gradient"):
        ext.matrix_mul_w4(xs, weight, out=room[:300 * 64].view(300, 64).requires_grad_())


@gpu
@pytest.mark.parametrize("m,k,dtype", [(128, 8192, "bf16"), (20, 14336, "f16"), (250, 4096, "bf16")])
def test_gave_up_between_codes_and_x(m, k, dtype):
    """The expanding kernel with every wait cut to 1 ns, over and over: it may give up between a
    unit's codes and the blocks of x that go with them.  The calls in between, at the full limit
    on the same SMs, give the same bits each time."""
    from tilec_b200 import TilecError, _native
    x, codes, scales, zeros, _ = _make(m, 260, k, 64, dtype)
    w = ext.pack_w4(codes, scales, zeros, 64).to("cuda")
    x = x.cuda()
    good = ext.matrix_mul_w4(x, w)
    ext.check_device()
    lib = _native.load()
    given_up = 0
    for _ in range(20):
        _native.check(lib.tilec_mm_set_wait_limit(1, None), "set_wait_limit")
        try:
            got = ext.matrix_mul_w4(x, w)
        finally:
            _native.check(lib.tilec_mm_set_wait_limit(0, None), "set_wait_limit")
        assert torch.equal(ext.matrix_mul_w4(x, w), good)
        nan = torch.isnan(got)
        assert torch.equal(got[~nan], good[~nan])
        try:
            ext.check_device()
            assert not nan.any()
        except TilecError as e:
            assert "TIMEOUT" in str(e)
            given_up += 1
    assert given_up


@gpu
@pytest.mark.parametrize("m,n,k,group,dtype,sdtype",
                         [(16, 40005, 2700, 32, "bf16", "f32"),    # two slabs of x, two groups of row tiles a CTA
                          (4, 40005, 1000, 64, "f16", "f16"),      # two groups
                          (6, 40005, 5400, 128, "f32", "f32"),     # both, x cut beforehand
                          (16, 260, 28672, 32, "f16", "f32")])     # slabs, K shared by a cluster
def test_gave_up_before_the_last_slab_or_group(m, n, k, group, dtype, sdtype):
    """A streaming warp that gave up goes on through the slabs of x and groups of row tiles that are
    left: its outputs are NaN (digits: right), the others right, and correct calls in between on the
    same SMs give the same bits each time."""
    from tilec_b200 import TilecError, _native
    x, codes, scales, zeros, _ = _make(m, n, k, group, dtype, sdtype=sdtype)
    w = ext.pack_w4(codes.cuda(), scales.cuda(), zeros.cuda(), group)
    x = x.cuda()
    good = ext.matrix_mul_w4(x, w)
    ext.check_device()
    w64 = _weight64(codes.cuda(), scales.cuda(), zeros.cuda(), group)
    y = x.double() @ w64.t()
    # twice the bound of few rows: groups' sums and parts added in fp32 in any order (see _long_bound)
    tol = 2 * _long_bound(x, w64, y, dtype, k, group)
    assert ((good.double() - y).abs() <= tol).all()
    lib = _native.load()
    given_up = 0
    flush = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")
    for _ in range(8):
        flush.zero_()   # the weight comes from memory: waits last longer than a step of the clock
        _native.check(lib.tilec_mm_set_wait_limit(1, None), "set_wait_limit")
        try:
            got = ext.matrix_mul_w4(x, w)
        finally:
            _native.check(lib.tilec_mm_set_wait_limit(0, None), "set_wait_limit")
        assert torch.equal(ext.matrix_mul_w4(x, w), good)
        nan = torch.isnan(got)
        assert ((got.double() - y).abs() <= tol)[~nan].all()
        try:
            ext.check_device()
            assert not nan.any()
        except TilecError as e:
            assert "TIMEOUT" in str(e)
            given_up += 1
    assert given_up or n < 1000    # few pieces a warp: they may all have landed before the first wait


def _long_bound(x, w64, y, dtype, k, group):
    """Up to 16 rows on the streaming kernel, any K, S = sum_k |x w|: one fp32 addition per group
    (of at most 128 k), per warp (16), CTA of a cluster (8) and slab of x (8), each off by 2^-24 S at
    worst, 8 more for the scale's product and the digits' sums; a group's 16-bit sums on the tensor
    cores as in the header (16 * 2^-23 S).  Digits hold x to 2^-30 of the power of two at or below
    the largest magnitude of its block of 128 k (fp32 x; a 16-bit row alone too)."""
    adds = -(-k // min(group, 128)) + 40
    s = x.double().abs() @ w64.abs().t()
    blocks = torch.nn.functional.pad(x.double().abs(), (0, -k % 128)).view(len(x), -1, 128)
    step = torch.exp2(torch.floor(torch.log2(blocks.amax(2).clamp(min=2.0 ** -90))) - 30)
    wb = torch.nn.functional.pad(w64.abs(), (0, -k % 128)).view(len(w64), -1, 128).sum(2)
    held = step @ wb.t()
    return (adds * 2.0 ** -24 + 2.0 ** -19) * s + held + 1.001 * U[dtype] * y.abs() + (
        2.0 ** -25 if dtype == "f16" else 0.0)


@gpu
def test_selection_table_and_workspace(monkeypatch):
    """fp32 x of many rows runs the product that the selection table selects, here too."""
    from tilec_b200 import _native, select
    data = _make(40, 300, 4096, 128, "f32")
    try:
        monkeypatch.setattr(select, "_installed", False)
        monkeypatch.setattr(select, "load_table",
                            lambda path=None: [[0, 40, 0, 40, 0, 40, _native.VARIANTS["simt"], 0]])
        _check(*data, 128, "f32")
        assert select._installed
        select.install([[0, 40, 0, 40, 0, 40, _native.VARIANTS["3xtf32"], 16]])
        _check(*data, 128, "f32")
    finally:
        monkeypatch.undo()
        select.install(select.load_table())


def test_refuses_forward_mode_tangents():
    """There is no derivative: a tangent of x, bias or out is refused, not dropped."""
    fw = torch.autograd.forward_ad
    w = ext.pack_w4(torch.zeros(4, 64, dtype=torch.uint8), torch.ones(4, 2), group_size=32)
    x, b, out = torch.ones(2, 64), torch.ones(4), torch.ones(2, 4)
    with fw.dual_level():
        def dual(t):
            return fw.make_dual(t, torch.ones_like(t))
        for args in ((dual(x), w), (x, w, dual(b)), (x, w, None, dual(out))):
            with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):
                ext.matrix_mul_w4(*args)
        with pytest.raises(ValueError, match="CUDA"):
            ext.matrix_mul_w4(x, w, b, out)


# (rows, N, K, group, type of x, type of scales).  From 2368 rows of the weight on a CTA has a row
# tile of its own and takes all of K, so that several rows of a long x come in slabs.
LONG = [(8, 2500, 14336, 128, "bf16", "bf16"), (8, 2401, 28672, 64, "f16", "f16"),    # 16-bit x in slabs
        (16, 2500, 8192, 128, "bf16", "f32"), (13, 2400, 11008, 32, "f16", "bf16"),
        (9, 2370, 4224, 64, "bf16", "f16"), (13, 8192, 8192, 128, "bf16", "bf16"),
        (1, 2500, 40000, 128, "f32", "f32"), (2, 2500, 30000, 32, "f32", "f32"),      # digits in slabs
        (3, 2500, 11008, 128, "f32", "f32"), (8, 2400, 8192, 64, "f32", "bf16"),
        (2, 9000, 16000, 64, "f16", "f16"), (1, 300, 60000, 256, "bf16", "bf16"),
        (8, 40005, 300, 128, "bf16", "bf16"), (1, 40005, 400, 64, "f16", "f16"),      # many row tiles
        (5, 70001, 160, 32, "f32", "f32"), (16, 40005, 2700, 64, "f16", "f32"),
        (17, 2500, 28672, 128, "bf16", "bf16"), (200, 1000, 14336, 64, "f16", "f16"),  # tcgen05
        (40, 500, 20000, 128, "bf16", "f16"), (20, 500, 20000, 128, "f32", "f32")]


@gpu
@pytest.mark.parametrize("m,n,k,group,dtype,sdtype", LONG)
def test_long_x_and_many_row_tiles(m, n, k, group, dtype, sdtype):
    """More of K than the shared copy of x holds at once, and more row tiles than a CTA sums at once;
    x in rows of a wider tensor, on and off 16-byte boundaries, gives the same bits."""
    x, codes, scales, zeros, bias = _make(m, n, k, group, dtype, bias=True, sdtype=sdtype)
    x, codes, scales, zeros, bias = (t.cuda() for t in (x, codes, scales, zeros, bias))
    w = ext.pack_w4(codes, scales, zeros, group)
    w64 = _weight64(codes, scales, zeros, group)
    y = x.double() @ w64.t()
    if m <= 8 or (m <= 16 and dtype != "f32" and sdtype != dtype):
        tol = _long_bound(x, w64, y, dtype, k, group)
    else:   # the weight rounded to x's type; sums of 16 (fp32: 8, three products), 2^-23 off each at worst
        s = x.double().abs() @ w64.abs().t()
        rel = 3 * -(-k // 8) * 2.0 ** -23 + 3 * 2.0 ** -20 if dtype == "f32" else -(-k // 16) * 2.0 ** -23 + U[dtype]
        tol = rel * s + 1.001 * U[dtype] * y.abs() + (2.0 ** -25 if dtype == "f16" else 0.0)
    y = y + bias.double()
    tol = tol + U[dtype] * y.abs() + 2.0 ** -23 * bias.double().abs()
    got = ext.matrix_mul_w4(x, w, bias)
    err = (got.double() - y).abs()
    assert torch.isfinite(got).all()
    assert (err <= tol).all(), f"worst {(err / tol).max():.2f} of the bound"
    for off in (0, 1, 8):
        wide = torch.full((m, k + 24), float("nan"), dtype=x.dtype, device="cuda")
        wide[:, off:off + k] = x
        view = wide[:, off:off + k]
        if dtype == "f32" and m > 8:   # the fp32 product picks its kernel by alignment
            assert ((ext.matrix_mul_w4(view, w, bias).double() - y).abs() <= tol).all()
        else:
            assert torch.equal(ext.matrix_mul_w4(view, w, bias), got)
    assert torch.equal(ext.matrix_mul_w4(x, w, bias), got)
    ext.check_device()


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("m", [1, 2, 5, 8])
def test_outliers_that_meet_no_weight(m, dtype):
    """x in digits is held to 2^-30 of its block's largest magnitude, whatever weight that meets:
    one element of each block is up to 2^20 times the others and its codes are the zero point, so
    that only what is held of the others counts."""
    x, codes, scales, zeros, _ = _make(m, 500, 1000, 128, dtype)
    x[:, 5::128] *= torch.tensor([2.0 ** 14, 2.0 ** 20, 1.0, 2.0 ** 8] * 2)[:len(x[0, 5::128])].to(x.dtype).clamp(
        max=2.0 ** 12 if dtype == "f16" else 2.0 ** 20)
    codes[:, 5::128] = zeros[:, :codes[:, 5::128].shape[1]]
    w64 = _weight64(codes, scales, zeros, 128).cuda()
    y = x.cuda().double() @ w64.t()
    got = ext.matrix_mul_w4(x.cuda(), ext.pack_w4(codes, scales, zeros, 128).to("cuda"))
    assert ((got.double() - y).abs() <= _long_bound(x.cuda(), w64, y, dtype, 1000, 128)).all()


@gpu
@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("m,dtype,top", [(1, "f32", 2.0 ** 13), (1, "f32", 2.0 ** 24), (2, "f32", 2.0 ** 20),
                                         (3, "f32", 2.0 ** 24), (5, "f32", 2.0 ** 40), (8, "f32", 2.0 ** 20),
                                         (8, "f32", 2.0 ** 100), (1, "bf16", 2.0 ** 15), (1, "f16", 2.0 ** 5),
                                         (2, "bf16", 2.0 ** 100), (8, "f16", 2.0 ** 12)])
def test_large_elements_cost_the_others_no_digits(m, dtype, top, group):
    """Each block of x has an element of `top` times the others' size whose codes are the zero point.
    The bound is relative to sum |x w|, in which it does not appear: every element of x counts with
    all its bits (fp32), or all that its output keeps."""
    x, codes, scales, zeros, _ = _make(m, 300, 2500, group, dtype)
    x[:, 7::32] = top
    codes[:, 7::32] = zeros.repeat_interleave(group // 32, 1)[:, :codes[:, 7::32].shape[1]]
    x, codes, scales, zeros = (t.cuda() for t in (x, codes, scales, zeros))
    w64 = _weight64(codes, scales, zeros, group)
    y = x.double() @ w64.t()
    got = ext.matrix_mul_w4(x, ext.pack_w4(codes, scales, zeros, group))
    s = x.double().abs() @ w64.abs().t()
    tol = ((-(-2500 // min(group, 128)) + 40) * 2.0 ** -24 + 2.0 ** -19) * s + 1.001 * U[dtype] * y.abs() + (
        2.0 ** -25 if dtype == "f16" else 0.0)
    assert ((got.double() - y).abs() <= tol).all(), f"{((got.double() - y).abs() / tol).max():.1f} of the bound"


def _huge(m, dtype, sdtype=None):
    """One element of x near the type's largest per row and block; with its weight the result is far
    from it, but codes times x, before the scale, are past fp32."""
    x, codes, scales, zeros, _ = _make(m, 150, 384, 64, dtype, sdtype=sdtype)
    x[:, 70::128] = 0.99 * torch.finfo(DT[dtype]).max * (torch.arange(m)[:, None] % 2 * 2 - 1)
    x[:, 71::128] = -x[:, 70::128] / 2
    return x, codes, (scales / 64).to(scales.dtype), zeros


@gpu
@pytest.mark.parametrize("m", [1, 2, 3, 8])
def test_huge_fp32_x_overflows_no_sum(m):
    x, codes, scales, zeros = _huge(m, "f32")
    _check(x, codes, scales, zeros, None, 64, "f32")


@gpu
@pytest.mark.parametrize("m,sdtype", [(1, "bf16"), (2, "bf16"), (3, "f32"), (8, "bf16"), (16, "f32"), (17, "bf16"),
                                      (40, "f32")])
def test_huge_bf16_x_overflows_no_sum(m, sdtype):
    x, codes, scales, zeros = _huge(m, "bf16", sdtype)
    _check(x, codes, scales, zeros, None, 64, "bf16")


@gpu
@pytest.mark.parametrize("m,n,k,dtype,top", [(1, 300, 2500, "bf16", 2.0 ** 30), (1, 300, 2500, "bf16", 2.0 ** 110),
                                             (1, 40005, 2500, "f16", 2.0 ** 15), (1, 2500, 40000, "bf16", 2.0 ** 23),
                                             (2, 9000, 16000, "bf16", 2.0 ** 40), (2, 9000, 16000, "f16", 2.0 ** 13),
                                             (1, 37, 300, "bf16", 2.0 ** 127)])
@pytest.mark.parametrize("few", [True, False])
def test_large_elements_beside_small_ones_in_16_bits(m, n, k, dtype, top, few):
    """The digits of one or two 16-bit rows hold 30 bits below a block's largest magnitude; what they
    leave out of a few elements, or of all, counts all the same.  Repeats give the same bits."""
    x, codes, scales, zeros, _ = _make(m, n, k, 64, dtype)
    if few:      # one block in five, most of whose elements are zeros, with a large one
        x.view(-1)[torch.rand(m * k, generator=torch.Generator().manual_seed(8)) < 0.97] = 0
    x[:, 7::640 if few else 32] = top
    x[:, 9::64] *= 2.0 ** -10
    codes[:, 7::32] = zeros.repeat_interleave(2, 1)[:, :codes[:, 7::32].shape[1]]
    x, codes, scales, zeros = (t.cuda() for t in (x, codes, scales, zeros))
    w64 = _weight64(codes, scales, zeros, 64)
    y = x.double() @ w64.t()
    w = ext.pack_w4(codes, scales, zeros, 64)
    got = ext.matrix_mul_w4(x, w)
    s = x.double().abs() @ w64.abs().t()
    # group sums (and, one by one, elements) added in fp32 in any order, 2^-24 S each at worst
    tol = ((k if not few else -(-k // 64) + 110) * 2.0 ** -24 + 2.0 ** -19) * s + 1.001 * U[dtype] * y.abs() + (
        2.0 ** -25 if dtype == "f16" else 0.0)
    assert ((got.double() - y).abs() <= tol).all(), f"{((got.double() - y).abs() / tol).max():.1f} of the bound"
    for _ in range(3):
        assert torch.equal(ext.matrix_mul_w4(x, w), got)


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("m", [1, 2, 4, 8, 13])
def test_not_finite_rows_follow_the_formula(m, dtype):
    """x infinite at one place gives the sign of that weight (NaN where it is zero), NaN gives NaN, and
    a huge finite row beside them its product."""
    if m > 8 and dtype == "f32":
        pytest.skip("from 9 rows on the fp32 product splits infinities")
    x, codes, scales, zeros = _huge(max(m, 4), dtype, "f32")
    w64 = _weight64(codes, scales, zeros, 64)
    w = ext.pack_w4(codes, scales, zeros, 64).to("cuda")
    nan, inf = x[1:2].clone(), _make(1, 150, 384, 64, dtype)[0]
    nan[0, 200], inf[0, 77] = float("nan"), float("-inf")
    for batch in ([nan, inf, x[:1], x[2:3]] * 4, [x[:1], inf, nan, x[3:4]] * 4, [inf] * 16, [nan] * 16):
        batch = torch.cat(batch)[:m]
        got = ext.matrix_mul_w4(batch.cuda(), w).cpu().double()
        for row, out in zip(batch, got):
            if torch.isnan(row).any():
                assert torch.isnan(out).all()
            elif torch.isinf(row).any():
                sign = -torch.sign(w64[:, 77])
                assert torch.equal(torch.isnan(out), sign == 0) and (out[sign != 0] == sign[sign != 0] * float("inf")).all()
            else:
                y = w64 @ row.double()
                tol = _bound(row[None], w64, y[None], dtype, 1)[0] if m <= 8 else 2.0 ** -13 * y.abs() + _bound(
                    row[None], w64, y[None], dtype, 9)[0]
                assert ((out - y).abs() <= tol).all()


@gpu
def test_a_nan_row_costs_the_batch_little():
    """A row of a batch that is not finite (a padded one, say) is not computed one output at a time:
    the call takes less than eight times the finite one (one at a time: some twenty times)."""
    g = torch.Generator(device="cuda").manual_seed(3)
    codes = torch.randint(0, 16, (8192, 8192), device="cuda", generator=g, dtype=torch.uint8)
    w = ext.pack_w4(codes, torch.rand(8192, 64, device="cuda", generator=g).bfloat16())
    x = torch.randn(8, 8192, device="cuda", generator=g).bfloat16()
    bad = x.clone()
    bad[3, 4000] = float("nan")

    def best(t):
        times = []
        for _ in range(20):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(4):
                ext.matrix_mul_w4(t, w)
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)

    assert best(bad) <= 8 * best(x)
