"""Block-scaled 8-bit operators on the GPU against plain implementations in 64 bits.

Tolerances, from the arithmetic:

* Quantisation is compared bit for bit: scales and quotients are correctly rounded fp32 divisions on
  both sides.
* Products.  The products of two e4m3 codes are exact in fp32 (4 + 4 significand bits).  A 128-wide
  step sums 128 of them and the steps are joined by fused multiply-adds of sums and scales, so with
  n = 128 + steps additions of at most one fp32 ulp (2^-23) each, and three more roundings for the
  scales' product, |error| <= (n + 3) 2^-23 sum |x w|.  Then half a step of the output type.
* The gated MLP's h is a product's output through the activation: its error follows from the gate's
  and the up product's, plus 2^-18 |h| for the exponential and the division.  A code of h is one of
  those between e4m3((h - e) / s) and e4m3((h + e) / s), e that error and s the scale, itself off by
  the error of the block's largest |h|; the spread of these codes goes through the down product.
"""

import pytest
import torch

gpu = pytest.mark.gpu
DEV = "cuda:0"


def _nat():
    from distributedmoe_b200 import _native as N
    return N


# ------------------------------------------------------------------------------- in 64 bits
def _blocks(n):
    return -(-n // 128)


def _e4m3(v):
    """Nearest e4m3 value, ties to even: eight steps to a power of two, none finer than 2^-9."""
    e = torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -30))).clamp_min(-6.0)
    step = torch.exp2(e - 3.0)
    return (torch.round(v / step) * step).clamp(-448.0, 448.0)


def _quantize64(x, block_rows=1):
    """(codes, scales) in float64 of a matrix of numbers of at most 32 bits."""
    x = x.double()
    rows, cols = x.shape
    R, C = -(-rows // block_rows), _blocks(cols)
    p = torch.zeros(R * block_rows, C * 128, dtype=torch.float64, device=x.device)
    p[:rows, :cols] = x
    b = p.view(R, block_rows, C, 128)
    fine = torch.isfinite(b)
    amax = torch.where(fine, b.abs(), 0.0).amax(dim=(1, 3))
    s = torch.where(amax > 0, (amax / 448).clamp_min(2.0 ** -126), 1.0).float().double()
    q = _e4m3((b / s[:, None, :, None]).float().double())
    q = torch.where(fine, q, float("nan"))
    return q.view(R * block_rows, C * 128)[:rows, :cols], s


def _spread(s, shape, block_rows):
    """Block scales over the elements they belong to."""
    s = s.double().repeat_interleave(128, dim=-1)[..., :shape[-1]]
    return s if block_rows == 1 else s.repeat_interleave(block_rows, dim=-2)[..., :shape[-2], :]


def _values(q, s, block_rows):
    return q.double() * _spread(s, q.shape, block_rows)


def _check(out, want, slack, eps):
    """|out - want| <= slack + half a step of the output type (eps: its epsilon)."""
    assert out.shape == want.shape
    off = (out.double() - want).abs() - (slack + eps / 2 * (want.abs() + slack))
    assert bool(torch.isfinite(out.double()).all())
    assert off.max().item() <= 0, f"off by {off.max().item():.3e} more than allowed"


def _product_slack(xa, wa):
    """Error bound of a product of matrices with these absolute values."""
    n = 128 + _blocks(xa.shape[1]) + 3
    return n * 2.0 ** -23 * (xa @ wa.T)


# ------------------------------------------------------------------------------- quantisation
def _hard_rows(rows, cols, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(rows, cols, generator=g, device=DEV)
    x = x * torch.exp2(torch.randint(-20, 12, (rows, 1), generator=g, device=DEV).float())
    x[rows // 2] = 0.0
    if rows > 3:
        x[1, cols // 2] = 6e4
        x[2, : min(16, cols)] = torch.finfo(dtype).tiny / 4  # subnormal in its type
        x[2, min(16, cols):] = 0.0
    return x.to(dtype)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(1, 16), (5, 144), (37, 1040), (130, 2064), (300, 4096)])
def test_quantize_rows_bit_for_bit(dtype, rows, cols):
    N = _nat()
    x = _hard_rows(rows, cols, dtype, rows + cols)
    q, s = N.quantize_blocks_e4m3(x)
    rq, rs = _quantize64(x)
    assert s.shape == (rows, _blocks(cols)) and torch.equal(s.double(), rs)
    assert q.dtype == torch.float8_e4m3fn and torch.equal(q.double(), rq)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 16), (127, 144), (129, 256), (3, 200, 400), (2, 2, 256, 128)])
def test_quantize_squares_bit_for_bit(dtype, shape):
    N = _nat()
    flat = _hard_rows(torch.Size(shape[:-1]).numel(), shape[-1], dtype, 7)
    x = flat.view(shape)
    q, s = N.quantize_blocks_e4m3(x, block_rows=128)
    assert s.shape == (*shape[:-2], _blocks(shape[-2]), _blocks(shape[-1]))
    for m, (qm, sm) in zip(x.reshape(-1, *shape[-2:]), zip(q.reshape(-1, *shape[-2:]), s.reshape(-1, *s.shape[-2:]))):
        rq, rs = _quantize64(m, 128)
        assert torch.equal(sm.double(), rs) and torch.equal(qm.double(), rq)


@gpu
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_what_is_not_finite(block_rows):
    """Infinities and NaN become NaN codes; the scale and the other codes of the block are as
    without them."""
    N = _nat()
    x = torch.randn(200, 384, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV)
    x[0, 5], x[70, 200], x[150, 383] = float("inf"), float("-inf"), float("nan")
    x[199] = float("nan")
    q, s = N.quantize_blocks_e4m3(x, block_rows)
    rq, rs = _quantize64(x, block_rows)
    assert torch.equal(s.double(), rs)
    assert torch.equal(q.double().isnan(), ~x.isfinite())
    assert torch.equal(q.double().nan_to_num(9.0), rq.nan_to_num(9.0))


@gpu
def test_quantize_every_16_bit_value():
    """All finite bf16 and f16 values under a spread of block maxima: the divisions are the
    correctly rounded ones."""
    N = _nat()
    bits = torch.arange(-2**15, 2**15, device=DEV).to(torch.int16)
    for dtype in (torch.bfloat16, torch.float16):
        v = bits.view(dtype)
        v = v[v.isfinite()]
        v = v[torch.argsort(v.abs().float())]
        v = v[:v.numel() // 128 * 128].view(-1, 128)
        for a, b in ((0, 128), (8, 120)):
            x = v[:, a:b].contiguous()
            q, s = N.quantize_blocks_e4m3(x)
            rq, rs = _quantize64(x)
            assert torch.equal(s.double(), rs) and torch.equal(q.double(), rq)


@gpu
def test_quantize_past_32_bit_offsets():
    N = _nat()
    cols = 8192
    rows = 2**32 // cols + 3
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device=DEV)
    tail = torch.randn(5, cols, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).to(torch.bfloat16)
    x[-5:] = tail
    q, s = N.quantize_blocks_e4m3(x)
    rq, rs = _quantize64(tail)
    assert torch.equal(q[-5:].double(), rq) and torch.equal(s[-5:].double(), rs)
    q2, s2 = N.quantize_blocks_e4m3(x, 128)
    assert int((s2[:-2] != 1).sum()) == 0
    assert torch.equal(q2[-4:].float().abs().amax() > 400, torch.tensor(True, device=DEV))
    del x, q, q2


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_widest_row(dtype):
    N = _nat()
    cols = 65535 * 1024 if dtype == torch.float32 else 2**26
    x = torch.zeros(2, cols, dtype=dtype, device=DEV)
    tail = torch.randn(2, 512, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).to(dtype)
    x[:, -512:] = tail
    q, s = N.quantize_blocks_e4m3(x)
    rq, rs = _quantize64(tail)
    assert torch.equal(q[:, -512:].double(), rq) and torch.equal(s[:, -4:].double(), rs)
    assert int(q[:, :-512].view(torch.uint8).count_nonzero()) == 0 and bool((s[:, :-4] == 1).all())
    with pytest.raises(N.DMoEError, match="columns|2.26"):
        N.quantize_blocks_e4m3(torch.zeros(1, cols + 16, dtype=dtype, device=DEV))


# ------------------------------------------------------------------------------- products
def _operands(seed, rows, E, Nn, K):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(rows, K, generator=g, device=DEV) * torch.exp(torch.randn(rows, 1, generator=g, device=DEV))
    w = torch.randn(E, Nn, K, generator=g, device=DEV) * 0.02 * torch.exp(torch.randn(E, Nn, 1, generator=g, device=DEV))
    N = _nat()
    return (*N.quantize_blocks_e4m3(x), *N.quantize_blocks_e4m3(w, 128))


def _table(sizes):
    ends, at = [], 0
    for n in sizes:
        at += n
        ends.append(at)
    return ends


def _product_cases():
    # (weights, N, K, rows of each segment, rows behind the last): every tile shape, segments of no
    # row, of one, longer than a tile and than several; N and K that end inside a block
    yield 1, 8, 16, [1], 0
    yield 1, 136, 144, [1], 3
    yield 1, 512, 4096, [1], 0       # few tiles, long reduction: split over a cluster
    yield 1, 264, 1040, [7], 0
    yield 3, 200, 400, [0, 5, 1, 0, 2], 4
    yield 4, 384, 2064, [17, 1, 0, 40], 0
    yield 4, 392, 272, [30, 33, 20, 31], 1
    yield 3, 640, 528, [64, 1, 70], 2
    yield 5, 256, 128, [60, 33, 129, 0, 3], 0
    yield 2, 904, 1168, [128, 65], 7
    yield 3, 264, 656, [100, 300, 20], 0
    yield 3, 776, 1296, [257, 1, 255], 5
    yield 6, 512, 384, [600, 0, 129, 256, 131, 400], 9
    yield 1, 1000, 2064, [77], 0


@gpu
@pytest.mark.parametrize("device_table", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("case", list(_product_cases()), ids=lambda c: f"E{c[0]}N{c[1]}K{c[2]}r{sum(c[3])}s{len(c[3])}")
def test_product(case, dtype, device_table):
    N = _nat()
    E, Nn, K, sizes, behind = case
    rows = sum(sizes) + behind
    xq, xs, wq, ws = _operands(Nn + K, rows, E, Nn, K)
    experts = [(7 * i + 1) % E for i in range(len(sizes))]
    ends = _table(sizes)
    table = (torch.tensor(experts, dtype=torch.int32, device=DEV), torch.tensor(ends, dtype=torch.int32, device=DEV)) \
        if device_table else (experts, ends)
    out = torch.full((rows, Nn), 7.0, dtype=dtype, device=DEV)
    got = N.grouped_matmul_fp8_blocks(xq, xs, wq, ws, *table, out)
    assert got is out
    x, w = _values(xq, xs, 1), _values(wq, ws, 128)
    a = 0
    for e, b in zip(experts, ends):
        if b > a:
            _check(out[a:b], x[a:b] @ w[e].T, _product_slack(x[a:b].abs(), w[e].abs()), torch.finfo(dtype).eps)
        a = b
    assert bool((out[a:] == 7.0).all()), "rows behind the last segment stay as they were"
    N.check_device_status(torch.device(DEV))


# Rows of three or more segments over 40 tiles of weights and a reduction of 49 blocks: 160 or 200 tiles
# on 148 SMs, whose last wave is split over pairs of SMs, and 240, whose last wave is too full for it.
_LAST_WAVES = [[33, 20, 1], [65, 20, 30], [129, 0, 259], [33, 33, 1, 1]]


@gpu
@pytest.mark.parametrize("device_table", [False, True])
@pytest.mark.parametrize("sizes", _LAST_WAVES, ids=lambda s: "r" + "_".join(map(str, s)))
def test_product_last_wave(sizes, device_table):
    """Whole tiles first, then parts of the last ones: twice the same bits, rows behind untouched."""
    N = _nat()
    E, Nn, K, rows = 2, 10232, 6160, sum(sizes) + 3
    xq, xs, wq, ws = _operands(3, rows, E, Nn, K)
    experts, ends = [i % E for i in range(len(sizes))], _table(sizes)
    table = (torch.tensor(experts, dtype=torch.int32, device=DEV), torch.tensor(ends, dtype=torch.int32, device=DEV)) \
        if device_table else (experts, ends)
    out = torch.full((rows, Nn), 7.0, dtype=torch.float32, device=DEV)
    N.grouped_matmul_fp8_blocks(xq, xs, wq, ws, *table, out)
    x, w = _values(xq, xs, 1), _values(wq, ws, 128)
    a = 0
    for e, b in zip(experts, ends):
        if b > a:
            _check(out[a:b], x[a:b] @ w[e].T, _product_slack(x[a:b].abs(), w[e].abs()), 2.0 ** -23)
        a = b
    assert bool((out[a:] == 7.0).all()), "rows behind the last segment stay as they were"
    assert torch.equal(N.grouped_matmul_fp8_blocks(xq, xs, wq, ws, *table, out_dtype=torch.float32)[:a], out[:a])
    N.check_device_status(torch.device(DEV))


@gpu
@pytest.mark.parametrize("sizes", _LAST_WAVES, ids=lambda s: "r" + "_".join(map(str, s)))
def test_gated_mlp_last_wave(sizes):
    N = _nat()
    E, d, I, rows = 2, 6160, 5120, sum(sizes)
    xq, xs, gq, gs = _operands(4, rows, E, I, d)
    _, _, uq, us = _operands(5, 1, E, I, d)
    _, _, dq, dsc = _operands(6, 1, E, d, I)
    ex = N.Fp8BlockExperts.from_quantized(gq, gs, uq, us, dq, dsc)
    experts, ends = [i % E for i in range(len(sizes))], _table(sizes)
    Y = N.grouped_gated_mlp_fp8_blocks(xq, xs, ex, experts, ends, N.ACT_SILU)
    assert torch.equal(Y, N.grouped_gated_mlp_fp8_blocks(xq, xs, ex, experts, ends, N.ACT_SILU))
    x = _values(xq, xs, 1)
    wg, wu, wd = _values(gq, gs, 128), _values(uq, us, 128), _values(dq, dsc, 128)
    a = 0
    for e, b in zip(experts, ends):
        if b > a:
            want, slack = _mlp_reference(x[a:b], wg[e], wu[e], wd[e], True)
            _check(Y[a:b], want, slack, 2.0 ** -7)
        a = b
    N.check_device_status(torch.device(DEV))


@gpu
@pytest.mark.parametrize("hint", [1, 17, 40, 100, 200])
def test_product_any_tile_shape_for_any_rows(hint):
    """rows_hint picks the tiles, not the result: wrong guesses in both directions."""
    N = _nat()
    E, Nn, K, sizes = 3, 520, 784, [1, 333, 0, 90]
    xq, xs, wq, ws = _operands(5, sum(sizes), E, Nn, K)
    experts, ends = [2, 0, 1, 2], _table(sizes)
    out = N.grouped_matmul_fp8_blocks(xq, xs, wq, ws, experts, ends, rows_hint=hint, out_dtype=torch.float32)
    x, w = _values(xq, xs, 1), _values(wq, ws, 128)
    a = 0
    for e, b in zip(experts, ends):
        if b > a:
            _check(out[a:b], x[a:b] @ w[e].T, _product_slack(x[a:b].abs(), w[e].abs()), 2.0 ** -23)
        a = b
    N.check_device_status(torch.device(DEV))


@gpu
@pytest.mark.parametrize("device_table", [False, True])
def test_product_of_the_largest_hint(device_table):
    """rows_hint may be any number: one past the rows is as good as the rows."""
    N = _nat()
    xq, xs, wq, ws = _operands(5, 90, 2, 520, 784)
    table = ([1, 0], [40, 90])
    if device_table:
        table = tuple(torch.tensor(v, dtype=torch.int32, device=DEV) for v in table)
    want = N.grouped_matmul_fp8_blocks(xq, xs, wq, ws, *table, rows_hint=90, out_dtype=torch.float32)
    for hint in (91, 2**30, 2**31 - 1):
        assert torch.equal(want, N.grouped_matmul_fp8_blocks(xq, xs, wq, ws, *table, rows_hint=hint, out_dtype=torch.float32))
    x, w = _values(xq, xs, 1), _values(wq, ws, 128)
    for part, e in ((slice(0, 40), 1), (slice(40, 90), 0)):
        _check(want[part], x[part] @ w[e].T, _product_slack(x[part].abs(), w[e].abs()), 2.0 ** -23)
    N.check_device_status(torch.device(DEV))


@gpu
@pytest.mark.parametrize("rows", [1, 16, 100, 200])
def test_matmul_strided_rows(rows):
    """Codes, scales and output whose rows are parts of wider rows."""
    N = _nat()
    Nn, K = 264, 400
    xq, xs, wq, ws = _operands(11, rows, 1, Nn, K)
    wide_q = torch.full((rows, K + 48), 0x7F, dtype=torch.uint8, device=DEV)  # NaN codes behind each row
    wide_q[:, :K] = xq.view(torch.uint8)
    wide_s = torch.full((rows, 9), float("nan"), device=DEV)
    wide_s[:, 2:2 + xs.shape[1]] = xs
    wide_y = torch.full((rows, Nn + 24), 5.0, dtype=torch.bfloat16, device=DEV)
    y = N.matmul_fp8_blocks(wide_q[:, :K].view(torch.float8_e4m3fn), wide_s[:, 2:2 + xs.shape[1]], wq[0], ws[0],
                            wide_y[:, :Nn])
    assert torch.equal(y, N.matmul_fp8_blocks(xq, xs, wq[0], ws[0]))
    assert bool((wide_y[:, Nn:] == 5.0).all())
    x, w = _values(xq, xs, 1), _values(wq, ws, 128)[0]
    _check(y, x @ w.T, _product_slack(x.abs(), w.abs()), 2.0 ** -7)


# Rows, output columns and K that reach each kernel and a split tile.
_KERNELS = {"whole": (5, 264, 400), "split": (3, 512, 4096), "single": (200, 264, 400), "pair": (600, 264, 400)}


@gpu
@pytest.mark.parametrize("rows,Nn,K", _KERNELS.values(), ids=_KERNELS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_product_of_scales_out_of_range(rows, Nn, K, dtype):
    """The product of two scales may be below the smallest normal number or past the largest while a step's
    sum times it is neither: codes reach from 2^-18 to 2^25 a step.  What fp32 holds of a result below
    2^-126 is a multiple of 2^-149, for each addition."""
    N = _nat()
    xq, xs, wq, ws = _operands(3, rows, 1, Nn, K)
    wq, ws = wq[0], ws[0].clone()
    xs = torch.full_like(xs, 2.0 ** -70) * (1 + torch.rand(xs.shape, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV))
    ws[:] = 1.3 * 2.0 ** -66
    ws[1] = 1.7 * 2.0 ** -75        # results that are subnormal themselves
    ws[-1, 1:] = 1.1 * 2.0 ** -40   # a column block with both kinds of steps
    xs[0] = 3e38
    xq.view(torch.uint8)[0] = 0     # the largest scale over nothing but zeros
    xs[1] = 2.0 ** 110              # past the largest number times ws[0] ..
    xq.view(torch.uint8)[1] = 0
    xq.view(torch.uint8)[1, 3] = 1  # .. the smallest code (2^-9) alone,
    wq.view(torch.uint8)[:, 3] = 1  # on both sides
    for scale in (ws, ws * 2.0 ** 100):
        x, w = _values(xq, xs, 1), _values(wq, scale, 128)
        y = N.matmul_fp8_blocks(xq, xs, wq, scale, out_dtype=dtype)
        want, slack = x @ w.T, _product_slack(x.abs(), w.abs()) + (_blocks(K) + 1) * 2.0 ** -149
        assert bool((y[0] == 0).all())
        small = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps  # a step of the output's subnormals
        _check(y, want, slack + small / 2, torch.finfo(dtype).eps)
    N.check_device_status(torch.device(DEV))


@gpu
@pytest.mark.parametrize("rows,I,d", _KERNELS.values(), ids=_KERNELS)
@pytest.mark.parametrize("silu", [True, False])
def test_gated_mlp_product_of_scales_out_of_range(rows, I, d, silu):
    """Gate sums near 2^-118, whose products of scales are below 2^-126, and up sums near 2^67 with one
    such step: h is an ordinary number."""
    N = _nat()
    I = I // 16 * 16
    xq, xs, gq, gs = _operands(1, rows, 1, I, d)
    _, _, uq, us = _operands(2, 1, 1, I, d)
    _, _, dq, dsc = _operands(3, 1, 1, d, I)
    xs[:] = 2.0 ** -70 * (1 + torch.rand(xs.shape, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV))
    gs[:] = 1.3 * 2.0 ** -64
    us[:] = 1.1 * 2.0 ** 120
    us[:, 0, 0] = 1.2 * 2.0 ** -60  # a block that adds next to nothing
    xs[1] = 2.0 ** 40               # this row's up scales pass the largest number, over zeros
    xq.view(torch.uint8)[1] = 0
    ex = N.Fp8BlockExperts.from_quantized(gq, gs, uq, us, dq, dsc)
    Y = N.grouped_gated_mlp_fp8_blocks(xq, xs, ex, [0], [rows], N.ACT_SILU if silu else N.ACT_RELU)
    x = _values(xq, xs, 1)
    want, slack = _mlp_reference(x, _values(gq, gs, 128)[0], _values(uq, us, 128)[0], _values(dq, dsc, 128)[0], silu)
    assert bool((Y[1] == 0).all())
    _check(Y, want, slack, 2.0 ** -7)
    N.check_device_status(torch.device(DEV))


@gpu
@pytest.mark.parametrize("rows", [3, 40, 200])
def test_product_keeps_nan_in_its_row(rows):
    N = _nat()
    Nn, K = 264, 400
    xq, xs, wq, ws = _operands(2, rows, 1, Nn, K)
    clean = N.matmul_fp8_blocks(xq, xs, wq[0], ws[0])
    xq.view(torch.uint8)[1, 130] = 0x7F
    xs[2, 1] = float("inf")
    y = N.matmul_fp8_blocks(xq, xs, wq[0], ws[0])
    assert bool(y[1].isnan().all()) and not bool(y[2].isfinite().all())
    keep = [r for r in range(rows) if r not in (1, 2)]
    assert torch.equal(y[keep], clean[keep])


@gpu
def test_product_weights_past_32_bit_offsets():
    N = _nat()
    E, Nn, K = 70, 8192, 8192
    wq = torch.zeros(E, Nn, K, dtype=torch.uint8, device=DEV)
    xq, xs, w1, s1 = _operands(4, 5, 1, Nn, K)
    wq[E - 1] = w1.view(torch.uint8)[0]
    ws = torch.ones(E, 64, 64, device=DEV)
    ws[E - 1] = s1[0]
    y = N.grouped_matmul_fp8_blocks(xq, xs, wq.view(torch.float8_e4m3fn), ws, [E - 1, 0], [4, 5], out_dtype=torch.float32)
    x, w = _values(xq, xs, 1), _values(w1, s1, 128)[0]
    _check(y[:4], x[:4] @ w.T, _product_slack(x[:4].abs(), w.abs()), 2.0 ** -23)
    assert int(y[4].count_nonzero()) == 0


@gpu
def test_product_rows_past_32_bit_offsets():
    """Row offsets of codes and output past 2^32 bytes, through both kernels."""
    N = _nat()
    Nn, K, rows = 8200, 16, 2**32 // (2 * 8200) + 200
    _, _, wq, ws = _operands(6, 1, 1, Nn, K)
    g = torch.Generator(device=DEV).manual_seed(1)
    xq, xs = N.quantize_blocks_e4m3(torch.randn(rows, K, generator=g, device=DEV))
    w = _values(wq, ws, 128)[0]
    for hint in (0, 100):
        y = N.grouped_matmul_fp8_blocks(xq, xs, wq, ws, [0], [rows], rows_hint=hint)
        for part in (slice(0, 3), slice(rows - 150, rows)):
            x = _values(xq[part], xs[part], 1)
            _check(y[part], x @ w.T, _product_slack(x.abs(), w.abs()), 2.0 ** -7)
        del y


# ------------------------------------------------------------------------------- the gated MLP
def _mlp_reference(x, wg, wu, wd, silu):
    """(y, allowed error) for one segment, operands in 64 bits."""
    g, u = x @ wg.T, x @ wu.T
    dg, du = _product_slack(x.abs(), wg.abs()), _product_slack(x.abs(), wu.abs())
    act = g * torch.sigmoid(g) if silu else g.clamp_min(0.0)
    h = act * u
    eh = 1.1 * dg * u.abs() + act.abs() * du + 1.1 * dg * du + 2.0 ** -18 * h.abs()  # |silu'| < 1.1
    rows, I = h.shape
    pad = _blocks(I) * 128 - I
    hb = torch.nn.functional.pad(h, (0, pad)).view(rows, -1, 128)
    eb = torch.nn.functional.pad(eh, (0, pad)).view(rows, -1, 128)
    amax = hb.abs().amax(2, keepdim=True)
    s = torch.where(amax > 0, (amax / 448).clamp_min(2.0 ** -126), 1.0)
    # the scale may be off by the error of the block's largest value, and by a rounding
    ds = torch.where(amax > 0, eb.amax(2, keepdim=True) / amax.clamp_min(1e-300), 0.0) + 2.0 ** -22
    far = (hb.abs() * ds + eb) / s * (1 + 2.0 ** -10)
    v = hb / s
    low, mid, high = _e4m3(v - far), _e4m3(v), _e4m3(v + far)
    hq = (mid * s).reshape(rows, -1)[:, :I]
    dh = (torch.maximum(high - mid, mid - low) * s + mid.abs() * s * ds).reshape(rows, -1)[:, :I]
    y = hq @ wd.T
    return y, _product_slack(hq.abs() + dh, wd.abs()) + dh @ wd.abs().T


def _mlp_cases():
    yield 1, 16, 16, [1], 0
    yield 2, 128, 128, [3], 1
    yield 4, 2048, 768, [1, 1, 0, 1], 0   # few tiles: split over a cluster
    yield 5, 208, 336, [1, 0, 20, 9, 4], 2
    yield 3, 400, 656, [20, 33, 31], 0
    yield 3, 272, 528, [70, 1, 64], 0
    yield 3, 256, 272, [128, 90, 100], 6
    yield 4, 528, 400, [300, 129, 0, 257], 3
    yield 2, 1024, 768, [511, 260], 0


@gpu
@pytest.mark.parametrize("silu", [True, False])
@pytest.mark.parametrize("case", list(_mlp_cases()), ids=lambda c: f"E{c[0]}d{c[1]}I{c[2]}r{sum(c[3])}s{len(c[3])}")
def test_gated_mlp(case, silu):
    N = _nat()
    E, d, I, sizes, behind = case
    rows = sum(sizes) + behind
    xq, xs, gq, gs = _operands(d + I, rows, E, I, d)
    _, _, uq, us = _operands(d + I + 1, 1, E, I, d)
    _, _, dq, dsc = _operands(d + I + 2, 1, E, d, I)
    ex = N.Fp8BlockExperts.from_quantized(gq, gs, uq, us, dq, dsc)
    experts, ends = [(3 * i + 1) % E for i in range(len(sizes))], _table(sizes)
    Y = torch.full((rows, d), 7.0, dtype=torch.bfloat16, device=DEV)
    act = N.ACT_SILU if silu else N.ACT_RELU
    N.grouped_gated_mlp_fp8_blocks(xq, xs, ex, experts, ends, act, Y)
    N.check_device_status(torch.device(DEV))
    x = _values(xq, xs, 1)
    wg, wu, wd = _values(gq, gs, 128), _values(uq, us, 128), _values(dq, dsc, 128)
    a = 0
    for e, b in zip(experts, ends):
        if b > a:
            want, slack = _mlp_reference(x[a:b], wg[e], wu[e], wd[e], silu)
            _check(Y[a:b], want, slack, 2.0 ** -7)
        a = b
    assert bool((Y[a:] == 7.0).all()), "rows behind the last segment stay as they were"
    again = N.grouped_gated_mlp_fp8_blocks(xq, xs, ex, torch.tensor(experts, dtype=torch.int32, device=DEV),
                                           torch.tensor(ends, dtype=torch.int32, device=DEV), act)
    if a:
        assert bool((again[:a].double() - Y[:a].double()).abs().max() <= 0.05 * Y[:a].double().abs().max())


@gpu
@pytest.mark.parametrize("hint", [0, 17, 100, 200])
@pytest.mark.parametrize("case", list(_mlp_cases()), ids=lambda c: f"E{c[0]}d{c[1]}I{c[2]}r{sum(c[3])}s{len(c[3])}")
def test_gated_mlp_device_table(case, hint):
    """A table on the device has its own choice of tiles: each element against the definition, as a host
    table's."""
    N = _nat()
    E, d, I, sizes, behind = case
    rows = sum(sizes) + behind
    xq, xs, gq, gs = _operands(d + I, rows, E, I, d)
    _, _, uq, us = _operands(d + I + 1, 1, E, I, d)
    _, _, dq, dsc = _operands(d + I + 2, 1, E, d, I)
    ex = N.Fp8BlockExperts.from_quantized(gq, gs, uq, us, dq, dsc)
    experts, ends = [(3 * i + 1) % E for i in range(len(sizes))], _table(sizes)
    Y = torch.full((rows, d), 7.0, dtype=torch.bfloat16, device=DEV)
    N.grouped_gated_mlp_fp8_blocks(xq, xs, ex, torch.tensor(experts, dtype=torch.int32, device=DEV),
                                   torch.tensor(ends, dtype=torch.int32, device=DEV), N.ACT_SILU, Y, rows_hint=hint)
    x = _values(xq, xs, 1)
    wg, wu, wd = _values(gq, gs, 128), _values(uq, us, 128), _values(dq, dsc, 128)
    a = 0
    for e, b in zip(experts, ends):
        if b > a:
            want, slack = _mlp_reference(x[a:b], wg[e], wu[e], wd[e], True)
            _check(Y[a:b], want, slack, 2.0 ** -7)
        a = b
    assert bool((Y[a:] == 7.0).all()), "rows behind the last segment stay as they were"
    N.check_device_status(torch.device(DEV))


@gpu
def test_gated_mlp_what_is_not_finite_stays_in_its_row():
    N = _nat()
    for rows in (5, 200):
        xq, xs, gq, gs = _operands(1, rows, 1, 272, 256)
        _, _, uq, us = _operands(2, 1, 1, 272, 256)
        _, _, dq, dsc = _operands(3, 1, 1, 256, 272)
        ex = N.Fp8BlockExperts.from_quantized(gq, gs, uq, us, dq, dsc)
        clean = N.grouped_gated_mlp_fp8_blocks(xq, xs, ex, [0], [rows], N.ACT_SILU)
        xq.view(torch.uint8)[3, 7] = 0xFF  # NaN
        xs[2, 0] = 3e38                    # h overflows to infinities
        Y = N.grouped_gated_mlp_fp8_blocks(xq, xs, ex, [0], [rows], N.ACT_SILU)
        assert bool(Y[3].isnan().all()) and bool(Y[2].isnan().any())
        keep = [r for r in range(rows) if r not in (2, 3)]
        assert torch.equal(Y[keep], clean[keep])


@gpu
@pytest.mark.parametrize("silu", [True, False])
@pytest.mark.parametrize("rows,d", [(5, 256), (3, 4096), (200, 256), (600, 256)],
                         ids=["whole", "split", "single", "pair"])
def test_gated_mlp_nan_in_the_gate_stack_alone(rows, d, silu):
    """A NaN gate is a NaN h whatever the activation, although the up value is finite: a code of one
    expert's gate stack and a scale of another's, each kernel and a split tile; the third expert's rows are
    as without them."""
    N = _nat()
    I = 272
    xq, xs, gq, gs = _operands(1, 3 * rows, 3, I, d)
    _, _, uq, us = _operands(2, 1, 3, I, d)
    _, _, dq, dsc = _operands(3, 1, 3, d, I)
    ex = N.Fp8BlockExperts.from_quantized(gq, gs, uq, us, dq, dsc)
    act = N.ACT_SILU if silu else N.ACT_RELU
    table = ([0, 1, 2], [rows, 2 * rows, 3 * rows])
    clean = N.grouped_gated_mlp_fp8_blocks(xq, xs, ex, *table, act)
    gq.view(torch.uint8)[0, 5, 7] = 0x7F
    gs[1, 2, 0] = float("nan")
    Y = N.grouped_gated_mlp_fp8_blocks(xq, xs, ex, *table, act)
    assert bool(clean.isfinite().all())
    assert bool(Y[:2 * rows].isnan().all())
    assert torch.equal(Y[2 * rows:], clean[2 * rows:])


@gpu
def test_experts_quantised_from_bf16():
    """The whole path a user takes: a bf16 stack quantised once, rows quantised per call, close to
    the bf16 experts within the rounding of e4m3 (half a step, 2^-4, in each of three operands)."""
    N = _nat()
    g = torch.Generator(device=DEV).manual_seed(9)
    E, d, I, rows = 4, 512, 768, 300
    w = [(torch.randn(E, *s, generator=g, device=DEV) * 0.02).to(torch.bfloat16) for s in ((I, d), (I, d), (d, I))]
    x = torch.randn(rows, d, generator=g, device=DEV).to(torch.bfloat16)
    ends = [100, 100, 230, 300]
    want = torch.empty(rows, d, dtype=torch.bfloat16, device=DEV)
    N.grouped_gated_mlp(x, *w, list(range(E)), ends, N.ACT_SILU, want)
    Y = N.grouped_gated_mlp_fp8_blocks(*N.quantize_blocks_e4m3(x), N.Fp8BlockExperts(*w), list(range(E)), ends, N.ACT_SILU)
    assert ((Y.float() - want.float()).norm() / want.float().norm()).item() <= 3 * 2.0 ** -4


# ------------------------------------------------------------------------------- how they are called
@gpu
def test_bad_device_table_is_reported():
    """Ends out of order or past the rows are clamped, an expert outside the stack is left out, and
    the status word says so."""
    N = _nat()
    xq, xs, wq, ws = _operands(8, 40, 2, 136, 256)
    good = N.grouped_matmul_fp8_blocks(xq, xs, wq, ws, [0, 1], [10, 40])
    for hint in (1, 200):
        for experts, ends in (([0, 5, 1], [10, 10, 40]), ([0, 1], [10, 4000]), ([0, 1, 1], [10, 5, 40]), ([0, -3, 1], [10, 12, 40])):
            out = torch.full((40, 136), 3.0, dtype=torch.bfloat16, device=DEV)
            N.grouped_matmul_fp8_blocks(xq, xs, wq, ws, torch.tensor(experts, dtype=torch.int32, device=DEV),
                                        torch.tensor(ends, dtype=torch.int32, device=DEV), out, rows_hint=hint)
            with pytest.raises(N.DMoEError, match="segment"):
                N.check_device_status(torch.device(DEV))
            first = 12 if ends[1] == 12 else 10
            assert (out[:10].double() - good[:10].double()).abs().max() <= 0.01 * good.double().abs().max()
            assert (out[first:].double() - good[first:].double()).abs().max() <= 0.01 * good.double().abs().max()
            assert bool((out[10:first] == 3.0).all())


@gpu
@pytest.mark.parametrize("hint", [1, 30, 200])
@pytest.mark.parametrize("experts,ends,parts", [
    ([0, 5, 1], [10, 10, 40], [(0, 0, 10), (1, 10, 40)]),
    ([0, 1], [10, 4000], [(0, 0, 10), (1, 10, 40)]),
    ([0, 1, 1], [10, 5, 40], [(0, 0, 10), (1, 10, 40)]),
    ([0, -3, 1], [10, 12, 40], [(0, 0, 10), (1, 12, 40)]),
    ([1, 0], [-7, 40], [(0, 0, 40)]),
    ([2, 1], [2**31 - 1, 40], []),
])
def test_what_a_bad_device_table_leaves(experts, ends, parts, hint):
    """The rows that remain after clamping, each against the definition; all others as they were."""
    N = _nat()
    xq, xs, wq, ws = _operands(8, 40, 2, 136, 256)
    x, w = _values(xq, xs, 1), _values(wq, ws, 128)
    out = torch.full((40, 136), 3.0, dtype=torch.bfloat16, device=DEV)
    N.grouped_matmul_fp8_blocks(xq, xs, wq, ws, torch.tensor(experts, dtype=torch.int32, device=DEV),
                                torch.tensor(ends, dtype=torch.int32, device=DEV), out, rows_hint=hint)
    with pytest.raises(N.DMoEError, match="segment"):
        N.check_device_status(torch.device(DEV))
    left = torch.ones(40, dtype=torch.bool, device=DEV)
    for e, a, b in parts:
        _check(out[a:b], x[a:b] @ w[e].T, _product_slack(x[a:b].abs(), w[e].abs()), 2.0 ** -7)
        left[a:b] = False
    assert bool((out[left] == 3.0).all())


@gpu
def test_wrapper_refusals():
    N = _nat()
    xq, xs, wq, ws = _operands(8, 4, 2, 136, 256)
    seg = ([0], [4])
    i32 = dict(dtype=torch.int32, device=DEV)
    bad = [
        lambda: N.quantize_blocks_e4m3(torch.zeros(4, 24, device=DEV)),
        lambda: N.quantize_blocks_e4m3(torch.zeros(4, 256, device=DEV), 64),
        lambda: N.quantize_blocks_e4m3(torch.zeros(256, device=DEV), 128),
        lambda: N.quantize_blocks_e4m3(torch.zeros(4, 256, dtype=torch.float64, device=DEV)),
        lambda: N.quantize_blocks_e4m3(torch.zeros(256, 4, device=DEV).T),
        lambda: N.grouped_matmul_fp8_blocks(xq.float(), xs, wq, ws, *seg),
        lambda: N.grouped_matmul_fp8_blocks(xq, xs.double(), wq, ws, *seg),
        lambda: N.grouped_matmul_fp8_blocks(xq, xs[:, :1], wq, ws, *seg),
        lambda: N.grouped_matmul_fp8_blocks(xq[:, :128], xs, wq, ws, *seg),
        lambda: N.grouped_matmul_fp8_blocks(xq, xs, wq, ws[:, :1], *seg),
        lambda: N.grouped_matmul_fp8_blocks(xq, xs, wq, ws, [0], [5]),
        lambda: N.grouped_matmul_fp8_blocks(xq, xs, wq, ws, [2], [4]),
        lambda: N.grouped_matmul_fp8_blocks(xq, xs, wq, ws, [0, 1], [4]),
        lambda: N.grouped_matmul_fp8_blocks(xq, xs, wq, ws, torch.zeros(1, **i32), [4]),
        lambda: N.grouped_matmul_fp8_blocks(xq, xs, wq, ws, torch.zeros(1, device=DEV), torch.zeros(1, **i32)),
        lambda: N.grouped_matmul_fp8_blocks(xq, xs, wq, ws, torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)),
        lambda: N.grouped_matmul_fp8_blocks(xq, xs, wq, ws, *seg, torch.zeros(3, 136, device=DEV)),
        lambda: N.grouped_matmul_fp8_blocks(xq, xs, wq, ws, *seg, torch.zeros(4, 136, device=DEV), out_dtype=torch.bfloat16),
        lambda: N.grouped_matmul_fp8_blocks(xq, xs, wq, ws, *seg, out_dtype=torch.float64),
        lambda: N.matmul_fp8_blocks(xq, xs, wq, ws),
        lambda: N.Fp8BlockExperts.from_quantized(wq, ws, wq, ws, wq, ws),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(N.DMoEError):
            call()
            raise AssertionError(f"call {i} went through")


@gpu
def test_streams_and_captured_graphs():
    """Two captured graphs and an eager call on a third stream, replayed together: no workspace is
    shared, and a replay reads the inputs as they are then."""
    N = _nat()
    g = torch.Generator(device=DEV).manual_seed(3)
    E, d, I = 4, 512, 384
    ex = N.Fp8BlockExperts(*[torch.randn(E, *s, generator=g, device=DEV) * 0.03 for s in ((I, d), (I, d), (d, I))])
    end = torch.tensor([3, 3, 40, 96], **dict(dtype=torch.int32, device=DEV))
    expert = torch.arange(E, dtype=torch.int32, device=DEV)

    def layer(x):
        return N.grouped_gated_mlp_fp8_blocks(*N.quantize_blocks_e4m3(x), ex, expert, end, N.ACT_SILU)

    xs = [torch.randn(96, d, generator=g, device=DEV).to(torch.bfloat16) for _ in range(3)]
    layer(xs[0])
    graphs, outs = [], []
    for x in xs[:2]:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(layer(x))
        graphs.append(graph)
    streams = [torch.cuda.Stream(DEV) for _ in range(3)]
    for turn in range(3):
        for x in xs:
            x.copy_(torch.randn(96, d, generator=g, device=DEV))
        torch.cuda.synchronize()
        want = [layer(x) for x in xs]
        torch.cuda.synchronize()
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        with torch.cuda.stream(streams[2]):
            third = layer(xs[2])
        torch.cuda.synchronize()
        for a, b in zip(outs + [third], want):
            assert torch.equal(a, b)
    N.check_device_status(torch.device(DEV))


@gpu
def test_same_bits_every_time():
    """No sum depends on the order in which CTAs run: repeated calls agree bit for bit, the cluster
    split among them."""
    N = _nat()
    for rows, Nn, K in ((1, 512, 4096), (20, 256, 7168), (300, 1000, 2048)):
        xq, xs, wq, ws = _operands(rows, rows, 1, Nn, K)
        first = N.matmul_fp8_blocks(xq, xs, wq[0], ws[0], out_dtype=torch.float32)
        for _ in range(5):
            assert torch.equal(first, N.matmul_fp8_blocks(xq, xs, wq[0], ws[0], out_dtype=torch.float32))


@gpu
def test_pair_products_repeat_and_match():
    """Several tiles a pair of SMs, each accumulator handed back by both CTAs many times: repeated calls
    agree bit for bit, and with the definition."""
    N = _nat()
    for rows, Nn, K in ((2048, 4104, 2064), (5000, 1032, 400)):
        xq, xs, wq, ws = _operands(rows, rows, 1, Nn, K)
        first = N.matmul_fp8_blocks(xq, xs, wq[0], ws[0], out_dtype=torch.float32)
        x, w = _values(xq, xs, 1), _values(wq, ws, 128)[0]
        _check(first, x @ w.T, _product_slack(x.abs(), w.abs()), 2.0 ** -23)
        for _ in range(20):
            assert torch.equal(first, N.matmul_fp8_blocks(xq, xs, wq[0], ws[0], out_dtype=torch.float32))
    N.check_device_status(torch.device(DEV))


@gpu
@pytest.mark.parametrize("rows", [3, 96, 700])
def test_calls_in_a_row_on_changing_inputs(rows):
    """Each kernel starts while the one before it drains, on buffers that the allocator hands round: codes,
    scales and h of another call are never seen."""
    N = _nat()
    g = torch.Generator(device=DEV).manual_seed(5)
    E, d, I = 3, 512, 384
    ex = N.Fp8BlockExperts(*[torch.randn(E, *s, generator=g, device=DEV) * 0.03 for s in ((I, d), (I, d), (d, I))])
    end = torch.tensor([rows // 3, rows // 2, rows], dtype=torch.int32, device=DEV)
    expert = torch.arange(E, dtype=torch.int32, device=DEV)
    xs = [(torch.randn(rows, d, generator=g, device=DEV) * 3.0 ** (i % 7 - 3)).to(torch.bfloat16) for i in range(12)]

    def layer(x):
        return N.grouped_gated_mlp_fp8_blocks(*N.quantize_blocks_e4m3(x), ex, expert, end, N.ACT_SILU)

    want = []
    for x in xs:
        torch.cuda.synchronize()
        want.append(layer(x))
        torch.cuda.synchronize()
    for _ in range(5):
        got = [layer(x) for x in xs]
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    N.check_device_status(torch.device(DEV))


@gpu
def test_no_rows_and_no_segments():
    N = _nat()
    xq, xs, wq, ws = _operands(8, 4, 2, 136, 256)
    assert N.quantize_blocks_e4m3(torch.empty(0, 256, device=DEV))[0].shape == (0, 256)
    assert N.matmul_fp8_blocks(xq[:0], xs[:0], wq[0], ws[0]).shape == (0, 136)
    out = torch.full((4, 136), 2.0, dtype=torch.bfloat16, device=DEV)
    N.grouped_matmul_fp8_blocks(xq, xs, wq, ws, [], [], out)
    N.grouped_matmul_fp8_blocks(xq, xs, wq, ws, [0, 1], [0, 0], out)
    zero = torch.zeros(2, dtype=torch.int32, device=DEV)
    for hint in (1, 200):
        N.grouped_matmul_fp8_blocks(xq, xs, wq, ws, zero, zero, out, rows_hint=hint)
    assert bool((out == 2.0).all())
    N.check_device_status(torch.device(DEV))


@gpu
def test_replaced_weights_are_used():
    """An expert stack whose tensors are exchanged is read as it is then."""
    N = _nat()
    xq, xs, gq, gs = _operands(1, 6, 1, 272, 256)
    _, _, dq, dsc = _operands(3, 1, 1, 256, 272)
    ex = N.Fp8BlockExperts.from_quantized(gq, gs, gq, gs, dq, dsc)
    first = N.grouped_gated_mlp_fp8_blocks(xq, xs, ex, [0], [6], N.ACT_SILU)
    ex.wd_scale = dsc * 2
    assert torch.equal(N.grouped_gated_mlp_fp8_blocks(xq, xs, ex, [0], [6], N.ACT_SILU), first * 2)
