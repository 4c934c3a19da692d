"""The 8-bit-integer operators on a B200 against plain computations in 64 bits.

Tolerances. ``e`` is the output type's unit (half a step: ``finfo.eps / 2``), ``u = 2**-24`` FP32's.
A product is ``float(sum) * sa * sb + bias``: the sum is exact, so four FP32 roundings of at most
the size of the result or of the product before the bias, then one of the output type, and half the
smallest subnormal step of FP16 where results are that small. The gate multiplies ``silu(g)`` and
the up product. ``silu`` is ``g * 1/(1 + exp(-g))``: the exponential is documented to ``2 +
1.173 |g|`` steps of ``2**-23`` and the quotient to 2, and its slope is below 1.1."""

import numpy as np
import pytest
import torch

from harness import int8, native

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
U = 2.0 ** -24
FP16_STEP = 2.0 ** -25


def rng_of(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def make_codes(g, *shape, extra=0):
    """Codes of the whole range, -128 included; rows ``extra`` bytes further apart than needed."""
    *lead, k = shape
    pitch = -(-k // 16) * 16 + extra
    return torch.randint(-128, 128, (*lead, pitch), dtype=torch.int8, device=DEV, generator=g)[..., :k]


def product_bounds(a, b, sa, sb, bias, gated, dtype):
    """(value, bound on the error) in 64 bits."""
    z = (a.double() @ b.double().T) * sa.double()[:, None] * sb.double()
    err = 4 * U * z.abs()
    if bias is not None:
        z = z + bias.double()
        err = err + 2 * U * (z.abs() + bias.double().abs())
    if gated:
        gate, up = z.chunk(2, dim=1)
        eg, eu = err.chunk(2, dim=1)
        s = gate * torch.sigmoid(gate)
        es = 1.1 * eg + s.abs() * ((2 + 1.173 * gate.abs() + 2 + 2) * 2 * U)
        z = s * up
        err = es * up.abs() + s.abs() * eu + es * eu + 2 * U * z.abs()
    e = torch.finfo(dtype).eps / 2
    return z, err * (1 + e) + e * z.abs() + (FP16_STEP if dtype == torch.float16 else 1e-44)


def assert_product(got, a, b, sa, sb, bias=None, gated=False):
    z, bound = product_bounds(a, b, sa, sb, bias, gated, got.dtype)
    over = (got.double() - z).abs() - bound
    assert got.shape == z.shape and not torch.isnan(got).any()
    assert (over <= 0).all(), f"{over.max().item()} over the bound, at {torch.nonzero(over > 0)[:4].tolist()}"


def guarded(rows, n, dtype, pitch=None, lead=3):
    """An output inside a larger buffer of a known filling; (view, check that the rest kept it)."""
    pitch = pitch or n + 5
    buffer = torch.full((rows + 2 * lead, pitch), 77.0, dtype=dtype, device=DEV)
    view = buffer[lead:lead + rows, 2:2 + n] if pitch > n + 1 else buffer[lead:lead + rows, :n]

    def check():
        rest = buffer.clone()
        (rest[lead:lead + rows, 2:2 + n] if pitch > n + 1 else rest[lead:lead + rows, :n]).fill_(77.0)
        assert (rest == 77.0).all(), "written outside the output"
    return view, check


DTYPES = (torch.bfloat16, torch.float16, torch.float32)


@pytest.mark.parametrize("m,n,k", [
    (1, 1, 1), (1, 8, 16), (1, 300, 7), (2, 129, 130), (7, 64, 128), (16, 128, 256), (17, 127, 1000),
    (31, 257, 144), (33, 1000, 96), (64, 64, 2048), (65, 33, 4097), (100, 515, 513), (127, 130, 127),
    (129, 256, 129), (255, 200, 384), (256, 256, 128), (257, 511, 640), (300, 1030, 2064),
    (513, 770, 1100), (1000, 96, 80), (1, 4096, 4096), (5, 2000, 8192), (40, 136, 16384)])
@pytest.mark.parametrize("gated", [False, True])
def test_product_over_sizes(m, n, k, gated):
    """Odd and small sizes, every output type, an output with rows of its own pitch, and no byte
    outside it."""
    g = rng_of(m * 1009 + n * 31 + k)
    width = 2 * n if gated else n
    a, b = make_codes(g, m, k, extra=16), make_codes(g, width, k)
    sa = 0.5 + torch.rand(m, device=DEV, generator=g)
    sb = (0.5 + torch.rand(width, device=DEV, generator=g)) * (2e-4 / k ** 0.5)
    bias = torch.randn(width, device=DEV, generator=g)
    for i, dtype in enumerate(DTYPES):
        with_bias = bias if i != 0 else None
        out, check = guarded(m, n, dtype, pitch=n + 5 if i else -(-n // 8) * 8)
        got = int8.gemm(a, b, sa, sb, bias=with_bias, gated=gated, out_dtype=dtype, out=out)
        assert got is out
        assert_product(got, a, b, sa, sb, with_bias, gated)
        check()
        again = int8.gemm(a, b, sa, sb, bias=with_bias, gated=gated, out_dtype=dtype)
        assert torch.equal(again, got), "the same call gave other bits"


@pytest.mark.parametrize("m,n,k", [(3, 96, 6832), (277, 256, 5136), (313, 416, 1500), (33, 130, 2049), (842, 40, 9008),
                                   (120, 24, 640), (60, 300, 4097), (2297, 585, 300)])
@pytest.mark.parametrize("gated", [False, True])
def test_products_of_few_tiles_and_great_depth(m, n, k, gated):
    """Few tiles: parts of k on several CTAs, whose integer sums give the bits of the same rows beside
    others (other tiles, other parts)."""
    g = rng_of(m + n + k)
    width = 2 * n if gated else n
    a, b = make_codes(g, m + 300, k), make_codes(g, width, k)
    sa = 0.5 + torch.rand(m + 300, device=DEV, generator=g)
    sb = (0.5 + torch.rand(width, device=DEV, generator=g)) * (2e-4 / k ** 0.5)
    for dtype in DTYPES:
        out, check = guarded(m, n, dtype)
        int8.gemm(a[:m], b, sa[:m], sb, gated=gated, out_dtype=dtype, out=out)
        check()
        assert_product(out, a[:m], b, sa[:m], sb, None, gated)
        for rows in (1, m // 2 + 1, m + 300):
            other = int8.gemm(a[:rows], b, sa[:rows], sb, gated=gated, out_dtype=dtype)
            assert torch.equal(other[:m], out[:rows])
        counts = torch.tensor([0, m // 3, m // 3, m], dtype=torch.int32, device=DEV)
        grouped = int8.grouped_gemm(a[:m], b.expand(1, width, k).repeat(3, 1, 1) if k % 16 == 0 else make_codes(g, 3, width, k),
                                    sa[:m], sb.repeat(3, 1), counts, gated=gated, out_dtype=dtype)
        if k % 16 == 0:
            assert torch.equal(grouped, out)
    int8.check_status(DEV)


def test_product_extremes():
    """All codes -128 at a depth near the largest: the 32-bit sum does not wrap, and FP32 output
    is it times the scales, rounded as written. Zero, infinite and NaN scales go through."""
    k = 131056
    a = torch.full((3, k), -128, dtype=torch.int8, device=DEV)
    b = torch.full((130, k), -128, dtype=torch.int8, device=DEV)
    b[1] = 127
    sa = torch.tensor([1.0, 0.0, 0.5], device=DEV)
    sb = torch.ones(130, device=DEV)
    sb[5], sb[6] = float("inf"), float("nan")
    y = int8.gemm(a, b, sa, sb, out_dtype=torch.float32)
    assert y[0, 0].item() == k * 128 * 128 and y[2, 0].item() == k * 64 * 128
    assert y[0, 1].item() == float(np.float32(-k * 128 * 127))
    assert (y[1, :5] == 0).all() and y[0, 5].item() == float("inf")
    assert torch.isnan(y[1, 5]) and torch.isnan(y[:, 6]).all()
    h = int8.gemm(a, b, sa, sb, out_dtype=torch.float16)
    assert h[0, 0].item() == float("inf")     # beyond FP16: infinite, not the largest value


def test_product_of_no_rows_and_of_views():
    g = rng_of(5)
    b, sb = make_codes(g, 40, 64), torch.rand(40, device=DEV, generator=g)
    assert int8.gemm(make_codes(g, 0, 64), b, torch.empty(0, device=DEV), sb).shape == (0, 40)
    big = make_codes(g, 60, 256)
    a = big[::3, 32:96]                       # rows 768 bytes apart, from the 32nd byte on
    wide = make_codes(g, 80, 128)
    sa = torch.rand(20, device=DEV, generator=g)
    got = int8.gemm(a, wide[::2, 64:], sa, sb, out_dtype=torch.float32)
    assert_product(got, a, wide[::2, 64:], sa, sb)
    with pytest.raises(ValueError):
        int8.gemm(big[:, 8:72], b, torch.rand(60, device=DEV), sb)     # 8 bytes off
    with pytest.raises(ValueError):
        int8.gemm(big[:1].expand(20, 256), make_codes(g, 40, 256), sa, sb)   # rows on top of each other
    with pytest.raises(ValueError):
        int8.gemm(a, b.cpu(), sa, sb)


@pytest.mark.parametrize("counts,n,k,gated", [
    ((1,), 8, 16, False), ((0, 0, 3), 100, 64, False), ((0, 0), 16, 32, False),
    ((5, 0, 130, 1, 0, 64), 72, 100, True), ((257, 3, 129), 136, 528, True), ((64,) * 8, 256, 256, False),
    ((1, 2, 3, 4, 5, 6, 7, 8, 9), 33, 1000, False), ((700, 0, 1), 513, 300, True),
    (tuple((i * 7) % 5 for i in range(300)), 24, 48, False), ((16,) * 32, 512, 2048, True)])
def test_grouped_product(counts, n, k, gated):
    """Ragged groups, empty ones among them, against each group's product; rows in front of the
    first group and behind the last keep what the output held."""
    g = rng_of(sum(counts) + n)
    experts, owned, front, behind = len(counts), sum(counts), 3, 4
    width = 2 * n if gated else n
    rows = front + owned + behind
    a, b = make_codes(g, rows, k), make_codes(g, experts, width, k)
    sa = 0.5 + torch.rand(rows, device=DEV, generator=g)
    sb = (0.5 + torch.rand((experts, width), device=DEV, generator=g)) * (2e-4 / k ** 0.5)
    edges = [front]
    for count in counts:
        edges.append(edges[-1] + count)
    offsets = torch.tensor(edges, dtype=torch.int32, device=DEV)
    for dtype in DTYPES:
        out, check = guarded(rows, n, dtype)
        int8.grouped_gemm(a, b, sa, sb, offsets, gated=gated, out_dtype=dtype, out=out)
        check()
        assert (out[:front] == 77.0).all() and (out[rows - behind:] == 77.0).all()
        for e, (lo, hi) in enumerate(zip(edges, edges[1:])):
            if hi > lo:
                assert_product(out[lo:hi], a[lo:hi], b[e], sa[lo:hi], sb[e], None, gated)


@pytest.mark.parametrize("n", [1304, 1305])
@pytest.mark.parametrize("k", [1, 200, 1024, 1040])
@pytest.mark.parametrize("gated", [False, True])
def test_shallow_products_of_several_tiles_a_cta(n, k, gated):
    """More tiles than the GPU has SMs, of a small depth: however D lies (rows on multiples of eight
    elements or not) the bits are the same and nothing beside them is written; in groups too, whose last
    rows end inside a tile."""
    g = rng_of(n + k)
    width, rows = 2 * n if gated else n, 5003
    a, b = make_codes(g, rows, k), make_codes(g, 2, width, k)
    sa = 0.5 + torch.rand(rows, device=DEV, generator=g)
    sb = (0.5 + torch.rand((2, width), device=DEV, generator=g)) * (2e-4 / k ** 0.5)
    bias = torch.randn(width, device=DEV, generator=g)
    offsets = torch.tensor([7, 2606, rows - 9], dtype=torch.int32, device=DEV)
    for dtype in (torch.bfloat16, torch.float16):
        dense, grouped = [], []
        for pitch in (-(-n // 8) * 8, n + 16 + -n % 8, n + 5):
            out, check = guarded(rows, n, dtype, pitch=pitch)
            dense.append(int8.gemm(a, b[0], sa, sb[0], bias=bias, gated=gated, out_dtype=dtype, out=out).clone())
            check()
            out, check = guarded(rows, n, dtype, pitch=pitch)
            int8.grouped_gemm(a, b, sa, sb, offsets, gated=gated, out_dtype=dtype, out=out)
            check()
            assert (out[:7] == 77.0).all() and (out[rows - 9:] == 77.0).all()
            grouped.append(out.clone())
        assert_product(dense[0], a, b[0], sa, sb[0], bias, gated)
        for e, (lo, hi) in enumerate(((7, 2606), (2606, rows - 9))):
            assert_product(grouped[0][lo:hi], a[lo:hi], b[e], sa[lo:hi], sb[e], None, gated)
        for other in dense[1:]:
            assert torch.equal(other, dense[0])
        for other in grouped[1:]:
            assert torch.equal(other, grouped[0])
    int8.check_status(DEV)


@pytest.mark.parametrize("rows", [32, 64, 96, 128, 256, 512])
def test_one_expert_that_owns_few_of_the_rows(rows):
    """The tile is made for all rows of the buffers, the group has fewer: its MMA is narrower than
    the tile's full copy."""
    g = rng_of(rows)
    a, b = make_codes(g, rows, 384), make_codes(g, 1, 200, 384)
    sa, sb = torch.rand(rows, device=DEV, generator=g), torch.rand((1, 200), device=DEV, generator=g)
    for lo, hi in ((0, 10), (3, rows // 2), (rows - 1, rows), (0, rows), (5, 5)):
        out, check = guarded(rows, 200, torch.float32)
        int8.grouped_gemm(a, b, sa, sb, torch.tensor([lo, hi], dtype=torch.int32, device=DEV),
                          out_dtype=torch.float32, out=out)
        check()
        assert (out[:lo] == 77.0).all() and (out[hi:] == 77.0).all()
        if hi > lo:
            assert_product(out[lo:hi], a[lo:hi], b[0], sa[lo:hi], sb[0])
    int8.check_status(DEV)


def test_grouped_product_of_strided_experts_equals_the_dense_one():
    g = rng_of(9)
    b = make_codes(g, 6, 200, 96)[::2]
    a, counts = make_codes(g, 333, 96), (100, 33, 200)
    sa = torch.rand(333, device=DEV, generator=g)
    sb = torch.rand((3, 200), device=DEV, generator=g)
    offsets = torch.tensor([0, 100, 133, 333], dtype=torch.int32, device=DEV)
    got = int8.grouped_gemm(a, b, sa, sb, offsets, out_dtype=torch.float32)
    want = torch.cat([int8.gemm(x, b[e], s, sb[e], out_dtype=torch.float32)
                      for e, (x, s) in enumerate(zip(a.split(counts), sa.split(counts)))])
    assert torch.equal(got, want)


@pytest.mark.parametrize("edges", [(-5, 4, 900), (0, 1 << 30, 1 << 30), (0, 60, 20), (100, 100, 100),
                                   (-(1 << 31), (1 << 31) - 1, 0)])
def test_offsets_never_reach_outside_the_rows(edges):
    """Offsets that no plan would make: cut to the rows of the buffers, and nothing else is
    written. The rows of the experts that are in order are right."""
    g = rng_of(3)
    rows, n, k = 90, 40, 64
    a, b = make_codes(g, rows, k), make_codes(g, 2, n, k)
    sa, sb = torch.rand(rows, device=DEV, generator=g), torch.rand((2, n), device=DEV, generator=g)
    out, check = guarded(rows, n, torch.float32)
    int8.grouped_gemm(a, b, sa, sb, torch.tensor(edges, dtype=torch.int32, device=DEV),
                      out_dtype=torch.float32, out=out)
    torch.cuda.synchronize()
    check()
    lo, hi = (min(max(v, 0), rows) for v in edges[:2])
    if hi > lo:
        assert_product(out[lo:hi], a[lo:hi], b[0], sa[lo:hi], sb[0])


def np_quantized(x):
    """(codes, scales) with numpy's correctly rounded FP32 divisions."""
    x = x.float().cpu().numpy()
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        scales = (np.abs(x).max(1) / np.float32(127)).astype(np.float32)
        live = np.isfinite(scales) & (scales > 0)
        q = np.clip(np.rint(x / np.where(live, scales, 1)[:, None].astype(np.float32)), -127, 127)
    return np.where(live[:, None], q, 0).astype(np.int8), scales


def assert_quantized(got, x):
    q, s = np_quantized(x)
    np.testing.assert_array_equal(got[1].cpu().numpy(), s)
    np.testing.assert_array_equal(got[0].cpu().numpy(), q)


@pytest.mark.parametrize("tokens,k", [(1, 1), (1, 2), (3, 7), (2, 8), (5, 63), (4, 64), (33, 255), (9, 1000),
                                      (300, 1024), (17, 2049), (6, 4096), (5, 5120), (3, 8191), (2, 8192),
                                      (3, 16384), (2, 16392), (1, 40001), (2, 131071), (1025, 40)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantiser_bit_for_bit(tokens, k, dtype):
    g = rng_of(tokens + k)
    x = torch.randn((tokens, k), device=DEV, generator=g)
    x *= torch.exp(2 * torch.randn((tokens, 1), device=DEV, generator=g))
    x = x.to(dtype)
    got = int8.quantize_tokens(x)
    assert got[0].stride(0) % 16 == 0 or tokens == 1
    assert_quantized(got, x)
    # Rows that start and lie where no wide load can.
    padded = torch.zeros((tokens, k + 3), dtype=dtype, device=DEV)
    padded[:, 1:k + 1] = x
    assert_quantized(int8.quantize_tokens(padded[:, 1:k + 1]), x)
    buffer = torch.full((tokens + 2, -(-k // 16) * 16 + 16), 99, dtype=torch.int8, device=DEV)
    scales = torch.empty(tokens, device=DEV)
    int8.quantize_tokens(x, out=(buffer[1:tokens + 1, :k], scales))
    assert_quantized((buffer[1:tokens + 1, :k], scales), x)
    assert (buffer[:, k:] == 99).all() and (buffer[0] == 99).all() and (buffer[-1] == 99).all()


@pytest.mark.parametrize("k", [5, 64, 3000])
def test_quantiser_of_special_rows(k):
    """Zero rows, infinities, NaN, subnormals, ties and the largest values."""
    x = torch.zeros((12, k), device=DEV)
    x[1, k // 2] = float("inf")
    x[2, k - 1] = float("-inf")
    x[3, 0] = float("nan")
    x[4] = 1e-45
    x[5] = 1e-40
    x[5, 1] = -3e-39
    x[6] = 3.4028234663852886e38
    x[7] = torch.arange(k, device=DEV) % 255 - 127.0            # exact codes
    x[8] = (torch.arange(k, device=DEV) % 253 - 126.0) + 0.5    # ties
    x[8, 0] = 127.0
    x[9] = -0.0
    x[10, 0] = -1.0
    x[11] = 1.0
    x[11, 2] = float("nan")
    x[11, 3] = float("inf")
    q, s = int8.quantize_tokens(x)
    assert_quantized((q[:11], s[:11]), x[:11])
    assert torch.isnan(s[11]) and not q[11].any()
    for bad in (1, 2, 3, 11):        # products of such rows are NaN
        y = int8.gemm(q[bad:bad + 1], q[7:8], s[bad:bad + 1], s[7:8], out_dtype=torch.float32)
        assert torch.isnan(y).all()


@pytest.mark.parametrize("k", [16, 100, 2880])
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantiser_gathers(k, dtype):
    """The same row several times, rows left out, and indices outside: their rows keep what the
    buffers held."""
    g = rng_of(k)
    x = torch.randn((7, k), device=DEV, generator=g).to(dtype)
    rows = torch.tensor([6, 0, 0, -1, 3, 7, 6, 1 << 30, -(1 << 31), 5], dtype=torch.int32, device=DEV)
    q = torch.full((10, -(-k // 16) * 16), 55, dtype=torch.int8, device=DEV)[:, :k]
    s = torch.full((10,), -3.0, device=DEV)
    int8.quantize_tokens(x, rows=rows, out=(q, s))
    valid = (rows >= 0) & (rows < 7)
    assert_quantized((q[valid], s[valid]), x[rows[valid].long()])
    assert (q[~valid] == 55).all() and (s[~valid] == -3.0).all()
    assert int8.quantize_tokens(x[:0], rows=rows[3:4], out=(q[3:4], s[3:4]))[1][0] == -3.0
    empty = int8.quantize_tokens(x, rows=rows[:0])
    assert empty[0].shape == (0, k) and empty[1].shape == (0,)


def norm_plain(x, residual, post, gate, scale, weight, eps):
    """(r, y, bound of r's error in FP32, bound of y's) in 64 bits."""
    p = x.double()
    parts = torch.zeros_like(p)
    if post is not None:
        p = p / (p.square().mean(1, keepdim=True) + eps).sqrt() * post.double()
    if gate is not None:
        p = p * gate.double().repeat_interleave(x.shape[0] // gate.shape[0], dim=0)
    r = p
    parts = 5 * U * p.abs()                 # rstd, two products, the gate, and to spare
    if residual is not None:
        r = residual.double() * scale + p
        parts = parts + 2 * U * (residual.double() * scale).abs() + U * r.abs()
    if weight is None:
        return r, None, parts, None
    rstd = 1 / (r.square().mean(1, keepdim=True) + eps).sqrt()
    y = r * rstd * weight.double()
    # An error d of r moves the row's root mean square by at most rms(d).
    moved = (parts.square().mean(1, keepdim=True).sqrt() * rstd).clamp(max=1.0)
    return r, y, parts, parts * rstd * weight.double().abs() * (1 + moved) + y.abs() * (moved * (1 + moved) + 4 * U)


def assert_norm(outputs, residual_dtype, y_dtype, plain):
    r, y, scales = outputs
    want_r, want_y, er, ey = plain
    if r is not None:
        e = torch.finfo(residual_dtype).eps / 2
        assert r.dtype == residual_dtype
        step = FP16_STEP if residual_dtype == torch.float16 else 1e-40
        assert ((r.double() - want_r).abs() <= er * (1 + e) + e * want_r.abs() + step).all()
    if want_y is None:
        assert y is None and scales is None
    elif scales is None:
        e = torch.finfo(y_dtype).eps / 2
        assert y.dtype == y_dtype
        step = FP16_STEP if y_dtype == torch.float16 else 1e-40
        assert ((y.double() - want_y).abs() <= ey * (1 + e) + e * want_y.abs() + step).all()
    else:
        assert y.dtype == torch.int8
        amax, at = want_y.abs().max(1)
        assert ((scales.double() - amax / 127).abs() <= ey.max(1).values / 127 + U * amax).all()
        # A code is half a step from its value, and the value off by its own error.
        off = (y.double() * scales.double()[:, None] - want_y).abs()
        assert (off <= scales.double()[:, None] * (0.5 + 127 * 4 * U) + ey).all()


@pytest.mark.parametrize("tokens,hidden", [(1, 1), (1, 7), (2, 8), (3, 63), (4, 128), (33, 255), (7, 1000),
                                           (200, 1024), (5, 2049), (6, 2880), (2, 4100), (4, 7168), (3, 8192),
                                           (2, 10001), (2, 16384), (1, 32767), (2, 32768), (1200, 24)])
@pytest.mark.parametrize("kind", range(4))
def test_norm_over_sizes(tokens, hidden, kind):
    g = rng_of(tokens * 7 + hidden)
    xt, rt, yt = ((torch.bfloat16, torch.bfloat16, torch.bfloat16), (torch.float32, torch.float16, torch.float32),
                  (torch.float16, torch.float32, torch.float16), (torch.float32, torch.bfloat16, torch.bfloat16))[kind]
    x = (3 * torch.randn((tokens, hidden), device=DEV, generator=g)).to(xt)
    residual = torch.randn((tokens, hidden), device=DEV, generator=g).to(rt)
    post = 0.5 + torch.rand(hidden, device=DEV, generator=g)
    weight = 0.5 + torch.rand(hidden, device=DEV, generator=g)
    gates = {0: 1, 1: tokens, 2: None, 3: 2 if tokens % 2 == 0 else 1}[kind]
    gate = torch.randn((gates, hidden), device=DEV, generator=g) if gates else None
    scale = (1.0, 0.5, 0.3, -2.0)[kind]
    if kind == 2:
        post = None
    f32scale = float(np.float32(scale))
    plain = norm_plain(x, residual, post, gate, f32scale, weight, 1e-6)
    call = dict(post_weight=post, gate=gate, residual_scale=scale, eps=1e-6)
    assert_norm(int8.residual_norm(x, residual, next_weight=weight, out_dtype=yt, **call), rt, yt, plain)
    coded = int8.residual_norm(x, residual, next_weight=weight, quantize=True, **call)
    assert_norm(coded, rt, None, plain)
    assert_norm(int8.residual_norm(x, residual, **call), rt, None, (*plain[:1], None, plain[2], None))
    # The codes are those of the FP32 rows.
    y32 = int8.residual_norm(x, residual, next_weight=weight, out_dtype=torch.float32, **call)[1]
    assert_quantized(coded[1:], y32)
    # The norm alone.
    alone = norm_plain(x, None, None, None, 1.0, weight, 1e-6)
    assert_norm(int8.residual_norm(x, next_weight=weight, out_dtype=yt), None, yt, alone)
    # In place, from rows that start and lie where no wide load can.
    off = torch.zeros((tokens, hidden + 3), dtype=rt, device=DEV)
    off[:, 1:hidden + 1] = residual
    xoff = torch.zeros((tokens, hidden + 5), dtype=xt, device=DEV)
    xoff[:, 3:hidden + 3] = x
    inplace = int8.residual_norm(xoff[:, 3:hidden + 3], off[:, 1:hidden + 1], next_weight=weight, quantize=True,
                                 residual_out=off[:, 1:hidden + 1], **call)
    assert torch.equal(inplace[0], coded[0]) and torch.equal(inplace[1], coded[1])
    assert torch.equal(inplace[2], coded[2])
    assert (off[:, 0] == 0).all() and (off[:, hidden + 1:] == 0).all()


def test_norm_into_given_tensors():
    g = rng_of(8)
    x, residual = (torch.randn((37, 264), device=DEV, generator=g).bfloat16() for _ in range(2))
    w = 0.5 + torch.rand(264, device=DEV, generator=g)
    want = int8.residual_norm(x, residual, post_weight=w, next_weight=w, out_dtype=torch.float16)
    view, check = guarded(37, 264, torch.float16)
    r = torch.empty_like(residual)
    got = int8.residual_norm(x, residual, post_weight=w, next_weight=w, out_dtype=torch.float16, out=view,
                             residual_out=r)
    assert got[0] is r and got[1] is view and torch.equal(r, want[0]) and torch.equal(view, want[1])
    check()
    want = int8.residual_norm(x, residual, post_weight=w, next_weight=w, quantize=True)
    q, s = torch.empty((37, 300), dtype=torch.int8, device=DEV)[:, :264], torch.empty(37, device=DEV)
    got = int8.residual_norm(x, residual, post_weight=w, next_weight=w, quantize=True, out=(q, s))
    assert got[1] is q and torch.equal(q, want[1]) and torch.equal(s, want[2])
    for bad in (torch.empty((37, 264), device=DEV), torch.empty((36, 264), dtype=torch.bfloat16, device=DEV)):
        with pytest.raises(ValueError):
            int8.residual_norm(x, residual, next_weight=w, out=bad)
    with pytest.raises(ValueError):
        int8.residual_norm(x, residual, out=view)


def test_norm_of_special_rows():
    """Zero rows give zeros, infinite and NaN rows poison only themselves."""
    x = torch.ones((5, 300), device=DEV)
    x[0] = 0
    x[1, 7] = float("inf")
    x[2, 299] = float("nan")
    x[3] = 1e30                          # the square overflows FP32, not the sum in 64 bits
    w = torch.full((300,), 2.0, device=DEV)
    _, y, _ = int8.residual_norm(x, next_weight=w, eps=1e-6)
    assert (y[0] == 0).all() and torch.isnan(y[1, 7]) and (y[1, :7] == 0).all() and torch.isnan(y[2]).all()
    torch.testing.assert_close(y[3], torch.full((300,), 2.0, device=DEV), rtol=4 * U, atol=0)
    _, q, s = int8.residual_norm(x, next_weight=w, quantize=True)
    assert s[0] == 0 and not q[:3].any() and torch.isnan(s[1]) and torch.isnan(s[2])
    assert (q[3:] == 127).all()
    assert int8.residual_norm(x[:0], next_weight=w)[1].shape == (0, 300)
    with pytest.raises(ValueError):
        int8.residual_norm(x, x, gate=torch.ones((2, 300), device=DEV), next_weight=w)


def test_calls_on_two_streams_and_from_two_threads():
    """Nothing is shared between calls: two streams at once give what one gives."""
    import threading

    g = rng_of(21)
    sets = []
    for m, n, k in ((200, 1000, 4096), (3, 4000, 2048)):
        x = torch.randn((m, k), device=DEV, generator=g)
        b, sb = int8.quantize_tokens(torch.randn((n, k), device=DEV, generator=g))
        a, sa = int8.quantize_tokens(x)
        sets.append((x, b, sb, int8.gemm(a, b, sa, sb)))
    torch.cuda.synchronize()
    results, errors = [[], []], []

    def work(i):
        try:
            stream = torch.cuda.Stream(DEV)
            x, b, sb, _ = sets[i]
            with torch.cuda.stream(stream):
                for _ in range(20):
                    a, sa = int8.quantize_tokens(x)
                    results[i].append(int8.gemm(a, b, sa, sb))
            stream.synchronize()
        except Exception as error:
            errors.append(error)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for (*_, want), got in zip(sets, results):
        assert len(got) == 20 and all(torch.equal(y, want) for y in got)


def test_a_captured_chain_replays_on_new_data():
    """Norm, product, quantiser and grouped product in one graph, replayed with other inputs and
    other offsets, equal the eager calls; two graphs of the same calls share nothing."""
    g = rng_of(31)
    tokens, hidden, inter, experts = 50, 192, 80, 4
    w = torch.rand(hidden, device=DEV, generator=g)
    b1, s1 = int8.quantize_tokens(torch.randn((2 * inter, hidden), device=DEV, generator=g))
    b2, s2 = int8.quantize_tokens(torch.randn((experts * hidden, inter), device=DEV, generator=g))
    b2 = torch.nn.functional.pad(b2, (0, 0)).contiguous().view(experts, hidden, inter)
    s2 = s2.view(experts, hidden)

    def chain(x, residual, offsets):
        r, q, s = int8.residual_norm(x, residual, post_weight=w, next_weight=w, quantize=True)
        h = int8.gemm(q, b1, s, s1, gated=True)
        q2, t = int8.quantize_tokens(h)
        return r, int8.grouped_gemm(q2, b2, t, s2, offsets, out_dtype=torch.float32)

    def inputs(seed):
        g = rng_of(seed)
        edges = [0, *sorted(torch.randint(0, tokens + 1, (experts - 1,), generator=torch.Generator().manual_seed(seed)).tolist()), tokens]
        return (torch.randn((tokens, hidden), device=DEV, generator=g),
                torch.randn((tokens, hidden), device=DEV, generator=g).bfloat16(),
                torch.tensor(edges, dtype=torch.int32, device=DEV))

    graphs = []
    for seed in (1, 2):
        static = inputs(seed)
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            chain(*static)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outputs = chain(*static)
        graphs.append((graph, static, outputs))
    for seed in (3, 4):
        fresh = [inputs(seed + 10 * i) for i in range(2)]
        for (graph, static, _), new in zip(graphs, fresh):
            for old, value in zip(static, new):
                old.copy_(value)
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        torch.cuda.synchronize()
        for (graph, *_), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for (_, _, outputs), new in zip(graphs, fresh):
            for got, want in zip(outputs, chain(*new)):
                assert torch.equal(got, want)


@pytest.mark.parametrize("name", ["int8_gemm", "int8_group_gemm", "int8_quantize", "residual_norm"])
def test_workload_smoke_cases(name):
    from harness import get_workload

    with get_workload(name).from_arch("sm_100a", device="cuda") as workload:
        for case in workload.get_cases():
            if case.suite != "smoke":
                continue
            inputs = workload.get_inputs(case)
            out = workload.run(inputs)
            workload.validate(workload.get_reference(inputs), out)
            launch, outputs = workload.prepare(inputs)
            allocated = torch.cuda.memory_stats()["allocation.all.allocated"]
            assert launch() is outputs
            assert torch.cuda.memory_stats()["allocation.all.allocated"] == allocated
            workload.validate(out, outputs)
        workload.check_status()


def test_offsets_and_placement_of_pairs():
    """Unpadded routing on the device: offsets are the prefix of the counts, every pair has a row
    of its expert, ids outside have none."""
    ids = torch.tensor([[3, 0], [3, 9], [-1, 0], [3, 1]], dtype=torch.int64, device=DEV)
    stream = torch.cuda.current_stream().cuda_stream
    counts, cursors = (torch.zeros(5, dtype=torch.int32, device=DEV) for _ in range(2))
    offsets = torch.full((6,), -7, dtype=torch.int32, device=DEV)
    row_of_pair, token_of_row = (torch.full((8,), -9, dtype=torch.int32, device=DEV) for _ in range(2))
    native.moe_count(ids.data_ptr(), True, 8, 5, counts.data_ptr(), stream)
    native.moe_offsets(counts.data_ptr(), 5, offsets.data_ptr(), stream)
    native.moe_place_offsets(ids.data_ptr(), True, 8, 2, 5, offsets.data_ptr(), 8, cursors.data_ptr(),
                             row_of_pair.data_ptr(), token_of_row.data_ptr(), stream)
    assert offsets.tolist() == [0, 2, 3, 3, 6, 6]
    rows = row_of_pair.tolist()
    assert sorted(rows[i] for i in (0, 2, 6)) == [3, 4, 5] and sorted(rows[i] for i in (1, 5)) == [0, 1]
    assert rows[7] == 2 and rows[3] == rows[4] == -1
    tokens = token_of_row.tolist()
    assert all(tokens[rows[i]] == i // 2 for i in (0, 1, 2, 5, 6, 7)) and tokens[6:] == [-1, -1]


def moe_plain(x, ids, weights, w13, s13, w2, s2):
    """The layer in 64 bits, with the two quantisers where the layer has them: the first on the
    tokens (numpy's, bit for bit), the second on the gate rounded to BF16."""
    experts, inter = w13.shape[0], w13.shape[1] // 2
    q, s = np_quantized(x)
    a = torch.from_numpy(q).to(DEV).double() * torch.from_numpy(s).to(DEV).double()[:, None]
    out = torch.zeros(x.shape, dtype=torch.float64, device=DEV)
    for e in range(experts):
        token, choice = torch.nonzero(ids == e, as_tuple=True)
        if token.numel() == 0:
            continue
        h = a[token] @ (w13[e].double() * s13[e].double()[:, None]).T
        h = (h[:, :inter] * torch.sigmoid(h[:, :inter]) * h[:, inter:]).to(torch.bfloat16)
        q2, t2 = np_quantized(h)
        b = torch.from_numpy(q2).to(DEV).double() * torch.from_numpy(t2).to(DEV).double()[:, None]
        y = b @ (w2[e].double() * s2[e].double()[:, None]).T
        out.index_add_(0, token, y * weights[token, choice].double()[:, None])
    return out


def moe_case(tokens, hidden, inter, experts, choices, dtype=torch.bfloat16):
    from harness import moe

    g = rng_of(tokens + hidden)
    w13, s13 = moe.quantize_int8_weights(torch.randn((experts, 2 * inter, hidden), device=DEV, generator=g) / hidden ** 0.5)
    w2, s2 = moe.quantize_int8_weights(torch.randn((experts, hidden, inter), device=DEV, generator=g) / inter ** 0.5)
    x = torch.randn((tokens, hidden), device=DEV, generator=g).to(dtype)
    scores = torch.rand((tokens, experts), device=DEV, generator=g)
    scores[:, experts - 1] = -1.0                   # an expert without tokens
    weights, ids = torch.topk(scores, choices, dim=1)
    return moe.Int8MoELayer(w13, s13, w2, s2), x, ids, weights


def assert_moe(got, x, ids, weights, layer):
    """Against the stages in 64 bits. A gate next to a rounding border of BF16 may land a step (2^-8
    of its value) apart and take its code along: a code's step is 1/127 of the row's largest value.
    Such values are rare (the gate's FP32 error is below 2^-19 of it, a step of BF16 2^-8: one in
    2^10) and their effect on an output is one term of the sum: 2^-7 * |h| * |w2|. The output is
    FP16 (2^-11 of its value) before the weighted FP32 sum. Rows are compared as vectors: the
    error's norm is below (2^-11 + 2^-7 * sqrt(2^-10) + a hundred FP32 roundings) of the row's."""
    want = moe_plain(x, ids, weights, layer.w13, layer.w13_scales, layer.w2, layer.w2_scales)
    bound = 2.0 ** -11 + 2.0 ** -7 * 2.0 ** -5 + 100 * U
    # The norm of a row's FP16 terms, not of their sum, is what the roundings are relative to.
    size = want.norm(dim=1).max()
    off = (got.double() - want).norm(dim=1)
    assert (off <= 4 * bound * size).all(), (off / size).max().item()


@pytest.mark.parametrize("tokens,hidden,inter,experts,choices,dtype", [
    (1, 64, 32, 4, 2, torch.bfloat16), (33, 256, 96, 6, 2, torch.float32), (200, 512, 256, 8, 3, torch.float16),
    (700, 256, 144, 5, 1, torch.bfloat16)])
def test_int8_layer_against_its_stages(tokens, hidden, inter, experts, choices, dtype):
    layer, x, ids, weights = moe_case(tokens, hidden, inter, experts, choices, dtype)
    got = layer.forward(x, ids, weights)
    assert got.shape == x.shape and got.dtype == torch.float32
    assert_moe(got, x, ids, weights, layer)
    assert torch.equal(got, layer.forward(x, ids.int(), weights))    # whatever the rows' order
    ids[0, 0] = experts + 3                                          # no expert: adds nothing
    dropped = weights.clone()
    dropped[0, 0] = 0
    ids_ok = ids.clone()
    ids_ok[0, 0] = 0
    assert torch.equal(layer.forward(x, ids, weights)[1:], layer.forward(x, ids_ok, dropped)[1:])
    torch.testing.assert_close(layer.forward(x, ids, weights)[0], layer.forward(x, ids_ok, dropped)[0], rtol=0, atol=0)
    assert layer.forward(x[:0], ids[:0], weights[:0]).shape == (0, hidden)
    with pytest.raises(ValueError):
        layer.forward(x[:, :-16], ids, weights)


@pytest.mark.parametrize("tokens", [1, 2, 130, 3000])
def test_int8_layer_of_uneven_routings(tokens):
    """The same expert twice in a token, every token at one expert, ids on both sides of the experts,
    rows of a wider buffer: each equals the layer's stages, and two streams equal one."""
    layer, x, ids, weights = moe_case(tokens, 256, 96, 6, 3)
    wide = torch.full((tokens, 256 + 24), float("nan"), device=DEV, dtype=x.dtype)
    wide[:, 8:264] = x
    for one in (torch.zeros_like(ids), torch.full_like(ids, 5), ids.clone()):
        one[0, 1:] = one[0, 0]
        assert_moe(layer.forward(wide[:, 8:264], one, weights), x, one, weights, layer)
        one[tokens // 2, 0], one[tokens // 3, 1] = -1, 1 << 40
        want = layer.forward(x, one, weights)
        assert_moe(want, x, one, weights, layer)
        streams = [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        got = []
        for turn in range(6):
            with torch.cuda.stream(streams[turn % 2]):
                got.append(layer.forward(x, one, weights))
        torch.cuda.synchronize()
        for other in got:
            assert torch.equal(other, want)
    with pytest.raises(ValueError):
        layer.forward(x, ids, weights.clone().requires_grad_())
    with torch.no_grad():
        layer.forward(x, ids, weights.clone().requires_grad_())
    int8.check_status(DEV)


def test_int8_block_chain_in_a_graph():
    """Two blocks, the first's last norm fused with the second's first, captured and replayed on new
    tokens, equal the same operators called one by one."""
    from harness import moe

    tokens, hidden = 40, 256
    layer, x, _, _ = moe_case(tokens, hidden, 96, 6, 2)
    g = rng_of(77)
    pre, post = (0.5 + torch.rand((2, hidden), device=DEV, generator=g) for _ in range(2))
    gate = torch.randn((2, 4, hidden), device=DEV, generator=g)
    router = torch.randn((hidden, 6), device=DEV, generator=g)
    blocks = [moe.MoEBlock(layer, pre[i], post[i], gate[i], 0.7) for i in range(2)]

    def route(n):
        weights, ids = torch.topk(torch.softmax(n.float() @ router, dim=1), 2, dim=1)
        return ids, weights

    def chain(residual):
        residual, normed = blocks[0].forward(residual, route, next_weight=pre[1])
        return blocks[1].forward(residual, route, normed)[0]

    static = x.clone()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        chain(static)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = chain(static)
    for seed in (1, 2):
        fresh = torch.randn(x.shape, device=DEV, generator=rng_of(seed)).bfloat16()
        static.copy_(fresh)
        graph.replay()
        want = fresh
        for i in range(2):
            n = int8.residual_norm(want, next_weight=pre[i])[1] if i == 0 else n
            y = layer.forward(n, *route(n))
            want, n, _ = int8.residual_norm(y, want, post_weight=post[i], gate=gate[i], residual_scale=0.7,
                                            next_weight=pre[1] if i == 0 else None)
        assert torch.equal(out, want)


def test_block_around_the_fp4_layer():
    """The norms serve the NVFP4 layers as well: the block equals norm, layer, norm."""
    from harness import moe
    from test_gpu_moe import quantised_weights, routing

    device = torch.device(DEV)
    w13, _, w13_blocked = quantised_weights(4, 256, 256, 1, device)
    w2, _, w2_blocked = quantised_weights(4, 256, 128, 2, device)
    layer = moe.RoutedMoELayer(w13, w13_blocked, w2, w2_blocked, max_pairs=128)
    g = rng_of(5)
    residual = torch.randn((50, 256), device=DEV, generator=g).bfloat16()
    pre, post = 0.5 + torch.rand((2, 256), device=DEV, generator=g)
    ids, weights = routing(50, 4, 2, 3, device)
    got, normed = moe.MoEBlock(layer, pre, post).forward(residual, lambda n: (ids, weights), next_weight=pre)
    n = int8.residual_norm(residual, next_weight=pre)[1]
    y = layer.forward(n, ids, weights)
    plain = norm_plain(y, residual, post, None, 1.0, pre, 1e-6)
    assert_norm((got, normed, None), torch.bfloat16, torch.bfloat16, plain)
    layer.close()


def test_offsets_beyond_32_bits():
    """Operands and results whose last elements lie more than 2^31 elements and 2^32 bytes in."""
    g = rng_of(99)
    m, n, k = 70001, 32768, 16
    a, b = make_codes(g, m, k), make_codes(g, n, k)
    sa, sb = torch.rand(m, device=DEV, generator=g), torch.rand(n, device=DEV, generator=g)
    y = int8.gemm(a, b, sa, sb)
    for rows in (slice(0, 3), slice(m - 3, m)):
        assert_product(y[rows], a[rows], b, sa[rows], sb)
    del y
    experts, n, k = 20, 16384, 16384                  # 5.4 GB of weights
    b = torch.empty((experts, n, k), dtype=torch.int8, device=DEV)
    b.view(torch.int32).random_(generator=g)
    a, sa = make_codes(g, 6, k), torch.rand(6, device=DEV, generator=g)
    sb = torch.rand((experts, n), device=DEV, generator=g)
    offsets = torch.zeros(experts + 1, dtype=torch.int32, device=DEV)
    offsets[1:] = 2
    offsets[experts] = 6
    y = int8.grouped_gemm(a, b, sa, sb, offsets, out_dtype=torch.float32)
    assert_product(y[:2], a[:2], b[0], sa[:2], sb[0])
    assert_product(y[2:], a[2:], b[-1], sa[2:], sb[-1])
    del b
    tokens, hidden = 262147, 8200
    x = torch.empty((tokens, hidden), dtype=torch.bfloat16, device=DEV)
    x.normal_(generator=g)
    q, s = int8.quantize_tokens(x)
    assert_quantized((q[-3:], s[-3:]), x[-3:])
    del q
    w = 0.5 + torch.rand(hidden, device=DEV, generator=g)
    out = int8.residual_norm(x, x, post_weight=w, next_weight=w)
    last = tuple(t[-3:] if t is not None else None for t in out)
    assert_norm(last, torch.bfloat16, torch.bfloat16, norm_plain(x[-3:], x[-3:], w, None, 1.0, w, 1e-6))
    del out
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens", [9, 400])
@pytest.mark.parametrize("k", [24, 25, 2048, 2050, 9000, 20008])
def test_quantiser_finds_every_extreme(dtype, tokens, k):
    """The largest magnitude at every kind of place and of either sign, infinities and NaN of either
    sign, in the few-row and many-row kernels of every row length."""
    g = rng_of(k + tokens)
    x = torch.randn((tokens, k), device=DEV, generator=g).to(dtype)
    at = torch.randint(0, k, (tokens,), device=DEV, generator=g)
    at[0], at[1], at[2], at[3] = 0, k - 1, k - 2, k // 2
    sign = torch.where(torch.arange(tokens, device=DEV) % 2 == 0, 1.0, -1.0)
    x[torch.arange(tokens, device=DEV), at] = (sign * 57.0).to(dtype)
    x[5] = -x[5].abs()
    x[6] = x[6].abs()
    assert_quantized(int8.quantize_tokens(x), x)
    for value in (float("inf"), float("-inf"), float("nan"), -float("nan")):
        y = x.clone()
        y[torch.arange(tokens, device=DEV), at] = value
        q, s = int8.quantize_tokens(y)
        assert not q.any() and not torch.isfinite(s).any()
        assert torch.isnan(s).all() if value != value else (s == float("inf")).all()
        _, q, s = int8.residual_norm(y, next_weight=torch.ones(k, device=DEV), quantize=True)
        assert not q.any() and torch.isnan(s).all()


def test_norm_codes_do_not_depend_on_how_rows_lie():
    """The same rows a few at a time and many at once, in whole pieces and one element at a time:
    the same codes and scales, bit for bit (the statistic is taken in 64 bits)."""
    g = rng_of(123)
    for hidden in (640, 4096, 8192, 16384):
        x = torch.randn((600, hidden), device=DEV, generator=g).bfloat16()
        residual = torch.randn((600, hidden), device=DEV, generator=g).half()
        w = 0.5 + torch.rand(hidden, device=DEV, generator=g)
        many = int8.residual_norm(x, residual, post_weight=w, next_weight=w, quantize=True)
        few = int8.residual_norm(x[:3], residual[:3], post_weight=w, next_weight=w, quantize=True)
        shifted = torch.empty((600, hidden + 1), dtype=x.dtype, device=DEV)
        shifted[:, 1:] = x
        single = int8.residual_norm(shifted[:, 1:], residual, post_weight=w, next_weight=w, quantize=True)
        for a, b, c in zip(many, few, single):
            assert torch.equal(a[:3], b) and torch.equal(a, c)


def layer_by_experts(layer, x, ids, weights):
    """(value, bound on the error) of the layer, an expert at a time. The codes and the gate's BF16 rows
    are the operators' own, each tested above; the down projections and their sum are in 64 bits. A down
    projection is an exact sum rounded to FP32 and two FP32 products, and the combine one fused
    multiply-add for each choice: 3 + choices roundings of at most the sum of the terms' sizes."""
    codes, scales = int8.quantize_tokens(x)
    value, size = (torch.zeros(x.shape, dtype=torch.float64, device=DEV) for _ in range(2))
    for e in range(layer.experts):
        token, choice = torch.nonzero(ids == e, as_tuple=True)
        if token.numel() == 0:
            continue
        h = int8.gemm(codes[token], layer.w13[e], scales[token], layer.w13_scales[e], gated=True)
        q, t = int8.quantize_tokens(h)
        y = (q.double() @ layer.w2[e].double().T) * t.double()[:, None] * layer.w2_scales[e].double()
        term = y * weights[token, choice].double()[:, None]
        value.index_add_(0, token, term)
        size.index_add_(0, token, term.abs())
    return value, (4 + ids.shape[1]) * U * size + 1e-40


@pytest.mark.parametrize("tokens,hidden,inter,experts,choices,dtype", [
    (1, 64, 32, 4, 2, torch.bfloat16), (5, 256, 96, 6, 3, torch.float32), (130, 512, 256, 8, 3, torch.float16),
    (700, 256, 144, 5, 1, torch.bfloat16), (3000, 256, 96, 6, 2, torch.bfloat16)])
@pytest.mark.parametrize("large", [1.0, 1e7])
def test_int8_layer_keeps_every_row(tokens, hidden, inter, experts, choices, dtype, large):
    """Each value by its own terms: rows of very different routing weights, weights of zero, and experts
    whose down projections pass the largest FP16 number while the result is an ordinary FP32 one."""
    layer, x, ids, weights = moe_case(tokens, hidden, inter, experts, choices, dtype)
    layer.w2_scales = layer.w2_scales * large
    g = rng_of(tokens + 1)
    weights = weights * torch.exp(4 * torch.randn((tokens, 1), device=DEV, generator=g))
    weights[::3, choices - 1] = 0.0
    want, bound = layer_by_experts(layer, x, ids, weights)
    got = layer.forward(x, ids, weights)
    assert torch.isfinite(got).all()
    assert ((got.double() - want).abs() <= bound).all()
    int8.check_status(DEV)


def test_norm_refuses_an_empty_gate():
    """A gate of no rows is not the same as none: its address is null."""
    x, w = torch.ones((6, 32), device=DEV), torch.ones(32, device=DEV)
    for gates in (0, 4, 7):
        with pytest.raises(ValueError):
            int8.residual_norm(x, x, gate=torch.ones((gates, 32), device=DEV), next_weight=w)
    with pytest.raises(ValueError):
        int8.residual_norm(x[:0], x[:0], gate=torch.ones((0, 32), device=DEV), next_weight=w)
    assert int8.residual_norm(x, x, gate=torch.ones((6, 32), device=DEV), next_weight=w)[0].shape == (6, 32)


def test_norms_and_block_of_no_tokens():
    """A batch without tokens (an expert-parallel rank may have none) gives empty results in every form."""
    from harness import moe

    x, w = torch.ones((0, 256), device=DEV), torch.ones(256, device=DEV)
    for residual in (x, x.bfloat16(), x.half()):
        for post in (None, w):
            for gate in (None, w, w.view(1, 256)):
                call = dict(post_weight=post, gate=gate, residual_scale=0.5)
                r, y, s = int8.residual_norm(x, residual, **call)
                assert r.shape == (0, 256) and r.dtype == residual.dtype and y is None and s is None
                r, y, s = int8.residual_norm(x, residual, next_weight=w, **call)
                assert r.shape == y.shape == (0, 256) and y.dtype == residual.dtype and s is None
                r, y, s = int8.residual_norm(x, residual, next_weight=w, quantize=True, **call)
                assert r.shape == y.shape == (0, 256) and y.dtype == torch.int8 and s.shape == (0,)
    layer, x, ids, weights = moe_case(4, 256, 96, 6, 2)
    block = moe.MoEBlock(layer, w, w, w.view(1, 256), 0.7)
    got, normed = block.forward(x[:0], lambda n: (ids[:0], weights[:0]), next_weight=w)
    assert got.shape == normed.shape == (0, 256)


@pytest.mark.parametrize("hidden", [40, 41, 2048])
def test_norm_with_the_smallest_eps(hidden):
    """Zero rows give zeros with every eps that is taken, rows of subnormals their value."""
    x = torch.zeros((3, hidden), device=DEV)
    x[1] = 1e-40
    w = torch.ones(hidden, device=DEV)
    want = x.double() / (x.double().square().mean(1, keepdim=True) + 1e-77).sqrt()
    _, y, _ = int8.residual_norm(x, next_weight=w, eps=1e-77)
    assert (y[0] == 0).all() and (y[2] == 0).all()
    torch.testing.assert_close(y.double(), want, rtol=4 * U, atol=0)
    _, q, s = int8.residual_norm(x, next_weight=w, eps=1e-77, quantize=True)
    assert not q[0].any() and (q[1] == 127).all() and s[0] == 0 and s[2] == 0
    for eps in (0.9e-77, 1e-100, 5e-324, 0.0, -1e-6):
        with pytest.raises(ValueError):
            int8.residual_norm(x, next_weight=w, eps=eps)


def test_layer_refuses_forward_gradients():
    from torch.autograd import forward_ad

    layer, x, ids, weights = moe_case(4, 256, 96, 6, 2)
    want = layer.forward(x, ids, weights)
    with forward_ad.dual_level():
        for call in (lambda: layer.forward(forward_ad.make_dual(x, torch.ones_like(x)), ids, weights),
                     lambda: layer.forward(x, ids, forward_ad.make_dual(weights, torch.ones_like(weights)))):
            with pytest.raises(ValueError):
                call()
        assert torch.equal(layer.forward(x, ids, weights), want)


@pytest.mark.parametrize("offsets", [[5, 6, 7, 7, 8, 8], [0, 0, 0, 0, -2, 0], [(1 << 31) - 1, 0, 0, -(1 << 31), 3, 3],
                                     [8, 8, 8, 8, 8, 8]])
def test_placement_never_reaches_outside_the_rows(offsets):
    """Offsets that are not those of the ids: pairs whose row would lie outside the buffers have none, and
    nothing beside the rows is written."""
    ids = torch.tensor([[3, 0], [3, 9], [-1, 0], [3, 1]], dtype=torch.int64, device=DEV)
    buffer = torch.full((24,), -9, dtype=torch.int32, device=DEV)
    token_of_row = buffer[8:16]
    row_of_pair, cursors = torch.full((8,), -9, dtype=torch.int32, device=DEV), torch.zeros(5, dtype=torch.int32, device=DEV)
    starts = torch.tensor(offsets, dtype=torch.int32, device=DEV)
    native.moe_place_offsets(ids.data_ptr(), True, 8, 2, 5, starts.data_ptr(), 8, cursors.data_ptr(),
                             row_of_pair.data_ptr(), token_of_row.data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert (buffer[:8] == -9).all() and (buffer[16:] == -9).all()
    # Every expert's pairs have its rows from its offset on, in any order, as far as they lie inside.
    rows = row_of_pair.tolist()
    for e, pairs in ((0, (1, 5)), (1, (7,)), (3, (0, 2, 6))):
        want = [offsets[e] + i if 0 <= offsets[e] + i < 8 else -1 for i in range(len(pairs))]
        assert sorted(rows[i] for i in pairs) == sorted(want)
    assert rows[3] == rows[4] == -1
    tokens = token_of_row.tolist()
    for row, token in enumerate(tokens):
        assert token in ([i // 2 for i in range(8) if rows[i] == row] or [-1])


@pytest.mark.parametrize("m,n,k", [(3, 96, 6832), (277, 256, 5136), (313, 416, 1500), (33, 130, 2049), (842, 40, 9008),
                                   (120, 24, 640), (60, 300, 4097), (2297, 585, 300)])
@pytest.mark.parametrize("gated", [False, True])
def test_groups_of_few_tiles_with_weights_of_their_own(m, n, k, gated):
    """Every expert's weights and scales differ: a product with another expert's fails at any depth."""
    g = rng_of(m * n + k)
    width = 2 * n if gated else n
    a, b = make_codes(g, m, k), make_codes(g, 4, width, k)
    sa = 0.5 + torch.rand(m, device=DEV, generator=g)
    sb = (0.5 + torch.rand((4, width), device=DEV, generator=g)) * (2e-4 / k ** 0.5)
    edges = [0, m // 3, m // 3, m - 1, m]
    offsets = torch.tensor(edges, dtype=torch.int32, device=DEV)
    for dtype in DTYPES:
        out, check = guarded(m, n, dtype)
        int8.grouped_gemm(a, b, sa, sb, offsets, gated=gated, out_dtype=dtype, out=out)
        check()
        for e, (lo, hi) in enumerate(zip(edges, edges[1:])):
            if hi > lo:
                assert_product(out[lo:hi], a[lo:hi], b[e], sa[lo:hi], sb[e], None, gated)
                alone = int8.gemm(a[lo:hi], b[e], sa[lo:hi], sb[e], gated=gated, out_dtype=dtype)
                assert torch.equal(alone, out[lo:hi])
    int8.check_status(DEV)


def test_a_captured_fork_and_join():
    """A product of what two streams made, one of them by a kernel that lets the next begin early: the
    graph waits for both."""
    g = rng_of(61)
    x, residual = (torch.randn((300, 2048), device=DEV, generator=g) for _ in range(2))
    w = 0.5 + torch.rand(2048, device=DEV, generator=g)
    b, sb = int8.quantize_tokens(torch.randn((512, 2048), device=DEV, generator=g))
    offsets = torch.tensor([0, 300], dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream(DEV)

    def work():
        here = torch.cuda.current_stream()
        side.wait_stream(here)
        with torch.cuda.stream(side):
            weights, scales = int8.quantize_tokens(residual[:256])
            scales.record_stream(here)
            weights.record_stream(here)
        _, q, s = int8.residual_norm(x, residual, post_weight=w, next_weight=w, quantize=True)
        here.wait_stream(side)
        y = int8.gemm(q, weights, s, scales, out_dtype=torch.float32)
        return y, int8.grouped_gemm(q, b[None], s, sb[None], offsets)

    work()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for seed in (1, 2, 3):
        for t in (x, residual):
            t.copy_(torch.randn(t.shape, device=DEV, generator=rng_of(seed + 10 * (t is x))))
        graph.replay()
        torch.cuda.synchronize()
        _, q, s = int8.residual_norm(x, residual, post_weight=w, next_weight=w, quantize=True)
        weights, scales = int8.quantize_tokens(residual[:256])
        torch.cuda.synchronize()
        assert torch.equal(out[0], int8.gemm(q, weights, s, scales, out_dtype=torch.float32))
        assert torch.equal(out[1], int8.gemm(q, b, s, sb))


def test_silu_over_its_whole_range():
    """Gates from -1000 to 1000 in FP32, against the accuracy that the header states: two roundings of
    2**-24, the exponential's and the reciprocal's 2**-22 and 2**-23, and 1.25 |gate| 2**-24 from the
    rounding of the exponent; the product by the up value (1 here) is exact."""
    gates = torch.cat([torch.linspace(-87, 87, 40001, device=DEV), torch.linspace(-1000, 1000, 4001, device=DEV),
                       torch.tensor([0.0, -0.0, 1e-30, -1e-30, 1e30, -1e30], device=DEV)])
    n = gates.numel()
    a, b = torch.ones((1, 16), dtype=torch.int8, device=DEV), torch.zeros((2 * n, 16), dtype=torch.int8, device=DEV)
    b[:, 0] = 1
    y = int8.gemm(a, b, torch.ones(1, device=DEV), torch.cat([gates, torch.ones_like(gates)]), gated=True,
                  out_dtype=torch.float32)[0].double()
    g = gates.double()
    want = g * torch.sigmoid(g)
    bound = torch.where(g >= -87, want.abs() * (8 + 1.25 * g.abs()) * U, torch.full_like(g, 1e-35))
    assert ((y - want).abs() <= bound).all()
