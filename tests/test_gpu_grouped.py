"""GPU tests of quantize_rows, gemm_i8, grouped_gemm, grouped_gemm_i8 and the two gradients of grouped_gemm against plain
forms in 64 bits.

Tolerances. 8-bit products: the integer sum is exact; float(sum) and the two scalings round once each (2^-24 relative),
then the result type rounds by half a step. 16-bit products: per step of 16 terms the fp32 accumulator and the step's
partial sum are cut at 2^-23 of at most S = sum |a||b|, and as much again for the terms inside the step, so L terms cost
(L / 16 + 4) * 2^-21 * S; then half a step of the result type (for fp16 at least half its smallest step, 2^-25)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def half_step(exact, dtype):
    rel = torch.finfo(dtype).eps / 2
    floor = {F16: 2.0 ** -25, BF16: 2.0 ** -134, F32: 2.0 ** -150}[dtype]
    return exact.abs() * rel + floor


def assert_within(got, exact, before_rounding):
    """|got - exact| <= error before rounding + half a step at the largest value that error allows."""
    assert torch.isfinite(got).all()
    bound = before_rounding + half_step(exact.abs() + before_rounding, got.dtype)
    off = (got.double() - exact).abs()
    assert (off <= bound).all(), f"off by {off.max().item():.3g}, {(off / bound).max().item():.3g} of the bound"


def product_error(s, terms):
    return (terms / 16 + 4) * 2.0 ** -21 * s


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def halves(g, shape, dtype, ld=None):
    """Normal values in a tensor whose rows are `ld` elements apart (16-byte granular by default)."""
    ld = ld or -(-shape[-1] // 8) * 8
    return torch.randn(*shape[:-1], ld, generator=g, device=DEV).to(dtype)[..., :shape[-1]]


def ints(g, shape, ld=None):
    ld = ld or -(-shape[-1] // 16) * 16
    return torch.randint(-128, 128, (*shape[:-1], ld), generator=g, device=DEV, dtype=torch.int8)[..., :shape[-1]]


def offsets_of(sizes, start=0, dtype=torch.int32):
    out = [start]
    for s in sizes:
        out.append(out[-1] + s)
    return torch.tensor(out, dtype=dtype, device=DEV)


# ------------------------------------------------------------------------------------------ quantize_rows
def quantized(x):
    """The definition: scale a product in fp32, q's quotient in 64 bits, so that no near-tie rounds the wrong way."""
    c = torch.tensor(1 / 127, dtype=F32, device=x.device)
    scale = torch.maximum(x.float().abs().amax(1) * c, torch.tensor(2.0 ** -126, device=x.device))
    q = torch.round(x.double() / scale.double()[:, None])
    ok = torch.isfinite(scale)
    return torch.where(ok[:, None], q, torch.zeros_like(q)).to(torch.int8), scale


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("m,k", [(1, 1), (3, 7), (1, 4096), (130, 1000), (33, 4099), (5, 16384), (2, 40000), (3000, 64), (700, 2056)])
def test_quantize_rows(cuda_ops, clean_status, dtype, m, k):
    x = (torch.randn(m, k, generator=gen(1), device=DEV) * torch.logspace(-3, 3, m, device=DEV)[:, None]).to(dtype)
    q = torch.full((m, k), 77, dtype=torch.int8, device=DEV)
    scale = torch.full((m,), -1.0, device=DEV)
    cuda_ops.quantize_rows(x, q, scale)
    want_q, want_s = quantized(x)
    assert torch.equal(scale, want_s) and torch.equal(q, want_q)


@pytest.mark.parametrize("x_off,ldx,q_off,ldq", [(0, 80, 0, 96), (1, 77, 3, 81), (8, 104, 16, 128), (0, 73, 0, 73)])
def test_quantize_rows_strides_leave_the_rest_alone(cuda_ops, clean_status, x_off, ldx, q_off, ldq):
    m, k = 37, 73
    for dtype in (F16, BF16, F32):
        store = torch.randn(m * ldx + x_off, generator=gen(2), device=DEV).to(dtype)
        x = store[x_off:].as_strided((m, k), (ldx, 1))
        q_store = torch.full((m * ldq + q_off + 8,), 77, dtype=torch.int8, device=DEV)
        q = q_store[q_off:].as_strided((m, k), (ldq, 1))
        scale = torch.empty(m, device=DEV)
        cuda_ops.quantize_rows(x, q, scale)
        want_q, want_s = quantized(x)
        assert torch.equal(q, want_q) and torch.equal(scale, want_s)
        q.fill_(77)
        assert (q_store == 77).all()


def test_quantize_rows_ties_go_to_the_even_integer(cuda_ops, clean_status):
    half = torch.arange(-127, 127, device=DEV) + 0.5
    for top in (127.0, 254.0, 127.0 * 2 ** -10):   # scale 1, 2 and 2^-10: the halves are exact ties
        x = torch.cat([torch.tensor([top], device=DEV), half * (top / 127)])[None]
        q = torch.empty(x.shape, dtype=torch.int8, device=DEV)
        scale = torch.empty(1, device=DEV)
        cuda_ops.quantize_rows(x, q, scale)
        assert scale.item() == top / 127   # a power of two: the rounding of 1/127 is lost in that of the product
        assert torch.equal(q[0, 1:].double(), torch.round(half.double())) and q[0, 0] == 127


def test_quantize_rows_next_to_a_tie(cuda_ops, clean_status):
    """fp32 values one to three steps around (j + 1/2) * scale for scales that are no power of two."""
    rows = []
    for top in (1.0, 3.3, 0.77, 1e-30, 5e30):
        scale = torch.tensor(top, dtype=F32) * torch.tensor(1 / 127, dtype=F32)
        at = ((torch.arange(-127, 127).double() + 0.5) * scale.double()).float()
        row = [torch.tensor([top], dtype=F32)]
        for steps in range(-3, 4):
            v = at.clone()
            for _ in range(abs(steps)):
                v = torch.nextafter(v, torch.full_like(v, math.inf if steps > 0 else -math.inf))
            row.append(v)
        rows.append(torch.cat(row))
    x = torch.stack(rows).to(DEV)
    q = torch.empty(x.shape, dtype=torch.int8, device=DEV)
    scale = torch.empty(x.shape[0], device=DEV)
    cuda_ops.quantize_rows(x, q, scale)
    want_q, want_s = quantized(x)
    assert torch.equal(scale, want_s) and torch.equal(q, want_q)


def test_quantize_rows_zero_tiny_and_undefined_rows(cuda_ops, clean_status):
    x = torch.zeros(6, 300, device=DEV)
    x[1] = torch.randn(300, generator=gen(3), device=DEV) * 1e-40     # subnormal: the scale stays at 2^-126
    x[2, 17] = math.nan
    x[3, 250] = -math.inf
    x[4] = 3.4e38
    x[5, :2] = torch.tensor([math.inf, math.nan])
    q = torch.full(x.shape, 77, dtype=torch.int8, device=DEV)
    scale = torch.empty(6, device=DEV)
    cuda_ops.quantize_rows(x, q, scale)
    assert scale[0].item() == 2.0 ** -126 and scale[1].item() == 2.0 ** -126
    assert math.isnan(scale[2].item()) and scale[3].item() == math.inf and math.isnan(scale[5].item())
    assert (q[0] == 0).all() and (q[2] == 0).all() and (q[3] == 0).all() and (q[5] == 0).all() and (q[4] == 127).all()
    assert torch.equal(q[1], torch.round(x[1].double() / 2.0 ** -126).to(torch.int8))


def test_quantize_rows_no_rows(cuda_ops, clean_status):
    cuda_ops.quantize_rows(torch.empty(0, 8, dtype=F16, device=DEV), torch.empty(0, 8, dtype=torch.int8, device=DEV), torch.empty(0, device=DEV))


# ------------------------------------------------------------------------------------------------ gemm_i8
def i8_exact(a, b, sa, sb):
    return (a.double() @ b.double().t()) * sa.double()[:, None] * sb.double()[None, :]


I8_SHAPES = [(1, 1, 1), (1, 64, 16), (1, 4096, 512), (2, 129, 33), (7, 300, 130), (16, 256, 256), (17, 1000, 1040), (32, 515, 128), (33, 128, 4096),
             (48, 2048, 272), (63, 100, 2000), (64, 640, 640), (65, 257, 96), (100, 1001, 130), (127, 128, 128), (128, 256, 64), (200, 77, 520),
             (255, 255, 255), (257, 513, 300), (300, 4096, 80), (777, 1001, 2064), (1024, 2304, 144), (2500, 3000, 48)]


@pytest.mark.parametrize("out", [F16, BF16, F32])
@pytest.mark.parametrize("m,n,k", I8_SHAPES)
def test_gemm_i8(cuda_ops, clean_status, m, n, k, out):
    g = gen(4)
    a, b = ints(g, (m, k)), ints(g, (n, k))
    sa = (torch.rand(m, generator=g, device=DEV) + 0.5) * 0.01
    sb = (torch.rand(n, generator=g, device=DEV) + 0.5) * 0.01
    c = torch.full((m, n), float("nan"), dtype=out, device=DEV)
    cuda_ops.gemm_i8(a, b, sa, sb, c)
    exact = i8_exact(a, b, sa, sb)
    assert_within(c, exact, exact.abs() * 3.01 * 2.0 ** -24)


def test_gemm_i8_sums_are_exact_up_to_the_largest_k(cuda_ops, clean_status):
    k = 131071
    a = torch.full((3, 131072), -128, dtype=torch.int8, device=DEV)[:, :k]
    b = ints(gen(5), (70, k))
    b[0] = -128
    c = torch.empty(3, 70, device=DEV)
    one = torch.ones(70, device=DEV)
    cuda_ops.gemm_i8(a, b, one[:3].contiguous(), one, c)
    assert torch.equal(c, (a.double() @ b.double().t()).float())
    assert c[0, 0].item() == float(131071 * 16384)


@pytest.mark.parametrize("m", [1, 5, 40, 300])
def test_gemm_i8_strides_and_guard_bands(cuda_ops, clean_status, m):
    n, k = 205, 100
    g = gen(6)
    a, b = ints(g, (m, k), ld=144), ints(g, (n, k), ld=112)
    sa, sb = torch.rand(m, generator=g, device=DEV), torch.rand(n, generator=g, device=DEV)
    exact = i8_exact(a, b, sa, sb)
    for out in (F16, F32):
        for ldc, off in ((n, 0), (n + 3, 1), (216, 8)):
            sa_, sb_ = (sa * 1e-3, sb) if out == F16 else (sa, sb)
            store = torch.full((m * ldc + off + 16,), -7.0, dtype=out, device=DEV)
            c = store[off:].as_strided((m, n), (ldc, 1))
            cuda_ops.gemm_i8(a, b, sa_, sb_, c)
            ex = i8_exact(a, b, sa_, sb_) if out == F16 else exact
            assert_within(c, ex, ex.abs() * 3.01 * 2.0 ** -24)
            c.fill_(-7.0)
            assert (store == -7.0).all()


def test_gemm_i8_scales_pass_through(cuda_ops, clean_status):
    """Zero, negative, infinite and undefined scales act as factors; other rows and columns are not touched by them."""
    g = gen(7)
    a, b = ints(g, (70, 64)), ints(g, (90, 64))
    sa, sb = torch.rand(70, generator=g, device=DEV), torch.rand(90, generator=g, device=DEV)
    sa[3], sa[4], sa[5] = 0.0, -1.0, math.nan
    sb[7] = math.inf
    c = torch.empty(70, 90, device=DEV)
    cuda_ops.gemm_i8(a, b, sa, sb, c)
    want = (a.double() @ b.double().t()).float() * sa[:, None] * sb[None, :]
    assert torch.equal(torch.isnan(c), torch.isnan(want)) and torch.equal(torch.isinf(c), torch.isinf(want))
    fine = torch.isfinite(want)
    assert torch.allclose(c[fine], want[fine], rtol=2.0 ** -22, atol=0)


def test_gemm_i8_no_rows(cuda_ops, clean_status):
    cuda_ops.gemm_i8(torch.empty(0, 16, dtype=torch.int8, device=DEV), ints(gen(8), (4, 16)), torch.empty(0, device=DEV),
                     torch.ones(4, device=DEV), torch.empty(0, 4, device=DEV))


def test_linear_in_8_bits_stays_near_the_unrounded_product(cuda_ops, clean_status):
    """quantize_rows for activations and weights, then gemm_i8, as a program uses them: each factor is off by at most half
    an integer step, so a product of K terms is off by at most sum(|x| sw/2 + |w| sx/2 + sx sw/4)."""
    g = gen(9)
    for m, n, k in ((1, 512, 256), (40, 300, 1024), (500, 640, 512)):
        x, w = halves(g, (m, k), BF16), halves(g, (n, k), BF16)
        qx, qw = (torch.empty(t.shape, dtype=torch.int8, device=DEV) for t in (x, w))
        sx, sw = torch.empty(m, device=DEV), torch.empty(n, device=DEV)
        c = torch.empty(m, n, dtype=BF16, device=DEV)
        cuda_ops.quantize_rows(w, qw, sw)
        cuda_ops.quantize_rows(x, qx, sx)
        cuda_ops.gemm_i8(qx, qw, sx, sw, c)
        exact = x.double() @ w.double().t()
        dx, dw = sx.double()[:, None] / 2, sw.double()[None, :] / 2
        err = x.double().abs().sum(1)[:, None] * dw + w.double().abs().sum(1)[None, :] * dx + k * dx * dw
        assert_within(c, exact, err * 1.001)


# ----------------------------------------------------------------------------------------- grouped products
def plain_forward(a, b, sizes, start):
    out = torch.zeros(a.shape[0], b.shape[1], dtype=torch.float64, device=DEV)
    s = torch.zeros_like(out)
    at = start
    for e, n in enumerate(sizes):
        out[at:at + n] = a[at:at + n].double() @ b[e].double().t()
        s[at:at + n] = a[at:at + n].double().abs() @ b[e].double().abs().t()
        at += n
    return out, s


def plain_wgrad(dc, a, sizes, start):
    out = torch.zeros(len(sizes), dc.shape[1], a.shape[1], dtype=torch.float64, device=DEV)
    s = torch.zeros_like(out)
    at = start
    for e, n in enumerate(sizes):
        out[e] = dc[at:at + n].double().t() @ a[at:at + n].double()
        s[e] = dc[at:at + n].double().abs().t() @ a[at:at + n].double().abs()
        at += n
    return out, s


def inside(total, sizes, start):
    m = torch.zeros(total, dtype=torch.bool, device=DEV)
    m[start:start + sum(sizes)] = True
    return m


# (sizes, first row, rows behind the last group, N, K)
GROUPS = [
    ([1], 0, 0, 1, 1), ([5], 0, 0, 64, 64), ([1, 1, 1], 0, 0, 130, 24), ([0, 3, 0, 2], 2, 3, 257, 136), ([0, 0], 0, 6, 40, 40),
    ([16, 17, 15], 0, 0, 512, 512), ([31, 32, 33, 1], 0, 7, 129, 264), ([64, 63, 2], 1, 0, 1001, 776), ([100, 0, 28], 0, 0, 256, 1000),
    ([128, 127, 129], 0, 3, 300, 72), ([255, 256, 257], 0, 0, 264, 200), ([300, 13, 0, 480], 5, 5, 520, 328), ([1, 700, 2], 0, 0, 384, 88),
    ([77] * 20, 0, 0, 200, 160), ([3] * 64, 0, 1, 320, 640), ([1100, 900], 0, 0, 1280, 1032), ([0] * 9 + [2] + [0] * 9, 0, 0, 128, 2056),
]
# Enough tiles for the kernel that works in pairs of SMs: (N, K) of the forward products, the other way round in the gradient
# to a; the weight gradient takes it for many experts, and cuts long sums over rows in pieces for few.
RAGGED = [300, 129, 0, 255, 257, 16, 511, 1, 200, 330]
WIDE = [(RAGGED, 3, 9, 2000, 136), (RAGGED, 0, 0, 1999, 328), ([700, 650], 0, 5, 8200, 72), ([1, 5000, 2], 0, 0, 1290, 1000)]
WIDE_SUMS = [(RAGGED, 3, 9, 520, 1000), ([16, 32, 48, 15, 17, 0, 127, 128, 129, 143, 144, 145], 0, 1, 777, 1032), ([4101], 2, 1, 200, 136),
             ([2500, 0, 1700], 0, 0, 130, 100), ([9000], 0, 0, 40, 64)]


@pytest.mark.parametrize("dtype,out", [(F16, F16), (BF16, BF16), (F16, F32)])
@pytest.mark.parametrize("sizes,start,behind,n,k", GROUPS + WIDE)
def test_grouped_gemm(cuda_ops, clean_status, sizes, start, behind, n, k, dtype, out):
    g = gen(10)
    total = start + sum(sizes) + behind
    a, b = halves(g, (total, k), dtype), halves(g, (len(sizes), n, k), dtype)
    mask = inside(total, sizes, start)
    a[~mask] = math.nan      # rows outside all groups may hold anything
    c = torch.full((total, n), -7.0, dtype=out, device=DEV)
    cuda_ops.grouped_gemm(a, b, offsets_of(sizes, start), c)
    exact, s = plain_forward(a, b, sizes, start)
    assert_within(c[mask], exact[mask], product_error(s[mask], k))
    assert (c[~mask] == -7.0).all()


@pytest.mark.parametrize("out", [F16, BF16, F32])
@pytest.mark.parametrize("sizes,start,behind,n,k", GROUPS + WIDE)
def test_grouped_gemm_i8(cuda_ops, clean_status, sizes, start, behind, n, k, out):
    g = gen(11)
    total = start + sum(sizes) + behind
    a, b = ints(g, (total, k)), ints(g, (len(sizes), n, k))
    sa = (torch.rand(total, generator=g, device=DEV) + 0.5) * 0.01
    sb = (torch.rand(len(sizes), n, generator=g, device=DEV) + 0.5) * 0.01
    mask = inside(total, sizes, start)
    sa[~mask] = math.nan
    c = torch.full((total, n), -7.0, dtype=out, device=DEV)
    cuda_ops.grouped_gemm_i8(a, b, sa, sb, offsets_of(sizes, start), c)
    exact, _ = plain_forward(a, b, sizes, start)
    group = torch.repeat_interleave(torch.arange(len(sizes), device=DEV), torch.tensor(sizes, device=DEV))
    exact = exact[mask] * sa[mask].double()[:, None] * sb.double()[group]
    assert_within(c[mask], exact, exact.abs() * 3.01 * 2.0 ** -24)
    assert (c[~mask] == -7.0).all()


@pytest.mark.parametrize("dtype,out", [(F16, F16), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("sizes,start,behind,n,k", GROUPS + [(s, a, b, k, n) for s, a, b, n, k in WIDE])
def test_grouped_gemm_dgrad(cuda_ops, clean_status, sizes, start, behind, n, k, dtype, out):
    g = gen(12)
    total = start + sum(sizes) + behind
    dc, b = halves(g, (total, n), dtype), halves(g, (len(sizes), n, k), dtype)
    mask = inside(total, sizes, start)
    dc[~mask] = math.nan
    da = torch.full((total, k), -7.0, dtype=out, device=DEV)
    cuda_ops.grouped_gemm_dgrad(dc, b, offsets_of(sizes, start), da)
    exact, s = plain_forward(dc, b.transpose(1, 2), sizes, start)
    assert_within(da[mask], exact[mask], product_error(s[mask], n))
    assert (da[~mask] == -7.0).all()


@pytest.mark.parametrize("dtype,out", [(F16, F16), (BF16, BF16), (F16, F32)])
@pytest.mark.parametrize("sizes,start,behind,n,k", GROUPS + WIDE_SUMS)
def test_grouped_gemm_wgrad(cuda_ops, clean_status, sizes, start, behind, n, k, dtype, out):
    g = gen(13)
    total = start + sum(sizes) + behind
    dc, a = halves(g, (total, n), dtype), halves(g, (total, k), dtype)
    mask = inside(total, sizes, start)
    dc[~mask] = math.nan
    a[~mask] = math.inf
    db = torch.full((len(sizes), n, k), math.nan, dtype=out, device=DEV)
    cuda_ops.grouped_gemm_wgrad(dc, a, offsets_of(sizes, start), db)
    exact, s = plain_wgrad(dc, a, sizes, start)
    assert_within(db, exact, product_error(s, max(sizes)))
    for e, size in enumerate(sizes):
        if size == 0:
            assert (db[e] == 0).all()


@pytest.mark.parametrize("n,k,scale", [(136, 72, 1), (1300, 1300, 1), (1300, 1300, 5)])
def test_an_undefined_row_stays_with_its_own_group(cuda_ops, clean_status, n, k, scale):
    """NaN and infinities in the last rows of one group and the first of the next must not reach the groups between,
    in any of the three products, and in the forward product not even the other rows of their own group."""
    sizes = [40 * scale, 30 * scale, 21 * scale, 50 * scale]
    g = gen(14)
    total, last, next_ = sum(sizes), sizes[0] - 1, sum(sizes[:3])
    a, b, dc = halves(g, (total, k), F16), halves(g, (4, n, k), F16), halves(g, (total, n), F16)
    a[last], a[next_], dc[last - 1], dc[next_ + 1] = math.nan, math.inf, math.inf, math.nan
    off = offsets_of(sizes)
    c, da = torch.empty(total, n, dtype=F16, device=DEV), torch.empty(total, k, dtype=F16, device=DEV)
    db = torch.empty(4, n, k, dtype=F16, device=DEV)
    cuda_ops.grouped_gemm(a, b, off, c)
    cuda_ops.grouped_gemm_dgrad(dc, b, off, da)
    cuda_ops.grouped_gemm_wgrad(dc, a, off, db)
    assert sorted(torch.nonzero(~torch.isfinite(c).all(1)).flatten().tolist()) == [last, next_]
    assert sorted(torch.nonzero(~torch.isfinite(da).all(1)).flatten().tolist()) == [last - 1, next_ + 1]
    assert [bool(torch.isfinite(db[e]).all()) for e in range(4)] == [False, True, True, False]


def test_grouped_no_rows(cuda_ops, clean_status):
    g = gen(15)
    b, off = halves(g, (3, 24, 16), F16), offsets_of([0, 0, 0])
    none = torch.empty(0, 16, dtype=F16, device=DEV)
    none_n = torch.empty(0, 24, dtype=F16, device=DEV)
    cuda_ops.grouped_gemm(none, b, off, none_n)
    cuda_ops.grouped_gemm_dgrad(none_n, b, off, none)
    for dtype in (F16, F32):
        store = torch.full((3, 26, 19), -7.0, dtype=dtype, device=DEV)
        cuda_ops.grouped_gemm_wgrad(none_n, none, off, store[:, 1:25, 2:18])
        assert (store[:, 1:25, 2:18] == 0).all()
        store[:, 1:25, 2:18] = -7.0
        assert (store == -7.0).all()
    cuda_ops.grouped_gemm_i8(torch.empty(0, 16, dtype=torch.int8, device=DEV), ints(g, (3, 24, 16)), torch.empty(0, device=DEV),
                             torch.ones(3, 24, device=DEV), off, torch.empty(0, 24, device=DEV))


@pytest.mark.parametrize("experts", [1, 33, 1000, 1024])
def test_many_experts_most_of_them_empty(cuda_ops, clean_status, experts):
    sizes = [(3 * e + 1) % 7 if e % 17 == 0 else 0 for e in range(experts)]
    n, k, total = 48, 40, sum(sizes)
    g = gen(16)
    a, b, dc = halves(g, (total, k), BF16), halves(g, (experts, n, k), BF16), halves(g, (total, n), BF16)
    c, da = torch.empty(total, n, dtype=BF16, device=DEV), torch.empty(total, k, dtype=BF16, device=DEV)
    db = torch.full((experts, n, k), math.nan, dtype=BF16, device=DEV)
    off = offsets_of(sizes, dtype=torch.int64)
    cuda_ops.grouped_gemm(a, b, off, c)
    cuda_ops.grouped_gemm_dgrad(dc, b, off, da)
    cuda_ops.grouped_gemm_wgrad(dc, a, off, db)
    exact, s = plain_forward(a, b, sizes, 0)
    assert_within(c, exact, product_error(s, k))
    exact, s = plain_forward(dc, b.transpose(1, 2), sizes, 0)
    assert_within(da, exact, product_error(s, n))
    exact, s = plain_wgrad(dc, a, sizes, 0)
    assert_within(db, exact, product_error(s, 8))


@pytest.mark.parametrize("rows", [50, 700])
def test_strided_operands_and_guard_bands(cuda_ops, clean_status, rows):
    """Expert stacks that are slices of larger ones, or interleaved ([N,E,K] seen as [E,N,K]), rows with gaps."""
    g = gen(17)
    e, n, k = 3, 70, 44
    sizes = [rows // 2, 0, rows - rows // 2]
    off = offsets_of(sizes)
    a, dc = halves(g, (rows, k), F16, ld=64), halves(g, (rows, n), F16, ld=96)
    stacked = torch.randn(5, 80, 56, generator=g, device=DEV).half()[1:4, 3:73, :k]
    interleaved = torch.randn(n, e, 48, generator=g, device=DEV).half().transpose(0, 1)[:, :, :k]
    for b in (stacked, interleaved):
        for out in (F16, F32):
            c_store = torch.full((rows + 2, n + 5), -7.0, dtype=out, device=DEV)
            c = c_store[1:-1, 2:-3]
            cuda_ops.grouped_gemm(a, b, off, c)
            exact, s = plain_forward(a, b, sizes, 0)
            assert_within(c, exact, product_error(s, k))
            c.fill_(-7.0)
            assert (c_store == -7.0).all()
            d_store = torch.full((rows + 2, 64), -7.0, dtype=out, device=DEV)
            da = d_store[1:-1, 8:8 + k]
            cuda_ops.grouped_gemm_dgrad(dc, b, off, da)
            exact, s = plain_forward(dc, b.transpose(1, 2), sizes, 0)
            assert_within(da, exact, product_error(s, n))
            da.fill_(-7.0)
            assert (d_store == -7.0).all()
    exact, s = plain_wgrad(dc, a, sizes, 0)
    for out in (F16, F32):
        for store in (torch.full((e, n + 2, 64), -7.0, dtype=out, device=DEV), torch.full((n + 2, e, 64), -7.0, dtype=out, device=DEV).transpose(0, 1)):
            db = store[:, 1:-1, 8:8 + k]
            cuda_ops.grouped_gemm_wgrad(dc, a, off, db)
            assert_within(db, exact, product_error(s, max(sizes)))
            db.fill_(-7.0)
            assert (store == -7.0).all()


def test_bad_offsets_are_clamped_and_reported(cuda_ops):
    from tiledcuda_b200 import _lib

    g = gen(18)
    n, k, total = 64, 48, 90
    a, b, dc = halves(g, (total, k), F16), halves(g, (4, n, k), F16), halves(g, (total, n), F16)
    for dtype, raw, sizes, start in ((torch.int32, [-5, 20, 10, 60, 1000], [20, 0, 50, 30], 0), (torch.int64, [0, 1 << 40, 7, 7, -(1 << 40)], None, None),
                                     (torch.int32, [2 ** 31 - 1, -2 ** 31, 0, 0, 90], None, None)):
        off = torch.tensor(raw, dtype=dtype, device=DEV)
        c = torch.zeros(total, n, device=DEV)
        db = torch.zeros(4, n, k, device=DEV)
        da = torch.zeros(total, k, device=DEV)
        assert _lib.device_status() == 0
        cuda_ops.grouped_gemm(a, b, off, c)
        assert _lib.device_status() == 16
        cuda_ops.grouped_gemm_dgrad(dc, b, off, da)
        assert _lib.device_status() == 16
        cuda_ops.grouped_gemm_wgrad(dc, a, off, db)
        assert _lib.device_status() == 16
        if sizes is None:
            continue
        # groups after clamping: [0, 20), empty, [10, 60), [60, 90); rows 10..19 are written by the first and the third
        clean = torch.cat([torch.arange(0, 10, device=DEV), torch.arange(20, 90, device=DEV)])
        owner = torch.tensor([0] * 10 + [2] * 40 + [3] * 30, device=DEV)
        exact = torch.einsum("tk,tnk->tn", a[clean].double(), b.double()[owner])
        s = torch.einsum("tk,tnk->tn", a[clean].double().abs(), b.double().abs()[owner])
        assert_within(c[clean], exact, product_error(s, k))


@pytest.mark.parametrize("scale,n,k", [(1, 136, 88), (9, 2600, 2056)])
def test_captured_calls_follow_the_offsets(cuda_ops, clean_status, scale, n, k):
    """One captured graph, replayed with other offsets and data: the sizes are read on the device at every replay."""
    g = gen(19)
    total, e = 333 * scale, 5
    a, b, dc = halves(g, (total, k), F16), halves(g, (e, n, k), F16), halves(g, (total, n), F16)
    off = offsets_of([100 * scale, 0, 33 * scale, 150 * scale, 50 * scale])
    c, da = torch.zeros(total, n, dtype=F16, device=DEV), torch.zeros(total, k, dtype=F16, device=DEV)
    db = torch.zeros(e, n, k, dtype=F16, device=DEV)

    def step():
        cuda_ops.grouped_gemm(a, b, off, c)
        cuda_ops.grouped_gemm_dgrad(dc, b, off, da)
        cuda_ops.grouped_gemm_wgrad(dc, a, off, db)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for sizes in ([333 * scale, 0, 0, 0, 0], [0, 1, 2, 3, 327], [60 * scale, 70, 80, 90, 33 * scale], [0, 0, 0, 0, 0]):
        off.copy_(offsets_of(sizes))
        a.copy_(halves(g, (total, k), F16))
        c.fill_(-7.0)
        graph.replay()
        torch.cuda.synchronize()
        mask = inside(total, sizes, 0)
        exact, s = plain_forward(a, b, sizes, 0)
        assert_within(c[mask], exact[mask], product_error(s[mask], k))
        assert (c[~mask] == -7.0).all()
        exact, s = plain_forward(dc, b.transpose(1, 2), sizes, 0)
        assert_within(da[mask], exact[mask], product_error(s[mask], n))
        exact, s = plain_wgrad(dc, a, sizes, 0)
        assert_within(db, exact, product_error(s, max(sizes)))


def test_calls_on_two_streams_at_once(cuda_ops, clean_status):
    """The operators keep no state between calls: different problems in flight on two streams do not meet."""
    g = gen(20)
    jobs = []
    for seed, (rows, n, k) in enumerate([(900, 512, 256), (40, 640, 1024)]):
        a, b = halves(g, (rows, k), BF16), halves(g, (4, n, k), BF16)
        sizes = [rows // 3, 0, rows // 2, rows - rows // 3 - rows // 2]
        jobs.append((a, b, offsets_of(sizes), torch.zeros(rows, n, dtype=BF16, device=DEV), sizes, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(20):
        for a, b, off, c, _, stream in jobs:
            with torch.cuda.stream(stream):
                cuda_ops.grouped_gemm(a, b, off, c)
    torch.cuda.synchronize()
    for a, b, _, c, sizes, _ in jobs:
        exact, s = plain_forward(a, b, sizes, 0)
        assert_within(c, exact, product_error(s, a.shape[1]))


def test_results_do_not_change_from_run_to_run(cuda_ops, clean_status):
    g = gen(21)
    for rows, n, k in ((20, 1024, 2048), (1500, 520, 264), (3000, 2600, 2600)):
        sizes = [rows // 4, rows // 2, rows - rows // 4 - rows // 2]
        a, b, dc = halves(g, (rows, k), F16), halves(g, (3, n, k), F16), halves(g, (rows, n), F16)
        off = offsets_of(sizes)
        first = None
        for _ in range(3):
            c, da = torch.empty(rows, n, device=DEV), torch.empty(rows, k, device=DEV)
            db = torch.empty(3, n, k, device=DEV)
            cuda_ops.grouped_gemm(a, b, off, c)
            cuda_ops.grouped_gemm_dgrad(dc, b, off, da)
            cuda_ops.grouped_gemm_wgrad(dc, a, off, db)
            if first is None:
                first = (c, da, db)
            else:
                assert all(torch.equal(x, y) for x, y in zip(first, (c, da, db)))


def test_gradients_match_differences(cuda_ops, clean_status):
    """loss = sum(c * dc) is linear in a and in b. With small multiples of 1/8 every sum is exact in fp32, so the change
    of the loss under a change of a (or b) equals the gradient's product with it to the last bit."""
    g = gen(22)
    sizes, n, k = [19, 0, 40, 1], 72, 56
    total = sum(sizes)
    off = offsets_of(sizes)

    def eighths(*shape):
        return (torch.randint(-8, 9, shape, generator=g, device=DEV).float() / 8).half()

    a, b, dc = eighths(total, k), eighths(4, n, k), eighths(total, n)
    da, db = torch.empty(total, k, device=DEV), torch.empty(4, n, k, device=DEV)
    cuda_ops.grouped_gemm_dgrad(dc, b, off, da)
    cuda_ops.grouped_gemm_wgrad(dc, a, off, db)

    def loss(a_, b_):
        c = torch.empty(total, n, device=DEV)
        cuda_ops.grouped_gemm(a_, b_, off, c)
        return (c.double() * dc.double()).sum()

    base = loss(a, b)
    for _ in range(4):
        step_a, step_b = eighths(total, k), eighths(4, n, k)
        assert loss(a + step_a, b) - base == (da.double() * step_a.double()).sum()
        assert loss(a, b + step_b) - base == (db.double() * step_b.double()).sum()


def test_offsets_beyond_31_bits_of_elements(cuda_ops, clean_status):
    """Operands whose elements lie more than 2^31 apart: rows of a and c, experts of b and db."""
    g = gen(23)
    n, k = 64, 48
    big = torch.empty(3 * (1 << 30) + (1 << 20), dtype=F16, device=DEV)
    wide = big.as_strided((4, k), (1 << 30, 1))          # the last row starts 3 * 2^30 elements in
    wide.copy_(halves(g, (4, k), F16))
    b = halves(g, (2, n, k), F16)
    c = torch.empty(4, n, dtype=F16, device=DEV)
    off = offsets_of([2, 2])
    cuda_ops.grouped_gemm(wide, b, off, c)
    exact, s = plain_forward(wide, b, [2, 2], 0)
    assert_within(c, exact, product_error(s, k))
    a = halves(g, (4, k), F16)
    c_wide = big.as_strided((4, n), (1 << 30, 1))
    cuda_ops.grouped_gemm(a, b, off, c_wide)
    exact, s = plain_forward(a, b, [2, 2], 0)
    assert_within(c_wide, exact, product_error(s, k))
    far = big.as_strided((4, n, k), (1 << 30, k, 1))
    far.copy_(halves(g, (4, n, k), F16))
    off4 = offsets_of([1, 1, 1, 1])
    cuda_ops.grouped_gemm(a, far, off4, c)
    exact, s = plain_forward(a, far, [1, 1, 1, 1], 0)
    assert_within(c, exact, product_error(s, k))
    dc = halves(g, (4, n), F16)
    cuda_ops.grouped_gemm_wgrad(dc, a, off4, far)
    exact, s = plain_wgrad(dc, a, [1, 1, 1, 1], 0)
    assert_within(far, exact, product_error(s, 1))


def test_expert_layer_as_a_program_runs_it(cuda_ops, clean_status):
    """Tokens sent to experts, in order: rows gathered by expert, quantised, multiplied in 8 bits, then the 16-bit
    layer and its two gradients on the same groups, and the rows scattered back with scatter_nd."""
    g = gen(24)
    tokens, e, n, k = 300, 6, 256, 192
    x = halves(g, (tokens, k), F16)
    expert = torch.randint(0, e, (tokens,), generator=g, device=DEV)
    order = torch.argsort(expert, stable=True)
    counts = torch.bincount(expert, minlength=e)
    off = torch.zeros(e + 1, dtype=torch.int64, device=DEV)
    off[1:] = counts.cumsum(0)
    sizes = counts.tolist()
    a = x[order].contiguous()
    b = halves(g, (e, n, k), F16)
    qa, sa = torch.empty(tokens, k, dtype=torch.int8, device=DEV), torch.empty(tokens, device=DEV)
    qb, sb = torch.empty(e, n, k, dtype=torch.int8, device=DEV), torch.empty(e, n, device=DEV)
    cuda_ops.quantize_rows(b.view(e * n, k), qb.view(e * n, k), sb.view(e * n))
    cuda_ops.quantize_rows(a, qa, sa)
    c8 = torch.empty(tokens, n, device=DEV)
    cuda_ops.grouped_gemm_i8(qa, qb, sa, sb, off, c8)
    c = torch.empty(tokens, n, dtype=F16, device=DEV)
    cuda_ops.grouped_gemm(a, b, off, c)
    exact, s = plain_forward(a, b, sizes, 0)
    assert_within(c, exact, product_error(s, k))
    owner = expert[order]
    dx, dw = sa.double()[:, None] / 2, sb.double()[owner] / 2
    w_abs = b.double().abs().sum(2)[owner]
    assert_within(c8, exact, (a.double().abs().sum(1)[:, None] * dw + w_abs * dx + k * dx * dw) * 1.001)
    back = torch.zeros(tokens, n, dtype=F16, device=DEV)
    cuda_ops.scatter_nd(back, order[:, None].contiguous(), c)
    assert torch.equal(back[order], c)
    da, db = torch.empty(tokens, k, dtype=F16, device=DEV), torch.empty(e, n, k, dtype=F16, device=DEV)
    cuda_ops.grouped_gemm_dgrad(c, b, off, da)
    cuda_ops.grouped_gemm_wgrad(c, a, off, db)
    exact, s = plain_forward(c, b.transpose(1, 2), sizes, 0)
    assert_within(da, exact, product_error(s, n))
    exact, s = plain_wgrad(c, a, sizes, 0)
    assert_within(db, exact, product_error(s, max(sizes)))


def test_torch_registry_and_python_package(cuda_ops, clean_status):
    """The same calls through torch.ops.tiledcuda and the pytiledcuda package give the same bits."""
    import pytiledcuda as pt

    g = gen(25)
    sizes, n, k = [20, 0, 45], 136, 72
    total, off = sum(sizes), offsets_of(sizes)
    a, b, dc = halves(g, (total, k), BF16), halves(g, (3, n, k), BF16), halves(g, (total, n), BF16)
    pairs = []
    for mod in (cuda_ops, pt):
        q, s = torch.empty(total, k, dtype=torch.int8, device=DEV), torch.empty(total, device=DEV)
        mod.quantize_rows(a, q, s)
        qp = torch.zeros(total, 80, dtype=torch.int8, device=DEV)[:, :k]
        qp.copy_(q)
        qb, sb = ints(gen(26), (3, n, k)), torch.rand(3, n, generator=gen(27), device=DEV)
        c1, c2, c3 = torch.empty(total, n, device=DEV), torch.empty(total, n, dtype=BF16, device=DEV), torch.empty(total, n, dtype=F16, device=DEV)
        da, db = torch.empty(total, k, dtype=BF16, device=DEV), torch.empty(3, n, k, device=DEV)
        mod.gemm_i8(qp, qb[0], s, sb[0], c1)
        mod.grouped_gemm(a, b, off, c2)
        mod.grouped_gemm_i8(qp, qb, s, sb, off, c3)
        mod.grouped_gemm_dgrad(dc, b, off, da)
        mod.grouped_gemm_wgrad(dc, a, off, db)
        pairs.append((q, s, c1, c2, c3, da, db))
    assert all(torch.equal(x, y) for x, y in zip(*pairs))
    with pytest.raises(RuntimeError, match="must be"):
        pt.grouped_gemm(a, b, off[:-1], c2)
    with pytest.raises(RuntimeError, match="must be"):
        pt.gemm_i8(qp, qb[0], s[:-1], sb[0], c1)


def test_the_route_without_the_op_library(cuda_ops, clean_status, monkeypatch):
    """Where libtiledcuda.so has not been built the calls go through ctypes, with the same result."""
    g = gen(29)
    sizes, n, k = [20, 0, 45], 136, 72
    total, off = sum(sizes), offsets_of(sizes)
    a, b, dc = halves(g, (total, k), BF16), halves(g, (3, n, k), BF16), halves(g, (total, n), BF16)
    qb, sb = ints(g, (3, n, k)), torch.rand(3, n, generator=g, device=DEV)
    results = []
    for registered in (None, {}):
        monkeypatch.setattr(cuda_ops, "_registered_ops", registered)
        q = torch.zeros(total, 80, dtype=torch.int8, device=DEV)[:, :k]
        s = torch.empty(total, device=DEV)
        c1, c2, c3 = torch.empty(total, n, device=DEV), torch.empty(total, n, dtype=BF16, device=DEV), torch.empty(total, n, dtype=F16, device=DEV)
        da, db = torch.empty(total, k, dtype=BF16, device=DEV), torch.empty(3, n, k, device=DEV)
        cuda_ops.quantize_rows(a, q, s)
        cuda_ops.gemm_i8(q, qb[0], s, sb[0], c1)
        cuda_ops.grouped_gemm(a, b, off, c2)
        cuda_ops.grouped_gemm_i8(q, qb, s, sb, off, c3)
        cuda_ops.grouped_gemm_dgrad(dc, b, off, da)
        cuda_ops.grouped_gemm_wgrad(dc, a, off, db)
        assert bool(cuda_ops._registered_ops) == (registered is None)
        results.append((q.clone(), s, c1, c2, c3, da, db))
    assert all(torch.equal(x, y) for x, y in zip(*results))


def test_operands_that_require_grad(cuda_ops, clean_status):
    """Parameters may be operands as they are; the operators are not recorded and results require no grad."""
    g = gen(30)
    a, b = halves(g, (40, 64), F16).requires_grad_(), halves(g, (2, 72, 64), F16).requires_grad_()
    off = offsets_of([15, 25])
    c, db = torch.empty(40, 72, dtype=F16, device=DEV), torch.empty(2, 72, 64, dtype=F16, device=DEV)
    cuda_ops.grouped_gemm(a, b, off, c)
    cuda_ops.grouped_gemm_wgrad(c, a, off, db)
    assert not c.requires_grad and not db.requires_grad
    exact, s = plain_forward(a.detach(), b.detach(), [15, 25], 0)
    assert_within(c, exact, product_error(s, 64))
    b.grad = db
    assert b.grad is db


def test_refusals_on_device_tensors(cuda_ops):
    """Wrong types, shapes and strides raise before anything is launched."""
    from tiledcuda_b200 import _lib

    g = gen(28)
    a, b, c = halves(g, (10, 16), F16), halves(g, (2, 24, 16), F16), torch.empty(10, 24, dtype=F16, device=DEV)
    off = offsets_of([4, 6])
    with pytest.raises(TypeError, match="offsets"):
        cuda_ops.grouped_gemm(a, b, off.float(), c)
    with pytest.raises(ValueError, match="offsets"):
        cuda_ops.grouped_gemm(a, b, off[:2], c)
    with pytest.raises(TypeError, match="b must be"):
        cuda_ops.grouped_gemm(a, b.bfloat16(), off, c)
    with pytest.raises(TypeError, match="c must be"):
        cuda_ops.grouped_gemm(a, b, off, c.bfloat16())
    with pytest.raises(ValueError, match="c must be"):
        cuda_ops.grouped_gemm(a, b, off, c[:, :-1])
    with pytest.raises(ValueError, match="inner stride"):
        cuda_ops.grouped_gemm(a, b.transpose(1, 2).contiguous().transpose(1, 2), off, c)
    with pytest.raises(_lib.TiledCudaError, match="row stride"):
        cuda_ops.grouped_gemm(torch.empty(10, 20, dtype=F16, device=DEV)[:, :16], b, off, c)
    with pytest.raises(_lib.TiledCudaError, match="aligned"):
        cuda_ops.grouped_gemm(torch.empty(10, 24, dtype=F16, device=DEV)[:, 1:17], b, off, c)
    with pytest.raises(_lib.TiledCudaError, match="leading dimension|stride"):
        cuda_ops.grouped_gemm(a, b[:1].expand(2, 24, 16), off, c)
    with pytest.raises(_lib.TiledCudaError, match="leading dimension"):
        cuda_ops.grouped_gemm(a, b, off, c[:1].expand(10, 24))
    with pytest.raises(ValueError, match="CUDA"):
        cuda_ops.grouped_gemm(a, b, off.cpu(), c)
    with pytest.raises(ValueError, match="contiguous"):
        cuda_ops.grouped_gemm_i8(a.to(torch.int8), b.to(torch.int8), torch.ones(10, device=DEV), torch.ones(2, 48, device=DEV)[:, :24], off, c)
    with pytest.raises(TypeError, match="scale_a"):
        cuda_ops.gemm_i8(a.to(torch.int8), b[0].to(torch.int8), torch.ones(10, device=DEV, dtype=torch.float64), torch.ones(24, device=DEV), c)


def test_calls_past_the_dispatcher(cuda_ops, clean_status):
    """Plain tensors and parameters skip the dispatcher, with the same result; a subclass or a dispatch mode sees its call."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Seen(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            names.append(func.name())
            return func(*args, **(kwargs or {}))

    class Sub(torch.Tensor):
        pass

    g = gen(31)
    sizes, n, k = [7, 0, 30], 72, 48
    off = offsets_of(sizes)
    a, b = halves(g, (sum(sizes), k), BF16), halves(g, (len(sizes), n, k), BF16)
    c = [torch.full((sum(sizes), n), float("nan"), device=DEV) for _ in range(4)]
    assert cuda_ops._registered("grouped_gemm") is not None
    direct = cuda_ops._direct_calls["grouped_gemm"]
    assert direct(a, torch.nn.Parameter(b), off, c[0]) is True
    names = []
    with Seen():
        assert direct(a, b, off, c[1]) is False
        cuda_ops.grouped_gemm(a, b, off, c[1])
    assert names == ["tiledcuda::grouped_gemm"]
    assert direct(a.as_subclass(Sub), b, off, c[2]) is False
    cuda_ops.grouped_gemm(a.as_subclass(Sub), b, off, c[2])
    assert direct(a, b, off[:-1], c[3]) is False and direct(a, b, off.cpu(), c[3]) is False and direct(a, b, off) is False
    assert bool(c[3].isnan().all())
    cuda_ops.grouped_gemm(a, b, off, c[3])
    assert all(torch.equal(c[0], x) for x in c[1:])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):   # the current stream is the one the call goes to
        c[1].fill_(float("nan"))
        assert direct(a, b, off, c[1]) is True
    side.synchronize()
    assert torch.equal(c[0], c[1])


# Few output tiles and long sums: the sum is cut into two, four or eight pieces, the last of them shorter or empty.
@pytest.mark.parametrize("m,n,k", [(300, 1024, 8192), (290, 1000, 6160), (1, 4096, 4096), (33, 128, 8208), (64, 500, 9000)])
def test_gemm_i8_sums_in_pieces(cuda_ops, clean_status, m, n, k):
    g = gen(32)
    a, b = ints(g, (m, k)), ints(g, (n, k))
    sa, sb = torch.rand(m, generator=g, device=DEV) + 0.5, torch.rand(n, generator=g, device=DEV) + 0.5
    c = torch.full((m, n), float("nan"), device=DEV)
    cuda_ops.gemm_i8(a, b, sa, sb, c)
    exact = i8_exact(a, b, sa, sb)
    assert_within(c, exact, exact.abs() * 3.01 * 2.0 ** -24)


@pytest.mark.parametrize("sizes,start,behind,n,x", [([300], 0, 0, 1024, 3136), ([290], 4, 3, 1000, 3400), ([30, 20, 0, 14], 1, 2, 300, 3200),
                                                    ([2, 1], 0, 0, 200, 5000), ([64], 0, 0, 512, 4200)])
def test_grouped_sums_in_pieces(cuda_ops, clean_status, sizes, start, behind, n, x):
    g = gen(33)
    total, off = start + sum(sizes) + behind, offsets_of(sizes, start)
    a, b = halves(g, (total, x), BF16), halves(g, (len(sizes), n, x), BF16)
    mask = inside(total, sizes, start)
    a[~mask] = math.nan
    exact, s = plain_forward(a, b, sizes, start)
    c = torch.full((total, n), -7.0, device=DEV)
    cuda_ops.grouped_gemm(a, b, off, c)
    assert_within(c[mask], exact[mask], product_error(s[mask], x))
    da = torch.full((total, n), -7.0, device=DEV)
    bt = torch.empty(len(sizes), x, -(-n // 8) * 8, dtype=BF16, device=DEV)[..., :n]
    bt.copy_(b.transpose(1, 2))
    cuda_ops.grouped_gemm_dgrad(a, bt, off, da)
    assert_within(da[mask], exact[mask], product_error(s[mask], x))
    assert (c[~mask] == -7.0).all() and (da[~mask] == -7.0).all()


@pytest.mark.parametrize("sizes,start,n,k", [([3200], 0, 512, 640), ([4096], 3, 512, 512), ([4001, 3000], 0, 320, 300), ([3333], 0, 500, 600)])
def test_wgrad_sums_in_pieces(cuda_ops, clean_status, sizes, start, n, k):
    g = gen(34)
    total = start + sum(sizes)
    dc, a = halves(g, (total, n), F16), halves(g, (total, k), F16)
    db = torch.full((len(sizes), n, k), math.nan, device=DEV)
    cuda_ops.grouped_gemm_wgrad(dc, a, offsets_of(sizes, start), db)
    exact, s = plain_wgrad(dc, a, sizes, start)
    assert_within(db, exact, product_error(s, max(sizes)))


# Around the size where groups with weights of their own change from lone tiles to pairs.
@pytest.mark.parametrize("sizes", [[125] * 16, [100] * 16, [250, 3, 0, 128, 129, 300, 1, 127, 64, 400, 0, 33, 90, 75], [95] * 20, [97] * 20])
@pytest.mark.parametrize("n", [1400, 2056])
def test_uneven_groups_of_about_a_tile(cuda_ops, clean_status, sizes, n):
    g = gen(35)
    k, total, off = 136, sum(sizes) + 2, offsets_of(sizes, 1)
    a, b = halves(g, (total, k), F16), halves(g, (len(sizes), n, k), F16)
    mask = inside(total, sizes, 1)
    exact, s = plain_forward(a, b, sizes, 1)
    c, da = torch.full((total, n), -7.0, dtype=F16, device=DEV), torch.full((total, n), -7.0, dtype=F16, device=DEV)
    cuda_ops.grouped_gemm(a, b, off, c)
    cuda_ops.grouped_gemm_dgrad(a, b.transpose(1, 2).contiguous(), off, da)
    for got in (c, da):
        assert_within(got[mask], exact[mask], product_error(s[mask], k))
        assert (got[~mask] == -7.0).all()


# Sums of more than 8192 terms run in pieces of that length, joined in fp32 to nearest: a piece is off as product_error says, and
# each joining by half a step of the total. One accumulator for the whole sum would be off by 2e-3 of it at 2^20 terms of one sign.
def long_product_error(s, terms):
    return product_error(s, min(terms, 8192)) + -(-terms // 8192) * 2.0 ** -24 * s


def uniform(g, shape, dtype):
    """Values of one sign with full mantissas, in rows that start on 16-byte boundaries."""
    ld = -(-shape[-1] // 8) * 8
    return (torch.rand(*shape[:-1], ld, generator=g, device=DEV) * 0.5 + 0.5).to(dtype)[..., :shape[-1]]


def exact_t(x, y):
    """x^T y in 64 bits, a few rows at a time."""
    out = torch.zeros(x.shape[1], y.shape[1], dtype=torch.float64, device=DEV)
    for i in range(0, x.shape[0], 1 << 14):
        out += x[i:i + (1 << 14)].double().t() @ y[i:i + (1 << 14)].double()
    return out


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("terms,n,k", [(1 << 20, 40, 64), (300007, 136, 24), (65536 + 17, 16, 8), (8192 * 9 + 1, 328, 72)])
def test_long_sums_keep_fp32_accuracy(cuda_ops, clean_status, terms, n, k, dtype):
    g = gen(40)
    dc, a = uniform(g, (terms, n), dtype), uniform(g, (terms, k), dtype)
    exact = exact_t(dc, a)
    db = torch.empty(1, n, k, device=DEV)
    cuda_ops.grouped_gemm_wgrad(dc, a, offsets_of([terms]), db)
    assert_within(db[0], exact, long_product_error(exact, terms))
    x = torch.zeros(n + 2, -(-terms // 8) * 8, dtype=dtype, device=DEV)[1:-1, :terms]
    x.copy_(dc.t())
    w = torch.zeros(1, k, -(-terms // 8) * 8, dtype=dtype, device=DEV)[..., :terms]
    w.copy_(a.t())
    c = torch.empty(n, k, device=DEV)
    cuda_ops.grouped_gemm(x, w, offsets_of([n]), c)
    assert_within(c, exact, long_product_error(exact, terms))
    c.fill_(math.nan)
    cuda_ops.grouped_gemm_dgrad(x, a[None], offsets_of([n]), c)
    assert_within(c, exact, long_product_error(exact, terms))


# Groups on both sides of one, two and three pieces in one call, in the split kernel (whose CTAs may take a part of a sum each)
# and, with enough output tiles, in the kernel of CTA pairs, where short sums follow long ones through the same accumulators.
@pytest.mark.parametrize("dtype,out", [(F16, F32), (BF16, BF16)])
@pytest.mark.parametrize("n,k", [(100, 72), (1300, 776)])
def test_wgrad_of_long_and_short_groups(cuda_ops, clean_status, n, k, dtype, out):
    sizes = [20000, 40, 8192, 8193, 0, 16384, 8207, 16389, 24576 + 5, 100, 8192 + 128, 3]
    g = gen(41)
    total, start = sum(sizes) + 9, 5
    dc, a = uniform(g, (total, n), dtype), uniform(g, (total, k), dtype)
    mask = inside(total, sizes, start)
    dc[~mask] = math.nan
    db = torch.full((len(sizes), n, k), math.nan, dtype=out, device=DEV)
    cuda_ops.grouped_gemm_wgrad(dc, a, offsets_of(sizes, start), db)
    at = start
    for e, size in enumerate(sizes):
        exact = exact_t(dc[at:at + size], a[at:at + size])
        assert_within(db[e], exact, long_product_error(exact, size))
        at += size


@pytest.mark.parametrize("sizes,n", [([3, 0, 20], 72), ([700, 250, 0, 1100], 2600)])
@pytest.mark.parametrize("x", [8192, 16392, 24600])
def test_forward_and_dgrad_of_long_sums(cuda_ops, clean_status, sizes, n, x):
    g = gen(42)
    total, off = sum(sizes) + 4, offsets_of(sizes, 2)
    a, b = uniform(g, (total, x), F16), uniform(g, (len(sizes), n, x), F16)
    mask = inside(total, sizes, 2)
    a[~mask] = math.nan
    exact = torch.zeros(total, n, dtype=torch.float64, device=DEV)
    at = 2
    for e, size in enumerate(sizes):
        exact[at:at + size] = a[at:at + size].double() @ b[e].double().t()
        at += size
    for call, w in ((cuda_ops.grouped_gemm, b), (cuda_ops.grouped_gemm_dgrad, b.transpose(1, 2).contiguous())):
        c = torch.full((total, n), -7.0, device=DEV)
        call(a, w, off, c)
        assert_within(c[mask], exact[mask], long_product_error(exact[mask], x))
        assert (c[~mask] == -7.0).all()


@pytest.mark.parametrize("op", ["gemm_i8", "wgrad"])
def test_the_wait_limit_does_not_count_the_kernel_in_front(cuda_ops, clean_status, op):
    """A GEMM on two SMs that runs for three seconds releases the SMs it does not use at once. The kernel behind it starts there,
    and its waits, limited to two seconds each, must not end before that GEMM does."""
    n, k = 16384, 65536
    b = torch.zeros(n, k, dtype=F16, device=DEV)
    a, c = torch.zeros(65536, k, dtype=F16, device=DEV), torch.empty(65536, n, device=DEV)

    def front(rows):
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        cuda_ops.gemm(a[:rows], b, c[:rows], max_sms=2)
        end.record()
        return start, end

    front(512)
    start, end = front(4096)
    end.synchronize()
    rows = min(65536, math.ceil(3000 / start.elapsed_time(end) * 8) * 512)
    g = gen(43)
    if op == "gemm_i8":
        x, w = ints(g, (2500, 2080)), ints(g, (3000, 2080))
        sx, sw = torch.rand(2500, generator=g, device=DEV) + 0.5, torch.rand(3000, generator=g, device=DEV) + 0.5
        out = torch.full((2500, 3000), math.nan, device=DEV)
        exact = i8_exact(x, w, sx, sw)
        error = exact.abs() * 3.01 * 2.0 ** -24
        call = lambda: cuda_ops.gemm_i8(x, w, sx, sw, out)
    else:
        sizes = [700, 333, 0, 1200, 90]
        dc, x = halves(g, (sum(sizes), 1300), F16), halves(g, (sum(sizes), 776), F16)
        out, off = torch.full((len(sizes), 1300, 776), math.nan, device=DEV), offsets_of(sizes)
        exact, s = plain_wgrad(dc, x, sizes, 0)
        error = product_error(s, max(sizes))
        call = lambda: cuda_ops.grouped_gemm_wgrad(dc, x, off, out)
    torch.cuda.synchronize()
    start, end = front(rows)
    call()
    torch.cuda.synchronize()
    assert start.elapsed_time(end) > 2100, "the kernel in front is over before a wait could run out"
    assert_within(out, exact, error)


def test_a_mode_that_refuses_is_heard(cuda_ops, clean_status):
    """An error that a dispatch mode raises for the call reaches the caller, and nothing is launched behind the mode's back."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class NotHere(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            raise RuntimeError("not here")

    g = gen(44)
    sizes, n, k = [7, 0, 30], 72, 48
    off, total = offsets_of(sizes), sum(sizes)
    a, b, dc = halves(g, (total, k), F16), halves(g, (3, n, k), F16), halves(g, (total, n), F16)
    q, qb, sa, sb = ints(g, (total, k)), ints(g, (3, n, k)), torch.ones(total, device=DEV), torch.ones(3, n, device=DEV)
    new_q, scale = torch.full((total, k), 77, dtype=torch.int8, device=DEV), torch.full((total,), -7.0, device=DEV)
    c, da, db = (torch.full(s, -7.0, dtype=F16, device=DEV) for s in ((total, n), (total, k), (3, n, k)))
    for call in (lambda: cuda_ops.quantize_rows(a, new_q, scale), lambda: cuda_ops.gemm_i8(q, qb[0], sa, sb[0], c),
                 lambda: cuda_ops.grouped_gemm(a, b, off, c), lambda: cuda_ops.grouped_gemm_i8(q, qb, sa, sb, off, c),
                 lambda: cuda_ops.grouped_gemm_dgrad(dc, b, off, da), lambda: cuda_ops.grouped_gemm_wgrad(dc, a, off, db)):
        with NotHere(), pytest.raises(RuntimeError, match="not here"):
            call()
    assert (new_q == 77).all() and all((t == -7.0).all() for t in (scale, c, da, db))


def test_tracers_and_profilers_see_the_calls(cuda_ops, clean_status):
    """torch.jit.trace records the operators, torch.profiler lists them; outside of both a plain call goes past the dispatcher."""
    g = gen(45)
    sizes, n, k = [7, 0, 30], 72, 48
    off, total = offsets_of(sizes), sum(sizes)

    def inputs():
        return [halves(g, (total, k), F16), halves(g, (3, n, k), F16), halves(g, (total, n), F16), ints(g, (3, n, k)),
                torch.rand(3, n, generator=g, device=DEV)]

    def step(a, b, dc, qb, sb):
        q, scale = torch.empty(total, k, dtype=torch.int8, device=DEV), torch.zeros(total, device=DEV)
        c, c1, c8 = torch.zeros(total, n, device=DEV), torch.zeros(total, n, device=DEV), torch.zeros(total, n, device=DEV)
        da, db = torch.zeros(total, k, device=DEV), torch.zeros(3, n, k, device=DEV)
        cuda_ops.quantize_rows(a, q, scale)
        cuda_ops.gemm_i8(q, qb[0], scale, sb[0], c1)
        cuda_ops.grouped_gemm_i8(q, qb, scale, sb, off, c8)
        cuda_ops.grouped_gemm(a, b, off, c)
        cuda_ops.grouped_gemm_dgrad(dc, b, off, da)
        cuda_ops.grouped_gemm_wgrad(dc, a, off, db)
        return q, scale, c1, c8, c, da, db

    names = ["quantize_rows", "gemm_i8", "grouped_gemm_i8", "grouped_gemm", "grouped_gemm_dgrad", "grouped_gemm_wgrad"]
    traced = torch.jit.trace(step, inputs(), check_trace=False)
    recorded = [node.kind() for node in traced.graph.nodes() if node.kind().startswith("tiledcuda::")]
    assert recorded == ["tiledcuda::" + name for name in names]
    other = inputs()
    assert all(torch.equal(x, y) for x, y in zip(traced(*other), step(*other)))
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as prof:
        step(*other)
    listed = {event.key for event in prof.key_averages()}
    assert listed.issuperset("tiledcuda::" + name for name in names)
    a, b = other[:2]
    assert cuda_ops._direct_calls["grouped_gemm"](a, b, off, torch.empty(total, n, device=DEV)) is True


# More than 32 tiles a pair of SMs: the ring in which a pair's tiles are worked out ahead goes round and is filled again.
MANY = [4000, 129, 0, 255, 257, 16, 5111, 1, 3131]


@pytest.mark.parametrize("dtype,out", [(F16, F16), (BF16, F32)])
def test_many_tiles_a_pair_forward_and_dgrad(cuda_ops, clean_status, dtype, out):
    g = gen(46)
    n, k = 12800, 24
    total = sum(MANY) + 3
    few = halves(g, (61, k), dtype)     # few distinct rows, so that the 64-bit products are quick: r and r + 61 are the same
    a = few.repeat(-(-total // 61), 1)[:total]
    b = halves(g, (len(MANY), n, k), dtype)
    off, mask = offsets_of(MANY, 2), inside(total, MANY, 2)
    for call, w in ((cuda_ops.grouped_gemm, b), (cuda_ops.grouped_gemm_dgrad, b.transpose(1, 2).contiguous())):
        c = torch.full((total, n), -7.0, dtype=out, device=DEV)
        call(a, w, off, c)
        at = 2
        for e, size in enumerate(MANY):
            exact = few.double() @ b[e].double().t()
            s = few.double().abs() @ b[e].double().abs().t()
            for i in range(at, at + size, 610):
                rows = torch.arange(i, min(i + 610, at + size), device=DEV)
                assert_within(c[rows], exact[rows % 61], product_error(s[rows % 61], k))
            at += size
        assert (c[~mask] == -7.0).all()


@pytest.mark.parametrize("out", [F16, F32])
def test_many_tiles_a_pair_i8(cuda_ops, clean_status, out):
    g = gen(47)
    m, n, k = 12900, 12800, 48
    few, b = ints(g, (61, k)), ints(g, (n, k))
    a = few.repeat(-(-m // 61), 1)[:m]
    sa = (torch.rand(m, generator=g, device=DEV) + 0.5) * 0.01
    sb = (torch.rand(n, generator=g, device=DEV) + 0.5) * 0.01
    c = torch.full((m, n), math.nan, dtype=out, device=DEV)
    cuda_ops.gemm_i8(a, b, sa, sb, c)
    sums = few.double() @ b.double().t() * sb.double()
    for i in range(0, m, 640):
        rows = torch.arange(i, min(i + 640, m), device=DEV)
        exact = sums[rows % 61] * sa[rows].double()[:, None]
        assert_within(c[rows], exact, exact.abs() * 3.01 * 2.0 ** -24)


@pytest.mark.parametrize("experts,n,k", [(128, 1288, 1288), (150, 1032, 1290)])
@pytest.mark.parametrize("dtype,out", [(F16, F32), (BF16, BF16)])
def test_many_tiles_a_pair_wgrad(cuda_ops, clean_status, experts, n, k, dtype, out):
    g = gen(48)
    sizes = [(7 * e) % 41 for e in range(experts)]
    total = sum(sizes) + 4
    dc, a = halves(g, (total, n), dtype), halves(g, (total, k), dtype)
    dc[:1], a[-3:] = math.nan, math.inf
    db = torch.full((experts, n, k), math.nan, dtype=out, device=DEV)
    cuda_ops.grouped_gemm_wgrad(dc, a, offsets_of(sizes, 1), db)
    at = 1
    for e, size in enumerate(sizes):
        x, y = dc[at:at + size].double(), a[at:at + size].double()
        assert_within(db[e], x.t() @ y, product_error(x.abs().t() @ y.abs(), size))
        at += size


@pytest.mark.parametrize("out", [F16, BF16, F32])
@pytest.mark.parametrize("m,n,k", [(2500, 3000, 1040), (2500, 2999, 777), (4200, 2100, 2300)])
def test_gemm_i8_in_pairs_over_several_stages(cuda_ops, clean_status, m, n, k, out):
    g = gen(49)
    a, b = ints(g, (m, k)), ints(g, (n, k))
    sa = (torch.rand(m, generator=g, device=DEV) + 0.5) * 0.01
    sb = (torch.rand(n, generator=g, device=DEV) + 0.5) * 0.01
    c = torch.full((m, n), math.nan, dtype=out, device=DEV)
    cuda_ops.gemm_i8(a, b, sa, sb, c)
    exact = i8_exact(a, b, sa, sb)
    assert_within(c, exact, exact.abs() * 3.01 * 2.0 ** -24)


# Out of range, decreasing, and groups that own the same rows, more of them than the grid has tiles for (which is made for groups
# that do not overlap): a row is then one of its groups' product or stays as it was, and nothing is written outside of the tensors.
@pytest.mark.parametrize("raw", [[-5, 700, 300, 1500, 5000], [0, 1 << 40, 7, 7, -(1 << 40)], [0, 2000, 0, 2000, 0], [0, 2000, 1, 1999, 0],
                                 [2 ** 31 - 1, -2 ** 31, 0, 2000, 3]])
@pytest.mark.parametrize("total,n,k", [(2000, 2056, 136), (2000, 136, 72)])
def test_bad_offsets_in_both_kernels(cuda_ops, raw, total, n, k):
    from tiledcuda_b200 import _lib

    g = gen(50)
    clamped = [min(max(x, 0), total) for x in raw]
    ranges = [(lo, max(lo, hi)) for lo, hi in zip(clamped, clamped[1:])]
    off = torch.tensor(raw, dtype=torch.int64, device=DEV)
    a, b = halves(g, (total, k), F16), halves(g, (4, n, k), F16)

    def guarded(rows, cols):
        store = torch.full((rows + 2, cols + 16), -7.0, device=DEV)
        return store, store[1:-1, 8:-8]

    def check_rows(store, c):
        own = torch.zeros(total, dtype=torch.long, device=DEV)
        for lo, hi in ranges:
            own[lo:hi] += 1
        assert (c[own == 0] == -7.0).all()
        fits = torch.zeros(c.shape, dtype=torch.bool, device=DEV)
        for e, (lo, hi) in enumerate(ranges):
            exact = a[lo:hi].double() @ b[e].double().t()
            s = a[lo:hi].double().abs() @ b[e].double().abs().t()
            bound = product_error(s, k) + half_step(exact.abs() + product_error(s, k), F32)
            fits[lo:hi] |= (c[lo:hi].double() - exact).abs() <= bound
        if (own > 1).any():
            fits |= c == -7.0
        assert fits[own > 0].all()
        c.fill_(-7.0)
        assert (store == -7.0).all()

    assert _lib.device_status() == 0
    store, c = guarded(total, n)
    cuda_ops.grouped_gemm(a, b, off, c)
    assert _lib.device_status() == 16
    check_rows(store, c)
    cuda_ops.grouped_gemm_dgrad(a, b.transpose(1, 2).contiguous(), off, c)
    assert _lib.device_status() == 16
    check_rows(store, c)
    q, qb, one = ints(g, (total, k)), ints(g, (4, n, k)), torch.ones(4, n, device=DEV)
    cuda_ops.grouped_gemm_i8(q, qb, torch.ones(total, device=DEV), one, off, c)
    assert _lib.device_status() == 16
    overlap = sum(hi - lo for lo, hi in ranges) > sum(1 for t in range(total) if any(lo <= t < hi for lo, hi in ranges))
    right, inside_any = torch.zeros(c.shape, dtype=torch.bool, device=DEV), torch.zeros(total, dtype=torch.bool, device=DEV)
    for e, (lo, hi) in enumerate(ranges):
        right[lo:hi] |= c[lo:hi] == (q[lo:hi].double() @ qb[e].double().t()).float()
        inside_any[lo:hi] = True
    assert (right | (c == -7.0) if overlap else right)[inside_any].all() and (c[~inside_any] == -7.0).all()
    c.fill_(-7.0)
    assert (store == -7.0).all()
    n2, k2 = (1300, 1300) if n > 2000 else (n, k)
    x, y = halves(g, (total, n2), F16), halves(g, (total, k2), F16)
    stores = torch.full((4, n2 + 2, k2 + 16), -7.0, device=DEV)
    db = stores[:, 1:-1, 8:-8]
    cuda_ops.grouped_gemm_wgrad(x, y, off, db)
    assert _lib.device_status() == 16
    for e, (lo, hi) in enumerate(ranges):
        xe, ye = x[lo:hi].double(), y[lo:hi].double()
        assert_within(db[e], xe.t() @ ye, product_error(xe.abs().t() @ ye.abs(), hi - lo))
    db.fill_(-7.0)
    assert (stores == -7.0).all()


def test_calls_from_several_host_threads(cuda_ops, clean_status):
    """Each thread on a stream of its own, through the same entry points at once (the calls give up the interpreter lock)."""
    import threading

    g = gen(51)
    sizes, n, k = [700, 650, 0, 1100, 33], 2056, 136
    total, off = sum(sizes), offsets_of(sizes)
    jobs = []
    for i in range(4):
        a, b, dc = halves(g, (total, k), F16), halves(g, (5, n, k), F16), halves(g, (total, n), F16)
        jobs.append([a, b, dc, torch.empty(total, n, device=DEV), torch.empty(total, k, device=DEV), torch.empty(5, n, k, device=DEV),
                     torch.empty(total, k, dtype=torch.int8, device=DEV), torch.empty(total, device=DEV)])
    torch.cuda.synchronize()
    errors = []

    def work(job):
        try:
            a, b, dc, c, da, db, q, s = job
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(30):
                    cuda_ops.quantize_rows(a, q, s)
                    cuda_ops.grouped_gemm(a, b, off, c)
                    cuda_ops.grouped_gemm_dgrad(dc, b, off, da)
                    cuda_ops.grouped_gemm_wgrad(dc, a, off, db)
                    with pytest.raises(ValueError, match="offsets"):
                        cuda_ops.grouped_gemm(a, b, off[:2], c)
        except BaseException as error:
            errors.append(error)

    threads = [threading.Thread(target=work, args=(job,)) for job in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    torch.cuda.synchronize()
    for a, b, dc, c, da, db, q, s in jobs:
        want_q, want_s = quantized(a)
        assert torch.equal(q, want_q) and torch.equal(s, want_s)
        exact, m = plain_forward(a, b, sizes, 0)
        assert_within(c, exact, product_error(m, k))
        exact, m = plain_forward(dc, b.transpose(1, 2), sizes, 0)
        assert_within(da, exact, product_error(m, n))
        exact, m = plain_wgrad(dc, a, sizes, 0)
        assert_within(db, exact, product_error(m, max(sizes)))
