"""The operators of the 8-bit and 4-bit formats against their definitions in 64 bits.

Products are tested twice. With whole entries and scales that are powers of two every partial sum is exact in fp32, so the result must be the
exact one, to the last bit (rounded once where the output is bf16): a wrong entry anywhere shows. With real entries the bound counts every
rounding: each of the K additions of a sum is off by at most 2^-23 of the sum of the products' sizes (an fp32 addition rounds by 2^-24; the
tensor cores may cut instead of rounding, which is twice that), and the output's rounding comes on top.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
E4M3 = torch.float8_e4m3fn
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def ops():
    from llm_steadyinfer_b200.csrc import ops as o
    return o


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def status_word():
    return torch.zeros(1, dtype=torch.int32, device=DEV)


# ---- rows to 8 bits ----------------------------------------------------------------------------------------------

def check_rows(out, scale, y, scale_tol):
    """``y``: the exact rows (fp64). The scale is off by ``scale_tol`` at most; a code by half a step of e4m3 (2^-4 of its value, 2^-10 below
    the least normal one) and by what the entry and the scale are off by before they are rounded."""
    want = y.abs().amax(1).clamp_min(2.0 ** -100) / 448
    assert ((scale.double() - want).abs() <= scale_tol * want).all()
    v = y / scale.double().unsqueeze(1)
    off = (out.float().double() - v).abs()
    assert (off <= torch.maximum(v.abs() * 2.0 ** -4, torch.tensor(2.0 ** -10, dtype=F64, device=DEV)) + 2 * scale_tol * v.abs()).all()


def norm_exact(resid, deltas, weight, eps, rows=None):
    h = resid.double()
    for d in deltas:
        h = h + d.double()
    if rows is not None:
        h = h[rows.long()]
    return h, weight.double() * h / torch.sqrt((h * h).mean(1, keepdim=True) + eps)


# width 1,336 has whole chunks of eight; 1,001 and 5 have not; 16,392 is wider than what a block holds in registers
@pytest.mark.parametrize("xdtype,wdtype", [(BF16, BF16), (BF16, F32), (F32, F32), (F32, BF16)])
@pytest.mark.parametrize("R,d", [(1, 4096), (3, 1336), (70, 1001), (2, 5), (1, 1), (300, 2048), (2, 16384), (2, 16392), (40, 4099), (3, 9001), (2, 16383), (2, 16385)])
def test_add_rmsnorm_q8(xdtype, wdtype, R, d):
    g = gen(R * d)
    resid = torch.randn(R, d, generator=g, device=DEV) * 3
    delta, delta2 = (torch.randn(R, d, generator=g, device=DEV).to(xdtype) for _ in range(2))
    weight = (1 + 0.2 * torch.randn(d, generator=g, device=DEV)).to(wdtype)
    # the sum of squares: at most 64 additions in a row (entries a thread, then threads), each off by 2^-24; the stream's own two roundings count twice in
    # a square; the root halves all of that; then the root itself, two products, the quotient and the scale: below 64 * 2^-24 together
    tol = 2.0 ** -18
    for deltas in ((), (delta,), (delta, delta2)):
        h, y = norm_exact(resid, deltas, weight, 1e-5)
        kw = {"delta2": deltas[1]} if len(deltas) == 2 else {}
        out, scale = torch.empty(R, d, dtype=E4M3, device=DEV), torch.full((R,), -1.0, device=DEV)
        stream, dst = resid.clone(), torch.full_like(resid, 7.0)
        ops().add_rmsnorm_q8(stream, deltas[0] if deltas else None, weight, 1e-5, out, scale, dst=dst, **kw)
        assert torch.equal(stream, resid)
        check_rows(out, scale, y, tol)
        # each of the two additions rounds once
        assert ((dst.double() - h).abs() <= 2 * 2.0 ** -24 * (resid.double().abs() + sum(t.double().abs() for t in deltas))).all()
        out2, scale2 = torch.empty_like(out), torch.empty_like(scale)
        ops().add_rmsnorm_q8(stream, deltas[0] if deltas else None, weight, 1e-5, out2, scale2, **kw)          # in place: the same, and the stream moves on
        assert torch.equal(stream, dst if deltas else resid) and torch.equal(out2.view(torch.uint8), out.view(torch.uint8)) and torch.equal(scale2, scale)


@pytest.mark.parametrize("d", [512, 513])
def test_add_rmsnorm_q8_of_chosen_rows(d):
    g = gen(5)
    resid, delta = torch.randn(9, d, generator=g, device=DEV), torch.randn(9, d, generator=g, device=DEV).to(BF16)
    weight = torch.ones(d, device=DEV)
    rows = torch.tensor([8, 0, 0, 3], dtype=torch.int32, device=DEV)                     # out of order, one of them twice
    out, scale = torch.empty(4, d, dtype=E4M3, device=DEV), torch.empty(4, device=DEV)
    before = resid.clone()
    ops().add_rmsnorm_q8(resid, delta, weight, 1e-5, out, scale, rows=rows)
    assert torch.equal(resid, before)
    check_rows(out, scale, norm_exact(resid, (delta,), weight, 1e-5, rows)[1], 2.0 ** -18)
    ahead = torch.zeros(1 << 20, device=DEV)
    out2, scale2 = torch.empty_like(out), torch.empty_like(scale)
    ops().add_rmsnorm_q8(resid, delta, weight, 1e-5, out2, scale2, rows=rows, ahead=ahead)
    assert torch.equal(out2.view(torch.uint8), out.view(torch.uint8)) and torch.equal(scale2, scale)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("R,F,group", [(1, 8192, 8), (5, 1336, 8), (3, 1336, None), (4, 90, 9), (2, 7, 1), (1, 1, None), (200, 2816, 8), (2, 14336, 8),
                                       (2, 16392, 8), (3, 24, 12), (3, 4099, None), (2, 9001, None), (2, 9012, 12), (2, 8200, 4), (2, 16383, None), (2, 16385, 5)])
def test_swiglu_q8(dtype, R, F, group):
    gu = (torch.randn(R, 2 * F, generator=gen(F), device=DEV) * 3).to(dtype)
    out, scale = torch.empty(R, F, dtype=E4M3, device=DEV), torch.empty(R, device=DEV)
    ops().swiglu_q8(gu, out, scale, group)
    f, n = torch.arange(F, device=DEV), group or F
    at = f // n * 2 * n + f % n
    gate, up = gu[:, at].double(), gu[:, at + n].double()
    # the quick exponential is off by 2 + 1.173 |x| units (of 2^-23 of the value), which reach the sum 1 + exp(-g) whole where exp(-g) is large; the sum
    # rounds by half a unit, the quick quotient by two, the product by a half, and the scale's quotient by a half
    check_rows(out, scale, gate / (1 + torch.exp(-gate)) * up, (6 + 1.173 * gate.abs().max().item()) * 2.0 ** -23)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("R,n,stride", [(1, 4096, 4096), (61, 4096, 6144), (7, 1001, 1001), (3, 1000, 1003), (2, 1, 5), (700, 64, 72), (2, 16384, 16384),
                                        (3, 20000, 20000), (3, 4099, 4099), (2, 9001, 9003), (2, 16383, 16383), (2, 16385, 16385)])
def test_quantize_q8(dtype, R, n, stride):
    x = (torch.randn(R, stride, generator=gen(n), device=DEV) * 5).to(dtype)[:, :n]
    out, scale = torch.empty(R, n, dtype=E4M3, device=DEV), torch.empty(R, device=DEV)
    ops().quantize_q8(x, out, scale)
    check_rows(out, scale, x.double(), 2.0 ** -22)            # a quotient and a product
    shifted = torch.empty(R * stride + 1, dtype=dtype, device=DEV)[1:].view(R, stride)[:, :n]      # a base that is not on a 16-byte boundary
    shifted.copy_(x)
    out2, scale2 = torch.empty_like(out), torch.empty_like(scale)
    ops().quantize_q8(shifted, out2, scale2)
    assert torch.equal(out2.view(torch.uint8), out.view(torch.uint8)) and torch.equal(scale2, scale)


@pytest.mark.parametrize("n", [512, 515])
def test_rows_of_zeros_infinities_and_nan(n):
    """A row of zeros has zero codes and a finite scale; entries that are NaN become NaN codes and leave the others alone; with an infinite entry
    the scale is infinite, the entry NaN and the others zero."""
    x = torch.randn(5, n, generator=gen(1), device=DEV)
    x[0] = 0
    x[1, 3] = float("nan")
    x[2, n - 1] = float("inf")
    x[3] *= 1e-38
    x[3, 5] = 3e38
    out, scale = torch.empty(5, n, dtype=E4M3, device=DEV), torch.empty(5, device=DEV)
    ops().quantize_q8(x, out, scale)
    v = out.float()
    assert (v[0] == 0).all() and scale[0].item() > 0
    assert torch.isnan(v[1]).sum() == 1 and torch.isnan(v[1, 3])
    ok = torch.arange(n, device=DEV) != 3
    check_rows(out[1:2, ok], scale[1:2], x[1:2, ok].double(), 2.0 ** -22)
    assert torch.isinf(scale[2]) and torch.isnan(v[2, n - 1]) and (v[2, :n - 1] == 0).all()
    check_rows(out[3:], scale[3:], x[3:].double(), 2.0 ** -22)
    # the norm of a row of zeros, without and with an eps that keeps its root finite
    resid, w = torch.zeros(2, n, device=DEV), torch.ones(n, device=DEV)
    ops().add_rmsnorm_q8(resid, None, w, 1e-30, out[:2], scale[:2])
    assert (out[:2].float() == 0).all() and torch.isfinite(scale[:2]).all()


def test_rows_of_no_rows():
    out, scale = torch.empty(0, 64, dtype=E4M3, device=DEV), torch.empty(0, device=DEV)
    ops().quantize_q8(torch.empty(0, 64, device=DEV), out, scale)
    ops().swiglu_q8(torch.empty(0, 128, device=DEV), out, scale)
    ops().add_rmsnorm_q8(torch.empty(0, 64, device=DEV), None, torch.ones(64, device=DEV), 1e-5, out, scale)


# ---- products of 8-bit rows and weights --------------------------------------------------------------------------

def whole_codes(g, R, n):
    """Entries -8 .. 8, all of them e4m3 values: products up to 64, sums of up to 8,192 of them below 2^24."""
    return torch.randint(-8, 9, (R, n), generator=g, device=DEV).float().to(E4M3)


def powers(g, n):
    return torch.exp2(torch.randint(-6, 7, (n,), generator=g, device=DEV).float())


ROWS = [1, 3, 8, 9, 16, 17, 40, 64, 127, 128, 129, 200, 257, 513]


@pytest.mark.parametrize("M", ROWS)
@pytest.mark.parametrize("N,K", [(256, 512), (1000, 1024), (8, 16), (33, 128), (130, 2816), (1, 8), (17, 5), (64, 136), (2048, 144), (384, 4112)])
def test_gemm_q8_whole_entries(M, N, K):
    g = gen(M * 7 + N + K)
    a, w, sa, sw = whole_codes(g, M, K), whole_codes(g, N, K), powers(g, M), powers(g, N)
    want = torch.mm(a.double(), w.double().t()) * sa.double().unsqueeze(1) * sw.double()
    for dtype in (BF16, F32):
        out, status = torch.full((M, N), float("nan"), dtype=dtype, device=DEV), status_word()
        ops().gemm_q8(a, sa, w, sw, out, status)
        assert status.item() == 0
        assert torch.equal(out, want.to(F32).to(dtype))          # the sum is exact in fp32, the scales only move its exponent


@pytest.mark.parametrize("M,N,K", [(129, 264, 8240), (176, 1000, 8240), (256, 136, 20000), (200, 64, 32768), (136, 4096, 8192), (112, 2048, 2048), (300, 4096, 8192),
                                   (700, 6144, 2048), (8, 28672, 2048), (16, 4096, 4096), (61, 11264, 2048), (1100, 1024, 2816)])
def test_gemm_q8_many_turns(M, N, K):
    """Long rows and many tiles: every stage of shared memory is filled over and over, again and again."""
    g = gen(M + N + K)
    a, w, sa, sw = whole_codes(g, M, K), whole_codes(g, N, K), powers(g, M), powers(g, N)
    want = (torch.mm(a.double(), w.double().t()) * sa.double().unsqueeze(1) * sw.double()).to(F32)
    for _ in range(6):
        out, status = torch.full((M, N), float("nan"), device=DEV), status_word()
        ops().gemm_q8(a, sa, w, sw, out, status)
        assert status.item() == 0 and torch.equal(out, want)


@pytest.mark.parametrize("M,N,K", [(1, 4096, 4096), (8, 2048, 5632), (16, 6144, 4096), (61, 4096, 14336), (128, 1000, 2048), (300, 1336, 2816), (600, 2048, 1000)])
def test_gemm_q8_real_entries(M, N, K):
    g = gen(K)
    a, w = torch.empty(M, K, dtype=E4M3, device=DEV), torch.empty(N, K, dtype=E4M3, device=DEV)
    sa, sw = torch.empty(M, device=DEV), torch.empty(N, device=DEV)
    ops().quantize_q8(torch.randn(M, K, generator=g, device=DEV), a, sa)
    ops().quantize_q8(torch.randn(N, K, generator=g, device=DEV) * 0.02, w, sw)
    scales = sa.double().unsqueeze(1) * sw.double()
    want = torch.mm(a.double(), w.double().t()) * scales
    bound = (K + 2) * 2.0 ** -23 * torch.mm(a.double().abs(), w.double().abs().t()) * scales
    for dtype in (BF16, F32):
        out, status = torch.empty(M, N, dtype=dtype, device=DEV), status_word()
        ops().gemm_q8(a, sa, w, sw, out, status)
        assert status.item() == 0
        off = (out.double() - want).abs()
        assert (off <= bound + (2.0 ** -8 * want.abs() if dtype == BF16 else 0)).all()
        # The bound takes every partial sum as large as all products' sizes together. For entries of random sign a partial sum is about their root
        # of the sum of squares, sqrt(K) where the sizes add up to 0.64 K: K roundings of 2^-24 of it add up to some 2^-23 of the sizes, and
        # cuts (all to one side) of 2^-23 every 32 entries to sqrt(K) / 20 * 2^-23, below 6 * 2^-23 here. 2^-20 of the sizes leaves room, and a kernel
        # that sums in fewer than 32 bits would not keep to it.
        assert (off <= 2.0 ** -20 * bound / ((K + 2) * 2.0 ** -23) + (2.0 ** -8 * want.abs() if dtype == BF16 else 0)).all()


@pytest.mark.parametrize("M", [1, 5, 16, 40, 128, 300])
@pytest.mark.parametrize("K,lda,ldw,shift", [(256, 272, 288, 0), (256, 264, 257, 0), (256, 256, 256, 3), (256, 320, 256, 16)])
def test_gemm_q8_strides_and_alignment(M, K, lda, ldw, shift):
    g = gen(M + lda)
    N = 200

    def laid(rows, ld):
        buf = torch.full((rows * ld + shift,), float("nan"), device=DEV).to(E4M3)          # what lies between the rows is never read into a sum
        t = buf[shift:].view(rows, ld)[:, :K]
        t.copy_(whole_codes(g, rows, K))
        return t

    a, w, sa, sw = laid(M, lda), laid(N, ldw), powers(g, M), powers(g, N)
    want = (torch.mm(a.double(), w.double().t()) * sa.double().unsqueeze(1) * sw.double()).to(F32)
    for dtype, ldo in ((BF16, 200), (BF16, 203), (F32, 208)):
        buf = torch.full((M, ldo), 77.0, dtype=dtype, device=DEV)
        status = status_word()
        ops().gemm_q8(a, sa, w, sw, buf[:, :N], status)
        assert status.item() == 0 and torch.equal(buf[:, :N], want.to(dtype)) and (buf[:, N:] == 77).all()


@pytest.mark.parametrize("M", [2, 40, 200])
def test_gemm_q8_nan_stays_in_its_row_and_column(M):
    g = gen(M)
    N, K = 160, 256
    a, w, sa, sw = whole_codes(g, M, K), whole_codes(g, N, K), powers(g, M), powers(g, N)
    want = torch.mm(a.double(), w.double().t()) * sa.double().unsqueeze(1) * sw.double()
    a[1, 7] = float("nan")
    w[33, 250] = float("nan")
    out = torch.empty(M, N, device=DEV)
    ops().gemm_q8(a, sa, w, sw, out, status_word())
    want[1] = float("nan")
    want[:, 33] = float("nan")
    assert torch.equal(torch.nan_to_num(out, nan=-1e9), torch.nan_to_num(want.to(F32), nan=-1e9))


# ---- products with 4-bit weights ---------------------------------------------------------------------------------

def w4_weight(g, N, K, group, zeros, whole=True):
    """(words, scales, zeros or None, the weight in fp64). ``whole``: scales are powers of two."""
    G = -(-K // group)
    q = torch.randint(0, 16, (N, K), generator=g, device=DEV)
    z = torch.randint(0, 16, (N, G), generator=g, device=DEV).to(torch.uint8) if zeros else None
    if whole:
        s = torch.exp2(torch.randint(-1, 2, (N, G), generator=g, device=DEV).float()).to(BF16)
    else:
        s = (0.002 + 0.01 * torch.rand(N, G, generator=g, device=DEV)).to(BF16)
    at = torch.arange(K, device=DEV) // group
    w = (q.double() - (z.double()[:, at] if zeros else 8.0)) * s.double()[:, at]
    return ops().pack_w4(q), s, z, w


@pytest.mark.parametrize("M", ROWS)
@pytest.mark.parametrize("N,K,group,zeros", [(256, 512, 128, False), (1000, 1024, 128, True), (16, 64, 32, True), (33, 136, 32, False), (130, 2816, 64, True),
                                             (1, 8, 128, False), (64, 200, 64, False), (2048, 384, 256, True), (384, 4104, 128, False), (48, 520, 1024, True)])
def test_gemm_w4_whole_entries(M, N, K, group, zeros):
    """Entries of x -4 .. 4, weights up to 30 in halves: every sum is a multiple of a half, below 2^23."""
    g = gen(M * 3 + N + K)
    words, s, z, w = w4_weight(g, N, K, group, zeros)
    x = torch.randint(-4, 5, (M, K), generator=g, device=DEV).to(BF16)
    want = torch.mm(x.double(), w.t()).to(F32)
    for dtype in (BF16, F32):
        out, status = torch.full((M, N), float("nan"), dtype=dtype, device=DEV), status_word()
        ops().gemm_w4(x, words, s, z, group, out, status)
        assert status.item() == 0
        assert torch.equal(out, want.to(dtype))


@pytest.mark.parametrize("M,N,K,group,zeros", [(1, 4096, 4096, 128, False), (8, 2048, 5632, 64, True), (16, 6144, 4096, 128, True), (61, 4096, 14336, 128, False),
                                               (128, 1000, 2048, 32, True), (300, 1336, 2816, 128, True), (600, 2048, 1000, 256, False)])
def test_gemm_w4_real_entries(M, N, K, group, zeros):
    g = gen(K)
    words, s, z, w = w4_weight(g, N, K, group, zeros, whole=False)
    x = torch.randn(M, K, generator=g, device=DEV).to(BF16)
    want, sizes = torch.mm(x.double(), w.t()), torch.mm(x.double().abs(), w.abs().t())
    for dtype in (BF16, F32):
        out, status = torch.empty(M, N, dtype=dtype, device=DEV), status_word()
        ops().gemm_w4(x, words, s, z, group, out, status)
        assert status.item() == 0
        # many rows round each weight to bf16 once (2^-8 of it); the sums as for 8 bits
        assert ((out.double() - want).abs() <= (2.0 ** -8 + (K + 2) * 2.0 ** -23) * sizes + (2.0 ** -8 * want.abs() if dtype == BF16 else 0)).all()
        # the roundings of the weights are independent: of K entries their sum is far below K times one (six standard deviations of the sum of
        # K roundings spread over +- 2^-8 of each product)
        spread = 6 * 2.0 ** -8 / 3 ** 0.5 * torch.sqrt(torch.mm(x.double() ** 2, (w ** 2).t()))
        assert ((out.double() - want).abs() <= spread + (K + 2) * 2.0 ** -23 * sizes + (2.0 ** -8 * want.abs() if dtype == BF16 else 0)).all()


@pytest.mark.parametrize("M", [1, 5, 16, 40, 128, 300])
@pytest.mark.parametrize("ldx,ldw,shift", [(264, 36, 0), (257, 33, 0), (256, 32, 1), (272, 64, 8)])
def test_gemm_w4_strides_and_alignment(M, ldx, ldw, shift):
    g = gen(M + ldx)
    N, K, group = 200, 256, 64
    words, s, z, w = w4_weight(g, N, K, group, True)
    wbuf = torch.full((N * ldw + shift,), -1, dtype=torch.int32, device=DEV)
    wv = wbuf[shift:].view(N, ldw)[:, :K // 8]
    wv.copy_(words)
    xbuf = torch.full((M * ldx + shift,), float("nan"), dtype=BF16, device=DEV)
    x = xbuf[shift:].view(M, ldx)[:, :K]
    x.copy_(torch.randint(-4, 5, (M, K), generator=g, device=DEV).to(BF16))
    want = torch.mm(x.double(), w.t()).to(F32)
    for dtype, ldo in ((BF16, 200), (BF16, 203), (F32, 208)):
        buf = torch.full((M, ldo), 77.0, dtype=dtype, device=DEV)
        status = status_word()
        ops().gemm_w4(x, wv, s, z, group, buf[:, :N], status)
        assert status.item() == 0 and torch.equal(buf[:, :N], want.to(dtype)) and (buf[:, N:] == 77).all()


@pytest.mark.parametrize("M", [1, 7, 12, 150])
@pytest.mark.parametrize("group", [32, 64, 128, 384])
def test_gemm_w4_scales_anywhere_and_slices_of_k(M, group):
    """Scales and zero points whose first entry lies on no boundary; rows long enough to be cut over several blocks, the last slice shorter."""
    g = gen(M + group)
    N, K = 176, 9984
    words, s, z, w = w4_weight(g, N, K, group, True)
    G = s.shape[1]
    x = torch.randint(-2, 3, (M, K), generator=g, device=DEV).to(BF16)
    want = torch.mm(x.double(), w.t()).to(F32)
    for shift in (0, 1, 3):
        sb, zb = torch.zeros(N * G + shift, dtype=BF16, device=DEV), torch.zeros(N * G + shift, dtype=torch.uint8, device=DEV)
        sv, zv = sb[shift:].view(N, G), zb[shift:].view(N, G)
        sv.copy_(s), zv.copy_(z)
        out, status = torch.empty(M, N, device=DEV), status_word()
        ops().gemm_w4(x, words, sv, zv, group, out, status)
        assert status.item() == 0 and torch.equal(out, want)


@pytest.mark.parametrize("M,N,K,group,zeros", [(12, 4096, 4096, 64, False), (100, 4096, 8192, 32, True), (200, 4096, 4096, 64, False), (700, 6144, 4096, 64, False),
                                               (937, 2048, 8192, 32, True), (333, 4096, 4096, 128, True), (4, 4096, 8192, 32, False), (8, 28672, 2048, 128, True)])
def test_gemm_w4_words_that_name_their_place(M, N, K, group, zeros):
    """Weights that tell their piece of 32 entries and their row, rows of x that pick one piece each: what a slow warp reads out of a stage that has
    already been filled again shows, with many blocks under way and rows long enough for many turns."""
    piece = torch.arange(K, device=DEV) // 32
    q = torch.where(torch.arange(K, device=DEV) % 2 == 0, piece & 15, piece >> 4).to(torch.uint8)
    q = q.expand(N, K) ^ (torch.arange(N, device=DEV).to(torch.uint8) & 15)[:, None]
    G = -(-K // group)
    s, z = torch.ones(N, G, dtype=BF16, device=DEV), torch.full((N, G), 3, dtype=torch.uint8, device=DEV) if zeros else None
    words = ops().pack_w4(q.contiguous())
    x = torch.where(torch.arange(K, device=DEV) % 2 == 0, 1.0, 16.0) * (piece[None] == (torch.arange(M, device=DEV) % (K // 32))[:, None])
    want = torch.mm(x.double(), (q.double() - (3 if zeros else 8)).t()).to(F32)
    for _ in range(6):
        out, status = torch.empty(M, N, device=DEV), status_word()
        ops().gemm_w4(x.to(BF16), words, s, z, group, out, status)
        assert status.item() == 0 and torch.equal(out, want)


@pytest.mark.parametrize("M", [1, 8, 9])
@pytest.mark.parametrize("K", [4352, 8192, 16640, 32768, 33024])
@pytest.mark.parametrize("group", [64, 128])
def test_gemm_w4_rows_longer_than_a_block_holds(M, K, group):
    """Few rows of up to 32,768 entries are cut over a cluster, of more go to the kernel for many: entries -1 .. 1, so that every sum is exact."""
    g = gen(M + K + group)
    N = 83
    words, s, z, w = w4_weight(g, N, K, group, True)
    x = torch.randint(-1, 2, (M, K), generator=g, device=DEV).to(BF16)
    want = torch.mm(x.double(), w.t()).to(F32)
    out, status = torch.full((M, N), float("nan"), device=DEV), status_word()
    ops().gemm_w4(x, words, s, z, group, out, status)
    assert status.item() == 0 and torch.equal(out, want)


@pytest.mark.parametrize("M", [1, 20, 70])
@pytest.mark.parametrize("N,K", [(500, 7000), (90, 4097), (33, 8191), (2000, 2003), (50, 8184), (300, 4088)])
def test_products_of_rows_on_no_boundary_cut_over_blocks(M, N, K):
    g = gen(M + N + K)
    a, w, sa, sw = whole_codes(g, M, K), whole_codes(g, N, K), powers(g, M), powers(g, N)
    want = (torch.mm(a.double(), w.double().t()) * sa.double().unsqueeze(1) * sw.double()).to(F32)
    for _ in range(3):
        out = torch.full((M, N), float("nan"), device=DEV)
        ops().gemm_q8(a, sa, w, sw, out)
        assert torch.equal(out, want)
    if K % 8 == 0:
        words, s, z, w4 = w4_weight(g, N, K, 64, True)
        x = torch.randint(-2, 3, (M, K), generator=g, device=DEV).to(BF16)
        buf = torch.full((M, N + 3), 7.0, device=DEV)
        ops().gemm_w4(x, words, s, z, 64, buf[:, :N])
        assert torch.equal(buf[:, :N], torch.mm(x.double(), w4.t()).to(F32)) and (buf[:, N:] == 7).all()


@pytest.mark.parametrize("M", [2, 40, 200])
def test_gemm_w4_nan_stays_in_its_row_and_column(M):
    g = gen(M)
    N, K, group = 160, 264, 64
    words, s, z, w = w4_weight(g, N, K, group, False)
    x = torch.randint(-4, 5, (M, K), generator=g, device=DEV).to(BF16)
    want = torch.mm(x.double(), w.t()).to(F32)
    x[1, 263] = float("nan")
    s[33, 4] = float("inf")                                     # the last group, of which the row holds eight entries
    want[1] = float("nan")
    out = torch.empty(M, N, device=DEV)
    ops().gemm_w4(x, words, s, z, group, out, status_word())
    keep = torch.arange(N, device=DEV) != 33
    assert torch.equal(torch.nan_to_num(out[:, keep], nan=-1e9), torch.nan_to_num(want[:, keep], nan=-1e9))
    assert not torch.isfinite(out[:, 33]).any() or (w[33, 256:] == 0).all()


@pytest.mark.parametrize("M", [1, 16, 33, 128, 140, 300])
def test_products_repeat_bit_for_bit_and_rows_stand_alone(M):
    """The same inputs give the same bits; a row's result does not change with the rows behind it as long as the kernel is the same one."""
    g = gen(M)
    N, K = 512, 4096
    a, w = torch.empty(M, K, dtype=E4M3, device=DEV), torch.empty(N, K, dtype=E4M3, device=DEV)
    sa, sw = torch.empty(M, device=DEV), torch.empty(N, device=DEV)
    ops().quantize_q8(torch.randn(M, K, generator=g, device=DEV), a, sa)
    ops().quantize_q8(torch.randn(N, K, generator=g, device=DEV), w, sw)
    words, s, z, _ = w4_weight(g, N, K, 128, True, whole=False)
    x = torch.randn(M, K, generator=g, device=DEV).to(BF16)
    first = None
    for _ in range(3):
        out, out4 = torch.empty(M, N, device=DEV), torch.empty(M, N, device=DEV)
        ops().gemm_q8(a, sa, w, sw, out, status_word())
        ops().gemm_w4(x, words, s, z, 128, out4, status_word())
        if first is None:
            first = (out, out4)
        assert torch.equal(out, first[0]) and torch.equal(out4, first[1])


# ---- as they are used: streams, graphs, one behind the other ------------------------------------------------------

def chain(o, g, M, d, F, stream_row, weights):
    """A gated feed-forward in 8 bits on the residual stream, as a layer runs it."""
    x, sx = torch.empty(M, d, dtype=E4M3, device=DEV), torch.empty(M, device=DEV)
    gu, act, sact, y = (torch.empty(M, 2 * F, dtype=BF16, device=DEV), torch.empty(M, F, dtype=E4M3, device=DEV), torch.empty(M, device=DEV),
                        torch.empty(M, d, dtype=BF16, device=DEV))
    st = status_word()

    def run():
        o.add_rmsnorm_q8(stream_row, None, weights["norm"], 1e-5, x, sx)
        o.gemm_q8(x, sx, weights["gu"], weights["sgu"], gu, st)
        o.swiglu_q8(gu, act, sact, 8)
        o.gemm_q8(act, sact, weights["down"], weights["sdown"], y, st)
        return y

    return run, st


@pytest.mark.parametrize("M", [1, 12, 40, 200])
def test_a_feed_forward_in_8_bits_eager_on_a_stream_and_captured(M):
    o, g, d, F = ops(), gen(M), 512, 1408
    w = {"norm": torch.ones(d, device=DEV)}
    wf = {"gu": torch.randn(2 * F, d, generator=g, device=DEV) * 0.05, "down": torch.randn(d, F, generator=g, device=DEV) * 0.05}
    for k, t in wf.items():
        w[k], w["s" + k] = torch.empty(t.shape, dtype=E4M3, device=DEV), torch.empty(t.shape[0], device=DEV)
        o.quantize_q8(t, w[k], w["s" + k])
    h = torch.randn(M, d, generator=g, device=DEV)
    run, st = chain(o, g, M, d, F, h, w)
    want = run().clone()
    # against fp32 weights and activations: two roundings to e4m3 a product, independent over the entries, of 2^-4 / sqrt(3) of each at most;
    # the relative error of a product of many entries is that of one (root of the sum of squares), of the two in turn below twice 0.055
    x = h / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-5)
    gu = (x @ wf["gu"].t()).view(M, -1, 2, 8)
    ref = (torch.nn.functional.silu(gu[:, :, 0]) * gu[:, :, 1]).reshape(M, F) @ wf["down"].t()
    assert (want.float() - ref).norm() <= 0.11 * ref.norm()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run().clone()
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            y = run()
    h2 = torch.randn(M, d, generator=g, device=DEV)
    keep = h.clone()
    h.copy_(h2)
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    replayed = y.clone()
    assert torch.equal(run(), replayed)
    h.copy_(keep)
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want) and st.item() == 0


def test_two_streams_at_once():
    """Two products that run at the same time share nothing."""
    o, g = ops(), gen(3)
    M, N, K = 24, 1024, 4096
    words, s, z, w = w4_weight(g, N, K, 128, True)
    xs = [torch.randint(-4, 5, (M, K), generator=g, device=DEV).to(BF16) for _ in range(2)]
    want = [torch.mm(x.double(), w.t()).to(F32) for x in xs]
    outs = [[torch.empty(M, N, device=DEV) for _ in range(8)] for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(8):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                o.gemm_w4(xs[k], words, s, z, 128, outs[k][i], None)
    torch.cuda.synchronize()
    assert all(torch.equal(outs[k][i], want[k]) for k in range(2) for i in range(8))


@pytest.mark.parametrize("M,N,K", [(17, 24, 4096), (17, 72, 8192), (23, 200, 4096), (33, 40, 14336), (41, 1000, 4096), (65, 104, 8192), (129, 56, 4096), (250, 24, 8192)])
def test_products_whose_blocks_add_up_few_sums(M, N, K):
    """Tiles cut over a cluster whose blocks have, at the end, sums to add for a part of a warp's lanes only, and columns that no lane stores."""
    g = gen(M + N + K)
    a, w, sa, sw = whole_codes(g, M, K), whole_codes(g, N, K), powers(g, M), powers(g, N)
    want = (torch.mm(a.double(), w.double().t()) * sa.double().unsqueeze(1) * sw.double()).to(F32)
    words, s, z, w4 = w4_weight(g, N, K, 128, True)
    x = torch.randint(-1, 2, (M, K), generator=g, device=DEV).to(BF16)
    want4 = torch.mm(x.double(), w4.t()).to(F32)
    for _ in range(3):
        out, out4, status = torch.full((M, N), float("nan"), device=DEV), torch.full((M, N), float("nan"), device=DEV), status_word()
        ops().gemm_q8(a, sa, w, sw, out, status)
        ops().gemm_w4(x, words, s, z, 128, out4, status)
        assert status.item() == 0 and torch.equal(out, want) and torch.equal(out4, want4)


@pytest.mark.parametrize("M", [1, 9, 40, 130, 300])
@pytest.mark.parametrize("K,group,zeros", [(288, 64, False), (288, 128, True), (416, 32, True), (416, 512, False), (4000, 128, False), (2848, 64, True)])
def test_gemm_w4_large_scales_behind_the_rows_end(M, K, group, zeros):
    """Rows that end inside a step, the last group's scale so large that anything but zero times it is infinite in what a step holds beyond the end: its entries
    stand for zero, but for one of size one step beside an x so small that the product is ordinary."""
    g = gen(M + K + group)
    N = 200
    G = -(-K // group)
    q = torch.randint(0, 16, (N, K), generator=g, device=DEV)
    z = torch.randint(1, 15, (N, G), generator=g, device=DEV).to(torch.uint8) if zeros else None
    s = torch.exp2(torch.randint(-1, 2, (N, G), generator=g, device=DEV).float())
    s[:, -1] = 2.0 ** 127
    lo = (G - 1) * group
    q[:, lo:] = z[:, -1:].long() if zeros else 8
    q[:, lo + 1] += torch.randint(-1, 2, (N,), generator=g, device=DEV)
    x = torch.randint(-4, 5, (M, K), generator=g, device=DEV).float()
    x[:, lo + 1] *= 2.0 ** -126
    at = torch.arange(K, device=DEV) // group
    w = (q.double() - (z.double()[:, at] if zeros else 8.0)) * s.double()[:, at]
    want = torch.mm(x.double(), w.t()).to(F32)
    out, status = torch.full((M, N), float("nan"), device=DEV), status_word()
    ops().gemm_w4(x.to(BF16), ops().pack_w4(q), s.to(BF16), z, group, out, status)
    assert status.item() == 0 and torch.equal(out, want)


@pytest.mark.parametrize("M", [1, 8, 16, 40, 128, 300, 600])
@pytest.mark.parametrize("N,K", [(160, 512), (150, 500), (24, 8192), (4096, 256), (61, 4100), (1000, 4096)])
def test_gemm_q8_scales_whose_product_is_no_fp32_number(M, N, K):
    """Scales down to 2^-100 and up to 2^119 (a row's scale is its largest entry over 448): their product may lie beyond fp32 on either side where the result does
    not, and the sum times one of them may where the result does not either. All are powers of two: one rounding, where the result is subnormal."""
    g = gen(M + N + K)
    a, w = whole_codes(g, M, K), whole_codes(g, N, K)
    w[3::7] = 0                                                  # sums that are zero, whatever the scales
    sa = torch.exp2(torch.tensor([-75.0, 0, 119, -100, 60], device=DEV))[torch.arange(M, device=DEV) % 5 if M > 4 else torch.arange(M, device=DEV) + 2]
    sw = torch.exp2(torch.tensor([-75.0, -60, 100, 0, -119, 70, -30], device=DEV))[torch.arange(N, device=DEV) % 7 if N < 1000 else torch.arange(N, device=DEV) // 7 % 7]
    want = (torch.mm(a.double(), w.double().t()) * sa.double().unsqueeze(1) * sw.double()).to(F32)
    for dtype in (F32, BF16):
        out, status = torch.full((M, N), float("nan"), dtype=dtype, device=DEV), status_word()
        ops().gemm_q8(a, sa, w, sw, out, status)
        assert status.item() == 0 and torch.equal(out, want.to(dtype))


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_codes_are_the_nearest_to_the_quotient(dtype, shift):
    """out[r] = x[r] / scale[r] rounded to e4m3, to the bit: every mantissa a row's largest entry can have in bfloat16, beside every bfloat16 entry of the
    fourteen binades below it. Many of them lie halfway between two codes."""
    top = torch.arange(128, 256, device=DEV).float()
    entries = (torch.arange(128, 256, device=DEV).float() * torch.exp2(torch.arange(-14, 1, device=DEV).float()).unsqueeze(1)).reshape(-1)
    x = torch.cat([torch.minimum(entries, top.unsqueeze(1)), top.unsqueeze(1).expand(128, 8)], 1)
    x = x * torch.exp2(torch.arange(128, device=DEV).float() % 5 - 2).unsqueeze(1) * torch.where(torch.arange(x.shape[1], device=DEV) % 2 == 0, 1.0, -1.0)
    n = x.shape[1]
    buf = torch.empty(128 * n + shift, dtype=dtype, device=DEV)[shift:].view(128, n)
    buf.copy_(x)
    out, scale = torch.empty(128, n, dtype=E4M3, device=DEV), torch.empty(128, device=DEV)
    ops().quantize_q8(buf, out, scale)
    # both sides divide in fp32 and then round to e4m3: the same two roundings
    assert torch.equal(scale, (x.abs().amax(1).double() / 448).to(F32))          # (in fp32 torch multiplies by the inverse of a number)
    assert torch.equal(out.float(), (x / scale.unsqueeze(1)).clamp(-448, 448).to(E4M3).float())


@pytest.mark.parametrize("M,m", [(2, 1), (8, 3), (16, 9), (33, 20), (128, 127), (140, 128), (300, 257), (600, 1)])
@pytest.mark.parametrize("K", [4096, 4088])
def test_rows_of_a_product_stand_alone(M, m, K):
    """A row's result does not change with what the rows behind it hold: NaN there, or other numbers."""
    g = gen(M + K)
    N = 520
    a, w = torch.empty(M, K, dtype=E4M3, device=DEV), torch.empty(N, K, dtype=E4M3, device=DEV)
    sa, sw = torch.empty(M, device=DEV), torch.empty(N, device=DEV)
    ops().quantize_q8(torch.randn(M, K, generator=g, device=DEV), a, sa)
    ops().quantize_q8(torch.randn(N, K, generator=g, device=DEV), w, sw)
    words, s, z, _ = w4_weight(g, N, K, 128, True, whole=False)
    x = torch.randn(M, K, generator=g, device=DEV).to(BF16)
    first = None
    for behind in (None, 3.0, float("nan"), float("inf")):
        if behind is not None:
            a[m:], sa[m:], x[m:] = behind, behind, behind
        out, out4, status = torch.empty(M, N, device=DEV), torch.empty(M, N, device=DEV), status_word()
        ops().gemm_q8(a, sa, w, sw, out, status)
        ops().gemm_w4(x, words, s, z, 128, out4, status)
        assert status.item() == 0
        if first is None:
            first = (out, out4)
        assert torch.equal(out[:m], first[0][:m]) and torch.equal(out4[:m], first[1][:m])


@pytest.mark.parametrize("M", [1, 8, 40, 128, 300])
@pytest.mark.parametrize("K,ld", [(250, 256), (257, 272), (1001, 1008), (4090, 4096), (8, 16)])
def test_gemm_q8_rows_that_end_before_their_stride(M, K, ld):
    """Rows on 16-byte boundaries whose length is no multiple of 16: the tcgen05 kernels' last box ends inside the row's padding, which holds NaN."""
    g = gen(M + K)
    N = 200

    def laid(rows):
        buf = torch.full((rows, ld), float("nan"), device=DEV).to(E4M3)
        buf[:, :K] = whole_codes(g, rows, K)
        return buf[:, :K]

    a, w, sa, sw = laid(M), laid(N), powers(g, M), powers(g, N)
    want = (torch.mm(a.double(), w.double().t()) * sa.double().unsqueeze(1) * sw.double()).to(F32)
    out, status = torch.full((M, N), float("nan"), device=DEV), status_word()
    ops().gemm_q8(a, sa, w, sw, out, status)
    assert status.item() == 0 and torch.equal(out, want)


@pytest.mark.parametrize("M", [1, 8, 40, 128, 300])
@pytest.mark.parametrize("K,ldx,ldw", [(1056, 1064, 136), (288, 512, 64), (4000, 4008, 504), (512, 520, 68)])
def test_gemm_w4_rows_that_end_before_their_stride(M, K, ldx, ldw):
    g = gen(M + K)
    N = 200
    words, s, z, w = w4_weight(g, N, K, 32, True)
    wbuf = torch.full((N, ldw), -1, dtype=torch.int32, device=DEV)
    wbuf[:, :K // 8] = words
    xbuf = torch.full((M, ldx), float("nan"), dtype=BF16, device=DEV)
    xbuf[:, :K] = torch.randint(-4, 5, (M, K), generator=g, device=DEV).to(BF16)
    want = torch.mm(xbuf[:, :K].double(), w.t()).to(F32)
    out, status = torch.full((M, N), float("nan"), device=DEV), status_word()
    ops().gemm_w4(xbuf[:, :K], wbuf[:, :K // 8], s, z, 32, out, status)
    assert status.item() == 0 and torch.equal(out, want)


@pytest.mark.parametrize("M", [1, 2, 5, 8])
@pytest.mark.parametrize("N,K,group,zeros", [(2048, 4096, 128, True), (512, 512, 256, False), (1000, 2816, 128, False), (256, 14336, 256, True), (96, 256, 1024, True)])
def test_gemm_w4_few_rows_round_no_weight(M, N, K, group, zeros):
    """Up to eight rows, groups of 128 and more, K a multiple of 256: a weight times its scale is never rounded. The products of x and q - z are exact; a
    product then passes at most 8 instructions of 16 products and a sum (17 additions each), the sum of two chunks of 128, of 16 warps and of 8 blocks, and a
    multiplication by the scale: 162 steps, each off by at most 2^-23 of the products' sizes. One rounding of each weight to bf16 would be off by some
    2^-9 / sqrt(K) of them, ten times as much and more over so many results."""
    g = gen(M + K)
    words, s, z, w = w4_weight(g, N, K, group, zeros, whole=False)
    x = torch.randn(M, K, generator=g, device=DEV).to(BF16)
    want, sizes = torch.mm(x.double(), w.t()), torch.mm(x.double().abs(), w.abs().t())
    out, status = torch.empty(M, N, device=DEV), status_word()
    ops().gemm_w4(x, words, s, z, group, out, status)
    assert status.item() == 0 and ((out.double() - want).abs() <= 162 * 2.0 ** -23 * sizes).all()
    rounded = torch.mm(x.double(), w.to(BF16).double().t())
    assert ((rounded - want).abs() > 162 * 2.0 ** -23 * sizes).any()          # the bound tells the two apart


@pytest.mark.parametrize("captured", [False, True])
def test_norm_takes_a_weight_that_was_just_written(captured):
    o, n = ops(), 4096
    resid, weight = torch.ones(8, n, device=DEV), torch.ones(n, device=DEV, dtype=BF16)
    out, scale = torch.empty(8, n, dtype=E4M3, device=DEV), torch.empty(60, 8, device=DEV)

    def run():
        for i in range(60):
            weight.fill_(2.0 ** (i % 7))
            o.add_rmsnorm_q8(resid, None, weight, 0.0, out, scale[i])

    run()
    if captured:
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            run()
    want = torch.exp2((torch.arange(60, device=DEV) % 7).float()).unsqueeze(1) / 448
    for _ in range(20):
        scale.zero_()
        graph.replay() if captured else run()
        assert ((scale - want).abs() <= 2.0 ** -20 * want).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("F", [64, 4096, 4099, 16390])
def test_swiglu_q8_rows_whose_gates_are_all_far_below_zero(dtype, F):
    """Gates down to where exp(-gate) is fp32's largest (-88.72), with ups so large that the results are ordinary; one row beyond, all zeros."""
    g = gen(F)
    gu = torch.empty(4, 2 * F, device=DEV)
    gu[:, :F] = -80 - 8.6 * torch.rand(4, F, generator=g, device=DEV)
    gu[1, :F] = -88.5
    gu[2, :F] = -87.5
    gu[3, :F] = -89
    gu[:, F:] = torch.randn(4, F, generator=g, device=DEV) * 2.0 ** 110
    gu = gu.to(dtype)
    out, scale = torch.empty(4, F, dtype=E4M3, device=DEV), torch.empty(4, device=DEV)
    ops().swiglu_q8(gu, out, scale)
    gate, up = gu[:3, :F].double(), gu[:3, F:].double()
    check_rows(out[:3], scale[:3], gate / (1 + torch.exp(-gate)) * up, (6 + 1.173 * 89) * 2.0 ** -23)          # as for other gates
    assert (out[3].float() == 0).all() and torch.isfinite(scale[3])


@pytest.mark.parametrize("n", [1000, 1003])
def test_codes_follow_the_quotient_at_every_size_of_a_row(n):
    """Rows from below the least maximum to fp32's largest: codes equal the quotient's to the bit, in every binade."""
    e = torch.arange(-140, 128, device=DEV).double()
    x = ((torch.rand(268, n, generator=gen(n), device=DEV).double() * 2 - 1) * torch.exp2(e).unsqueeze(1)).float()
    out, scale = torch.empty(268, n, dtype=E4M3, device=DEV), torch.empty(268, device=DEV)
    ops().quantize_q8(x, out, scale)
    assert torch.equal(scale, (x.abs().amax(1).clamp_min(2.0 ** -100).double() / 448).float())
    assert torch.equal(out.float(), (x / scale.unsqueeze(1)).clamp(-448, 448).to(E4M3).float())
