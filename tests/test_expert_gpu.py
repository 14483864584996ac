"""GPU tests of the expert-layer operators against plain 64-bit references of their formulas.

Tolerances.  A value rounded to a type of machine epsilon eps is off by at most eps/2 of itself (bf16 2^-8, fp16 2^-11, fp32
2^-24, e4m3 2^-4).  A sum of n terms in fp32, each addition off by at most one unit of the 24-bit significand (2^-23 of
the running sum, which covers an adder that truncates), is off by at most n * 2^-23 * sum|terms|.
"""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

F8, F8E5 = torch.float8_e4m3fn, torch.float8_e5m2
TOP = {F8: 448.0, F8E5: 57344.0}
FLOATS = [torch.bfloat16, torch.float16, torch.float32]
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24, F8: 2.0 ** -4, F8E5: 2.0 ** -3}
SMALLEST = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -149}   # subnormal step


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def within(got, want, tol, what=""):
    got, want, tol = got.double().cpu(), want.double().cpu(), tol.double().cpu() if torch.is_tensor(tol) else torch.tensor(tol)
    assert got.shape == want.shape
    over = ((got - want).abs() - tol)
    assert not torch.isnan(over).any() and (over <= 0).all(), f"{what}: {int((over > 0).sum())} of {over.numel()} beyond the bound, worst by {over.max():.3e}"


def rounding(want, dtype):
    return want.abs() * HALF_STEP[dtype] + SMALLEST[dtype] / 2


# ------------------------------------------------------------------------------------------------ quantiser
def quant_ref(x, code, row_block=1):
    """The formula in fp32 on the CPU: codes and scales, bit for bit (a NaN does not enter the maximum)."""
    v = x.float().reshape(-1, x.shape[-1])
    rows, d = v.shape
    kb, rb = -(-d // 128), -(-rows // row_block)
    p = torch.zeros(rb * row_block, kb * 128)
    p[:rows, :d] = v
    p = p.view(rb, row_block, kb, 128)
    top = torch.nan_to_num(p.abs(), nan=0.0, posinf=float("inf")).amax((1, 3))
    s = torch.where(top > 0, torch.clamp(top / TOP[code], min=2.0 ** -126), torch.ones(()))
    y = p * (1.0 / s)[:, None, :, None]
    q = torch.where(torch.isnan(y), y, y.clamp(-TOP[code], TOP[code])).to(code)
    return q.view(torch.uint8).view(rb * row_block, kb * 128)[:rows, :d].reshape(x.shape), s


def activations(g, shape, dtype):
    return (torch.randn(shape, generator=g) * torch.exp(torch.randn(shape[-1], generator=g))).to(dtype)


@pytest.mark.parametrize("code", [F8, F8E5])
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("shape", [(1, 1), (1, 128), (3, 8), (5, 127), (7, 129), (4, 1000), (2, 3, 4096), (129, 640), (33, 5003)])
def test_block_quant_bit_exact(pkg, dev, shape, dtype, code):
    x = activations(gen(11), shape, dtype)
    q, s = pkg.block_quant_fp8(x.to(dev), dtype=code)
    rq, rs = quant_ref(x, code)
    assert torch.equal(s.cpu().reshape(rs.shape), rs)
    assert torch.equal(q.view(torch.uint8).cpu(), rq)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("shape", [(1, 1), (128, 128), (130, 300), (257, 1024), (500, 77)])
def test_tile_quant_bit_exact(pkg, dev, shape, dtype):
    x = activations(gen(12), shape, dtype)
    q, s = pkg.block_quant_fp8(x.to(dev), row_block=128)
    rq, rs = quant_ref(x, F8, 128)
    assert torch.equal(s.cpu(), rs) and torch.equal(q.view(torch.uint8).cpu(), rq)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_block_quant_special_values(pkg, dev, dtype):
    x = torch.zeros(6, 256, dtype=dtype)
    x[1, 3] = float("nan"); x[1, 4] = 2.0
    x[2, 5] = float("inf"); x[2, 6] = -3.0
    x[3, :] = torch.finfo(dtype).max
    x[4, 0] = 2.0 ** -133; x[4, 1] = -(2.0 ** -130)        # subnormal block: the scale stays normal
    x[5, 200] = -0.0
    for code in (F8, F8E5):
        q, s = pkg.block_quant_fp8(x.to(dev), dtype=code)
        rq, rs = quant_ref(x, code)
        assert torch.equal(s.cpu(), rs)
        got, want = q.cpu().float(), rq.view(code).float()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(got, nan=0.0), torch.nan_to_num(want, nan=0.0))


def test_block_quant_unaligned_view(pkg, dev):
    """A row slice whose address is not 16-byte aligned, and codes written at an odd address."""
    x = activations(gen(13), (9, 136), torch.bfloat16)
    flat = torch.empty(9 * 136 + 1, dtype=torch.bfloat16, device=dev)
    flat[1:] = x.to(dev).reshape(-1)
    q, s = pkg.block_quant_fp8(flat[1:].view(9, 136))
    rq, rs = quant_ref(x, F8)
    assert torch.equal(s.cpu(), rs) and torch.equal(q.view(torch.uint8).cpu(), rq)


@pytest.mark.parametrize("code", [F8, F8E5])
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("shape", [(1, 2), (3, 256), (5, 2 * 130), (4, 2 * 77), (300, 2 * 1536), (2, 2, 2 * 4096)])
def test_swiglu_block_quant(pkg, dev, shape, dtype, code):
    x = activations(gen(14), shape, dtype)
    q, s = pkg.swiglu_block_quant_fp8(x.to(dev), dtype=code)
    d = shape[-1] // 2
    a, b = x.double()[..., :d].reshape(-1, d), x.double()[..., d:].reshape(-1, d)
    g = a * torch.sigmoid(a) * b
    # sigmoid in fp32: the exponent's argument is off by 2^-24 of itself (twice: log2 e and the product), the
    # exponential and the quotient by a few units; then two products
    off = g.abs() * (2 * a.abs() * 1.4427 + 12) * 2.0 ** -23
    kb = -(-d // 128)
    pad = lambda v: torch.nn.functional.pad(v, (0, kb * 128 - d)).view(-1, kb, 128)
    want_s = pad(g).abs().amax(-1) / TOP[code]
    within(s.reshape(want_s.shape), want_s, pad(off).amax(-1) / TOP[code] + want_s * 2.0 ** -23 + 2.0 ** -126, "scales")
    sc = s.double().cpu().reshape(-1, kb)
    got = pad(q.double().cpu().reshape(-1, d)) * sc[..., None]
    # the code: half a step of the value, or of the subnormal range (e4m3 2^-9, e5m2 2^-16)
    sub = (2.0 ** -10 if code == F8 else 2.0 ** -17) * sc[..., None]
    within(got, pad(g), pad(off) * 1.125 + torch.maximum(pad(g).abs() * HALF_STEP[code], sub) * (1 + 2.0 ** -20), "values")


# ------------------------------------------------------------------------------------------------ block matmul
def codes(g, rows, k, code):
    x = activations(g, (rows, k), torch.float32)
    q, s = quant_ref(x, code)
    return q.view(code), s


def weights(g, e, k, n, nk):
    a, b = (n, k) if nk else (k, n)
    q = torch.empty((e, a, b), dtype=torch.uint8)
    s = torch.empty((e, -(-a // 128), -(-b // 128)))
    for i in range(e):
        w = torch.randn((a, b), generator=g) * 0.02 * (1 + i % 3)
        q[i], s[i] = quant_ref(w, F8, 128)
    return q.view(F8), s


def mm_ref(x, xs, w, ws, nk):
    """(value, sum of absolute terms) in 64 bits."""
    wide = lambda s, n: s.double().repeat_interleave(128, -1)[..., :n]
    xd = x.double() * wide(xs, x.shape[1])
    wd = w.double() * wide(ws, w.shape[1]).repeat_interleave(128, 0)[:w.shape[0]]
    wd = wd.t() if nk else wd
    return xd @ wd, xd.abs() @ wd.abs()


def mm_tol(want, mag, k, dtype):
    return rounding(want, dtype) + (k + 8) * 2.0 ** -23 * mag


MM_SHAPES = [(1, 1, 1), (1, 128, 128), (3, 130, 70), (1, 4096, 512), (5, 16, 1040), (17, 400, 144), (33, 512, 272), (64, 1040, 2000), (100, 2064, 384),
             (128, 256, 128), (129, 384, 640), (200, 144, 1000), (300, 1152, 528), (513, 640, 1296), (1000, 272, 2064), (16, 7184, 256)]


@pytest.mark.parametrize("nk", [False, True])
@pytest.mark.parametrize("shape", MM_SHAPES)
def test_block_matmul(pkg, dev, shape, nk):
    M, K, N = shape
    g = gen(M * 7 + K + N)
    x, xs = codes(g, M, K, F8)
    w, ws = weights(g, 1, K, N, nk)
    want, mag = mm_ref(x, xs, w[0], ws[0], nk)
    for dtype in FLOATS:
        out = pkg.block_quant_matmul(x.to(dev), xs.to(dev), w[0].to(dev), ws[0].to(dev), transposed=nk, out_dtype=dtype)
        within(out, want, mm_tol(want, mag, K, dtype), f"{shape} {dtype}")


@pytest.mark.parametrize("nk", [False, True])
@pytest.mark.parametrize("kinds", [(F8E5, F8), (F8, F8E5), (F8E5, F8E5)])
@pytest.mark.parametrize("M", [2, 48, 300])
def test_block_matmul_e5m2(pkg, dev, kinds, M, nk):
    K, N = 528, 400
    g = gen(M)
    x, xs = codes(g, M, K, kinds[0])
    w = torch.randn((N, K) if nk else (K, N), generator=g)
    q, ws = quant_ref(w, kinds[1], 128)
    w = q.view(kinds[1])
    want, mag = mm_ref(x, xs, w, ws, nk)
    out = pkg.block_quant_matmul(x.to(dev), xs.to(dev), w.to(dev), ws.to(dev), transposed=nk, out_dtype=torch.float32)
    within(out, want, mm_tol(want, mag, K, torch.float32))


# rows that do not start on 16 bytes, on four, on any boundary; both types on both sides, long enough for several blocks of K
@pytest.mark.parametrize("nk", [False, True])
@pytest.mark.parametrize("kinds", [(F8, F8), (F8E5, F8), (F8, F8E5), (F8E5, F8E5)])
@pytest.mark.parametrize("shape", [(70, 516, 204), (5, 519, 206), (130, 129, 67), (64, 2, 3), (200, 1027, 129)])
def test_block_matmul_odd_rows(pkg, dev, shape, kinds, nk):
    (M, K, N), (tx, tw) = shape, kinds
    g = gen(M + K)
    x, xs = codes(g, M, K, tx)
    w, ws = quant_ref(torch.randn((N, K) if nk else (K, N), generator=g), tw, 128)
    w = w.view(tw)
    want, mag = mm_ref(x, xs, w, ws, nk)
    for dtype in FLOATS:
        out = pkg.block_quant_matmul(x.to(dev), xs.to(dev), w.to(dev), ws.to(dev), transposed=nk, out_dtype=dtype)
        within(out, want, mm_tol(want, mag, K, dtype), f"{dtype}")


@pytest.mark.parametrize("nk", [False, True])
@pytest.mark.parametrize("M", [4, 96, 260])
def test_block_matmul_tail_meets_nan_codes(pkg, dev, M, nk):
    """K ends inside a block and N inside a tile: what lies behind the ends (the next rows' codes, here the next
    tensor's NaN codes) takes no part."""
    K, N = 336, 208
    g = gen(M + 1)
    x, xs = codes(g, M, K, F8)
    w, ws = weights(g, 1, K, N, nk)
    def surrounded(t):
        t = t.contiguous().view(torch.uint8).reshape(-1)
        buf = torch.full((t.numel() + 65536,), 0x7F, dtype=torch.uint8, device=dev)
        buf[32768:32768 + t.numel()] = t.to(dev)
        return buf[32768:32768 + t.numel()]
    xd = surrounded(x).view(F8).view(M, K)
    wd = surrounded(w[0]).view(F8).view(w[0].shape)
    want, mag = mm_ref(x, xs, w[0], ws[0], nk)
    out = pkg.block_quant_matmul(xd, xs.to(dev), wd, ws[0].to(dev), transposed=nk, out_dtype=torch.float32)
    within(out, want, mm_tol(want, mag, K, torch.float32))


def test_block_matmul_special_values(pkg, dev):
    """A NaN code reaches its row only; a zero scale gives zeros; an infinite scale gives what the formula gives."""
    for M in (6, 200):
        K, N = 384, 256
        g = gen(M)
        x, xs = codes(g, M, K, F8)
        w, ws = weights(g, 1, K, N, True)
        x.view(torch.uint8)[2, 130] = 0x7F
        xs[3, :] = 0.0
        xs[4, 1] = float("inf")
        out = pkg.block_quant_matmul(x.to(dev), xs.to(dev), w[0].to(dev), ws[0].to(dev), transposed=True, out_dtype=torch.float32).cpu()
        assert torch.isnan(out[2]).all() and (out[3] == 0).all() and not torch.isfinite(out[4]).any()
        rest = [i for i in range(M) if i not in (2, 3, 4)]
        want, mag = mm_ref(x[rest], xs[rest], w[0], ws[0], True)
        within(out[rest], want, mm_tol(want, mag, K, torch.float32))


@pytest.mark.parametrize("M", [3, 70, 400])
def test_block_matmul_unaligned_pointers(pkg, dev, M):
    K, N = 256, 320
    g = gen(M)
    x, xs = codes(g, M, K, F8)
    w, ws = weights(g, 1, K, N, False)
    def shifted(t):
        b = torch.empty(t.numel() + 1, dtype=torch.uint8, device=dev)
        b[1:] = t.contiguous().view(torch.uint8).reshape(-1).to(dev)
        return b[1:].view(F8).view(t.shape)
    want, mag = mm_ref(x, xs, w[0], ws[0], False)
    for xd, wd in ((shifted(x), w[0].to(dev)), (x.to(dev), shifted(w[0]))):
        out = torch.empty(M * N + 1, dtype=torch.bfloat16, device=dev)[1:].view(M, N)
        pkg.block_quant_matmul(xd, xs.to(dev), wd, ws[0].to(dev), out=out)
        within(out, want, mm_tol(want, mag, K, torch.bfloat16))


def mm_ref_on(dev, x, xs, w, ws, nk):
    """mm_ref computed on the device, for sizes that take the CPU seconds."""
    want, mag = mm_ref(x.to(dev), xs.to(dev), w.to(dev), ws.to(dev), nk)
    return want.cpu(), mag.cpu()


# few wide tiles and a long K: the sums of a tile come from 2 or 4 pairs of CTAs (251 rows), or 2 to 8 CTAs (others)
@pytest.mark.parametrize("shape", [(250, 14320, 4080, True), (251, 8176, 2032, False), (251, 8176, 2040, True), (130, 14336, 4096, False), (60, 4096, 1000, True),
                                   (9, 7184, 264, True)])
def test_block_matmul_cut_along_k(pkg, dev, shape):
    M, K, N, nk = shape
    g = gen(M)
    x, xs = codes(g, M, K, F8)
    w, ws = weights(g, 1, K, N, nk)
    want, mag = mm_ref_on(dev, x, xs, w[0], ws[0], nk)
    for dtype in (torch.bfloat16, torch.float32):
        args = (x.to(dev), xs.to(dev), w[0].to(dev), ws[0].to(dev))
        out = pkg.block_quant_matmul(*args, transposed=nk, out_dtype=dtype)
        within(out, want, mm_tol(want, mag, K, dtype), f"{shape} {dtype}")
        assert torch.equal(out, pkg.block_quant_matmul(*args, transposed=nk, out_dtype=dtype))      # the parts meet in order


# more tiles than SMs, rows and columns ending inside them
@pytest.mark.parametrize("shape", [(2500, 528, 5000, True), (1100, 1040, 12304, False), (33, 272, 30000, True)])
def test_block_matmul_many_tiles(pkg, dev, shape):
    M, K, N, nk = shape
    g = gen(N)
    x, xs = codes(g, M, K, F8)
    w, ws = weights(g, 1, K, N, nk)
    want, mag = mm_ref_on(dev, x, xs, w[0], ws[0], nk)
    for dtype in (torch.float16, torch.float32):
        out = pkg.block_quant_matmul(x.to(dev), xs.to(dev), w[0].to(dev), ws[0].to(dev), transposed=nk, out_dtype=dtype)
        within(out, want, mm_tol(want, mag, K, dtype), f"{shape} {dtype}")


@pytest.mark.parametrize("nk", [False, True])
@pytest.mark.parametrize("M", [1, 75, 300])
def test_block_matmul_gradient_of_x(pkg, dev, M, nk):
    """The gradient of x is the product with the same weight and scales read the other way round, dense and per expert."""
    K, N, E = 528, 304, 3
    g = gen(M + 90)
    w, ws = weights(g, E, K, N, nk)
    dy, dys = codes(g, M, N, F8E5)
    dyv = dy.double() * dys.double().repeat_interleave(128, 1)[:, :N]
    wide = [w[e].double() * ws[e].double().repeat_interleave(128, 0).repeat_interleave(128, 1)[:w.shape[1], :w.shape[2]] for e in range(E)]
    x = torch.randn((M, K), generator=g, dtype=torch.float64).requires_grad_()
    rows = [M // 2, 0, M - M // 2]
    for counts in (None, rows):
        if counts is None:
            y = x @ (wide[0].t() if nk else wide[0])
            mag = dyv.abs() @ (wide[0] if nk else wide[0].t()).abs()
            got = pkg.block_quant_matmul(dy.to(dev), dys.to(dev), w[0].to(dev), ws[0].to(dev), transposed=not nk, out_dtype=torch.float32)
        else:
            parts = torch.split(x, counts)
            y = torch.cat([v @ (wide[e].t() if nk else wide[e]) for e, v in enumerate(parts)])
            mag = torch.cat([v.abs() @ (wide[e] if nk else wide[e].t()).abs() for e, v in enumerate(torch.split(dyv, counts))])
            got = pkg.block_quant_grouped_matmul(dy.to(dev), dys.to(dev), w.to(dev), ws.to(dev), torch.tensor(counts, device=dev), transposed=not nk,
                                                 out_dtype=torch.float32)
        want, = torch.autograd.grad((y * dyv).sum(), x)
        within(got, want, mm_tol(want, mag, N, torch.float32), f"{counts}")


GROUPS = {
    "even": [40, 40, 40, 40], "ragged": [1, 0, 129, 77, 0, 3, 256, 128, 5], "one": [0, 0, 300, 0], "none": [0, 0, 0], "behind": [10, 20, 0],
    "many": [i % 5 for i in range(67)], "single": [1] * 40, "large": [700, 3, 513], "most": [3 if i % 7 == 0 else 0 for i in range(1024)],
    "middle": [90, 0, 200, 17, 64, 33, 255, 1],
}


@pytest.mark.parametrize("nk", [False, True])
@pytest.mark.parametrize("which", sorted(GROUPS))
@pytest.mark.parametrize("kn", [(272, 400), (1024, 256), (100, 60)])
def test_grouped_matmul(pkg, dev, which, kn, nk):
    counts, (K, N) = GROUPS[which], kn
    E, rows = len(counts), sum(counts)
    M = rows + (37 if which in ("behind", "none", "ragged") else 0)
    g = gen(E + K)
    x, xs = codes(g, M, K, F8)
    w, ws = weights(g, E, K, N, nk)
    out = torch.full((M, N), 7.0, dtype=torch.bfloat16, device=dev)
    pkg.block_quant_grouped_matmul(x.to(dev), xs.to(dev), w.to(dev), ws.to(dev), torch.tensor(counts, device=dev), transposed=nk, out=out)
    assert (out[rows:] == 7.0).all()                       # rows behind the last expert's are left as they were
    at = 0
    for e, c in enumerate(counts):
        if c:
            want, mag = mm_ref(x[at:at + c], xs[at:at + c], w[e], ws[e], nk)
            within(out[at:at + c], want, mm_tol(want, mag, K, torch.bfloat16), f"expert {e}")
        at += c


def test_grouped_matmul_counts_that_do_not_add_up(pkg, dev):
    """Negative counts count as 0, and rows end at M whatever the counts say."""
    K, N, M, E = 256, 144, 50, 4
    g = gen(3)
    x, xs = codes(g, M, K, F8)
    w, ws = weights(g, E, K, N, True)
    out = torch.full((M, N), 7.0, device=dev)
    counts = torch.tensor([20, -5, 1 << 40, 9], device=dev)
    pkg.block_quant_grouped_matmul(x.to(dev), xs.to(dev), w.to(dev), ws.to(dev), counts, transposed=True, out=out)
    for lo, hi, e in ((0, 20, 0), (20, 50, 2)):
        want, mag = mm_ref(x[lo:hi], xs[lo:hi], w[e], ws[e], True)
        within(out[lo:hi], want, mm_tol(want, mag, K, torch.float32))


# ------------------------------------------------------------------------------------------------ permutation
def route_ref(ids, E):
    flat = ids.reshape(-1).long()
    key = torch.where((flat < 0) | (flat >= E), torch.full_like(flat, E), flat)
    order = torch.sort(key, stable=True).indices
    place = torch.empty_like(order)
    place[order] = torch.arange(order.numel())
    place[key == E] = -1
    return place.view(ids.shape).int(), torch.bincount(key, minlength=E + 1)[:E]


def routing(g, T, k, E, away=0.0):
    ids = torch.stack([torch.randperm(max(E, k), generator=g)[:k] % E for _ in range(T)]) if T else torch.zeros((0, k), dtype=torch.int64)
    ids[torch.rand(ids.shape, generator=g) < away] = -1
    return ids


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, F8, torch.int8])
@pytest.mark.parametrize("case", [(1, 1, 1, 16), (1, 8, 64, 4096), (5, 2, 3, 33), (64, 8, 256, 130), (300, 4, 1024, 1024), (1000, 6, 60, 72), (0, 2, 4, 64), (7, 64, 100, 48),
                                  (257, 33, 40, 4100), (3000, 8, 7, 16), (9001, 8, 60, 16), (1100, 3, 1023, 24), (70000, 1, 130, 4)])
def test_permute(pkg, dev, case, dtype):
    T, k, E, H = case
    g = gen(T + k)
    for away, idt in ((0.0, torch.int32), (0.3, torch.int64)):
        ids = routing(g, T, k, E, away)
        if away and T > 1:
            ids[1, 0] = E            # just outside, and far outside
            ids[0, -1] = (1 << 40) if idt == torch.int64 else -7
        x = torch.randint(-100, 100, (T, H), generator=g).to(torch.int8) if dtype in (torch.int8, F8) else torch.randn((T, H), generator=g).to(dtype)
        x = x.view(F8) if dtype == F8 else x
        S = -(-H // 128)
        sc = torch.randn((T, S), generator=g)
        raw = lambda t: t.contiguous().view(torch.uint8)
        out = torch.full((T * k + 3, H), 1.0, device=dev).to(x.dtype)
        sout = torch.full((T * k + 3, S), 9.0, device=dev)
        rows, place, counts, srows = pkg.moe_token_permute(x.to(dev), ids.to(idt).to(dev), E, scales=sc.to(dev), out=out, scales_out=sout)
        want_place, want_counts = route_ref(ids, E)
        assert torch.equal(place.cpu(), want_place) and torch.equal(counts.cpu(), want_counts)
        want, wants = torch.full((T * k + 3, H), 1.0).to(x.dtype), torch.full((T * k + 3, S), 9.0)
        there = want_place.reshape(-1) >= 0
        src = torch.arange(T).repeat_interleave(k)[there]
        raw(want).view(T * k + 3, -1)[want_place.reshape(-1)[there].long()] = raw(x).view(T, -1)[src] if T else raw(x).view(0, raw(want).view(T * k + 3, -1).shape[1])
        wants[want_place.reshape(-1)[there].long()] = sc[src]
        assert torch.equal(raw(rows.cpu()), raw(want)) and torch.equal(srows.cpu(), wants)


def test_permute_same_expert_twice_and_all_away(pkg, dev):
    ids = torch.tensor([[2, 2], [0, 2], [2, 0]], dtype=torch.int32)
    x = torch.arange(3.0).view(3, 1).repeat(1, 8)
    rows, place, counts = pkg.moe_token_permute(x.to(dev), ids.to(dev), 4)
    assert place.tolist() == [[2, 3], [0, 4], [5, 1]] and counts.tolist() == [2, 0, 4, 0]
    assert rows[:, 0].tolist() == [1, 2, 0, 0, 1, 2]
    out = torch.full((6, 8), 5.0, device=dev)
    rows, place, counts = pkg.moe_token_permute(x.to(dev), torch.full((3, 2), -1, dtype=torch.int32, device=dev), 4, out=out)
    assert (place == -1).all() and (counts == 0).all() and (rows == 5.0).all()
    assert (pkg.moe_token_unpermute(rows, place, torch.ones(3, 2, device=dev)) == 0).all()


def gather_ref(rows, place, probs):
    R = rows.shape[0]
    ok = (place >= 0) & (place < R)
    v = rows.double()[place.long().clamp(0, max(R - 1, 0))] * ok[..., None] if R else torch.zeros(place.shape + (rows.shape[1],), dtype=torch.float64)
    p = (probs.double() if probs is not None else torch.ones(place.shape, dtype=torch.float64))[..., None]
    return (p * v).sum(1), (p * v).abs().sum(1)


CASES = [(1, 1, 1, 8), (1, 8, 64, 4096), (5, 2, 3, 33), (64, 8, 256, 130), (130, 4, 16, 1024), (9, 40, 50, 264), (31, 6, 60, 2056), (2, 3, 4, 1)]


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("case", CASES)
def test_unpermute_and_permute_gradient(pkg, dev, case, dtype):
    T, k, E, H = case
    g = gen(T * 3 + k)
    place, _ = route_ref(routing(g, T, k, E, 0.2), E)
    rows = torch.randn((T * k, H), generator=g).to(dtype)
    gone = torch.ones(T * k, dtype=torch.bool)
    gone[place[place >= 0].long()] = False
    rows[gone] = float("nan")                               # rows without a pair are never read
    for pt in (torch.float32, dtype):
        probs = torch.rand((T, k), generator=g).to(pt)
        want, mag = gather_ref(torch.nan_to_num(rows), place, probs)
        out = pkg.moe_token_unpermute(rows.to(dev), place.to(dev), probs.to(dev))
        within(out, want, rounding(want, dtype) + (k + 1) * 2.0 ** -23 * mag)
    want, mag = gather_ref(torch.nan_to_num(rows), place, None)
    for out in (pkg.moe_token_permute_grad(rows.to(dev), place.to(dev)), pkg.moe_token_unpermute(rows.to(dev), place.to(dev))):
        within(out, want, rounding(want, dtype) + (k + 1) * 2.0 ** -23 * mag)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("case", CASES)
def test_unpermute_gradient(pkg, dev, case, dtype):
    T, k, E, H = case
    g = gen(T * 5 + k)
    place, _ = route_ref(routing(g, T, k, E, 0.2), E)
    rows, dout = torch.randn((T * k, H), generator=g).to(dtype), torch.randn((T, H), generator=g).to(dtype)
    for pt in (torch.float32, dtype):
        probs = torch.rand((T, k), generator=g).to(pt)
        buf = torch.full((T * k, H), 3.0, dtype=dtype, device=dev)
        drows, dprobs = pkg.moe_token_unpermute_grad(dout.to(dev), rows.to(dev), place.to(dev), probs.to(dev), out=buf)
        ok = place >= 0
        v = rows.double()[place.long().clamp_min(0)] * ok[..., None]
        want_p = (dout.double()[:, None] * v).sum(-1)
        mag_p = (dout.double()[:, None] * v).abs().sum(-1)
        within(dprobs, want_p, rounding(want_p, pt) + (H + 8) * 2.0 ** -23 * mag_p, "probs")
        want = torch.full((T * k, H), 3.0, dtype=torch.float64)
        want[place[ok].long()] = (probs.double()[..., None] * dout.double()[:, None])[ok]
        tol = rounding(want, dtype) + want.abs() * 2.0 ** -23
        named = torch.zeros(T * k, dtype=torch.bool)
        named[place[ok].long()] = True
        tol[~named] = 0.0                                    # rows that no pair names are left as they were
        within(drows, want, tol, "rows")


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("H", [40, 33, 2048])
def test_places_that_name_no_row(pkg, dev, dtype, H):
    """Places below 0 and behind the last row stand for no row: their weights (NaN here) take no part, their gradients are 0."""
    T, k, R = 5, 3, 9
    g = gen(H)
    place = torch.tensor([[0, -1, 8], [9, 1, -(1 << 31)], [(1 << 31) - 1, 9, -1], [2, 3, 4], [5, 100, 6]], dtype=torch.int32)
    ok = (place >= 0) & (place < R)
    rows, dout, probs = torch.randn((R, H), generator=g).to(dtype), torch.randn((T, H), generator=g).to(dtype), torch.rand((T, k), generator=g)
    nan_probs = torch.where(ok, probs, torch.full_like(probs, float("nan")))
    want, mag = gather_ref(rows, torch.where(ok, place, torch.full_like(place, -1)), probs * ok)
    out = pkg.moe_token_unpermute(rows.to(dev), place.to(dev), nan_probs.to(dev))
    within(out, want, rounding(want, dtype) + (k + 1) * 2.0 ** -23 * mag)
    assert (out[2] == 0).all()
    buf = torch.full((R, H), 3.0, dtype=dtype, device=dev)
    drows, dprobs = pkg.moe_token_unpermute_grad(dout.to(dev), rows.to(dev), place.to(dev), nan_probs.to(dev), out=buf)
    assert (dprobs.cpu()[~ok] == 0).all() and (drows[7] == 3.0).all() and torch.isfinite(drows).all()
    v = rows.double()[place.long().clamp(0, R - 1)] * ok[..., None]
    within(dprobs, (dout.double()[:, None] * v).sum(-1), rounding((dout.double()[:, None] * v).sum(-1), torch.float32) + (H + 8) * 2.0 ** -23 *
           (dout.double()[:, None] * v).abs().sum(-1))


def test_swiglu_far_from_zero(pkg, dev):
    """Gates whose exponential leaves fp32's range: the value, not 0 or NaN."""
    a = torch.tensor([-200.0, -100.0, -88.5, -87.4, -50.0, 50.0, 88.5, 100.0, 200.0, 0.0, -0.0])
    x = torch.zeros((len(a), 256))
    x[:, 0], x[:, 128] = a, 1e30
    q, s = pkg.swiglu_block_quant_fp8(x.to(dev))
    g = a.double() * torch.sigmoid(a.double()) * 1e30
    got = q[:, 0].double().cpu() * s[:, 0].double().cpu()
    # the value is the block's maximum, so its code is exact: what is left is the sigmoid's and the scale's rounding
    # (below 2^-126 the exponential is a subnormal number, off by 2^-149)
    tol = g.abs() * ((2 * a.double().abs() * 1.4427 + 14) * 2.0 ** -23 + 2.0 ** -24) + a.double().abs() * 2.0 ** -149 * 1e30
    within(got, g, tol)


def test_gradients_against_differences(pkg, dev):
    """Both sums are linear in their rows and weights, so a difference quotient is exact up to rounding."""
    T, k, E, H = 40, 4, 12, 200
    g = gen(8)
    ids = routing(g, T, k, E, 0.1)
    x = torch.randn((T, H), generator=g).to(dev)
    rows, place, _ = pkg.moe_token_permute(x, ids.int().to(dev), E, out=torch.zeros((T * k, H), device=dev))
    y, probs = torch.randn((T * k, H), generator=g).to(dev), torch.rand((T, k), generator=g).to(dev)
    dout = torch.randn((T, H), generator=g).to(dev)
    loss = lambda y, p: (dout.double() * pkg.moe_token_unpermute(y, place, p).double()).sum()
    drows, dprobs = pkg.moe_token_unpermute_grad(dout, y, place, probs)
    dy, dp = torch.randn((T * k, H), generator=g).to(dev), torch.randn((T, k), generator=g).to(dev)
    # each loss is a sum of T*H values off by (k + 3) * 2^-24 of their terms (<= 4 * 4 * 8 in magnitude); a step of 1/2
    tol = 2 * 2 * T * H * (k + 3) * 2.0 ** -24 * 128
    within((loss(y + 0.5 * dy, probs) - loss(y - 0.5 * dy, probs)), (drows.double() * dy.double()).sum(), tol)
    within((loss(y, probs + 0.5 * dp) - loss(y, probs - 0.5 * dp)), (dprobs.double() * dp.double()).sum(), tol)
    # the permutation: <grad_rows, permute(x)> differentiated along dx
    grows = torch.randn((T * k, H), generator=g).to(dev)
    dx = torch.randn((T, H), generator=g).to(dev)
    zero = lambda: torch.zeros((T * k, H), device=dev)
    perm = lambda v: (grows.double() * pkg.moe_token_permute(v, ids.int().to(dev), E, out=zero())[0].double()).sum()
    grad = pkg.moe_token_permute_grad(grows, place)
    within(perm(x + 0.5 * dx) - perm(x - 0.5 * dx), (grad.double() * dx.double()).sum(), tol)


# ------------------------------------------------------------------------------------------------ together
class Layer:
    """One expert layer through the package's calls; every intermediate is kept."""

    def __init__(self, pkg, dev, T, k, E, H, F, seed, away=0.0):
        g = gen(seed)
        self.pkg, self.dims = pkg, (T, k, E, H, F)
        self.x = torch.randn((T, H), generator=g).to(torch.bfloat16).to(dev)
        self.ids = routing(g, T, k, E, away).int().to(dev)
        self.probs = torch.softmax(torch.randn((T, k), generator=g), -1).to(dev)
        w1, s1 = weights(g, E, H, 2 * F, True)
        w2, s2 = weights(g, E, F, H, True)
        self.w1, self.s1, self.w2, self.s2 = w1.to(dev), s1.to(dev), w2.to(dev), s2.to(dev)
        self.rows_out = torch.zeros((T * k, H), dtype=torch.uint8, device=dev).view(F8)
        self.scales_out = torch.ones((T * k, -(-H // 128)), device=dev)
        self.h_out = torch.zeros((T * k, 2 * F), dtype=torch.bfloat16, device=dev)
        self.y_out = torch.zeros((T * k, H), dtype=torch.bfloat16, device=dev)

    def run(self):
        p, E = self.pkg, self.dims[2]
        self.q, self.s = p.block_quant_fp8(self.x)
        self.rows, self.place, self.counts, self.rs = p.moe_token_permute(self.q, self.ids, E, scales=self.s, out=self.rows_out, scales_out=self.scales_out)
        self.h = p.block_quant_grouped_matmul(self.rows, self.rs, self.w1, self.s1, self.counts, transposed=True, out=self.h_out)
        self.q2, self.s2q = p.swiglu_block_quant_fp8(self.h)
        self.y = p.block_quant_grouped_matmul(self.q2, self.s2q, self.w2, self.s2, self.counts, transposed=True, out=self.y_out)
        self.out = p.moe_token_unpermute(self.y, self.place, self.probs)
        return self.out


@pytest.mark.parametrize("dims", [(1, 2, 4, 256, 384), (50, 4, 16, 400, 272), (300, 2, 4, 512, 640)])
def test_expert_layer(pkg, dev, dims):
    """A whole layer: each stage against its formula on the stage before, and the result against the layer in 64 bits
    on the quantised values."""
    T, k, E, H, F = dims
    L = Layer(pkg, dev, *dims, seed=sum(dims), away=0.15)
    L.run()
    rq, rs = quant_ref(L.x.cpu(), F8)
    assert torch.equal(L.q.view(torch.uint8).cpu(), rq) and torch.equal(L.s.cpu(), rs)
    place, counts = route_ref(L.ids.cpu(), E)
    assert torch.equal(L.place.cpu(), place) and torch.equal(L.counts.cpu(), counts)
    want_out = torch.zeros((T, H), dtype=torch.float64)
    tol_out = torch.zeros((T, H), dtype=torch.float64)
    e_of = torch.repeat_interleave(torch.arange(E), counts)
    for t in range(T):
        for j in range(k):
            r = int(place[t, j])
            if r < 0:
                continue
            e = int(e_of[r])
            q, s = L.q[t:t + 1].cpu(), L.s[t:t + 1].cpu()
            h, mag = mm_ref(q, s, L.w1[e].cpu(), L.s1[e].cpu(), True)
            within(L.h[r:r + 1], h, mm_tol(h, mag, H, torch.bfloat16), "gate and up")
            y, mag = mm_ref(L.q2[r:r + 1].cpu(), L.s2q[r:r + 1].cpu(), L.w2[e].cpu(), L.s2[e].cpu(), True)
            within(L.y[r:r + 1], y, mm_tol(y, mag, F, torch.bfloat16), "down")
            p = float(L.probs[t, j])
            want_out[t] += p * y[0]
            tol_out[t] += p * (mm_tol(y, mag, F, torch.bfloat16)[0] + (k + 1) * 2.0 ** -23 * y[0].abs())
    within(L.out, want_out, tol_out + (want_out.abs() + tol_out) * 2.0 ** -8, "layer")


def test_expert_layer_captured_and_replayed(pkg, dev):
    """The layer in a CUDA graph gives the direct call's bits, also after its inputs changed; two graphs of two layers
    replayed in turns keep apart."""
    a, b = Layer(pkg, dev, 33, 4, 8, 256, 256, seed=1, away=0.1), Layer(pkg, dev, 200, 2, 4, 384, 256, seed=2)
    want = {}
    for L in (a, b):
        want[L] = L.run().clone()
    torch.cuda.synchronize()
    graphs = {}
    for L in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            L.run()
        graphs[L] = g
    for _ in range(3):
        for L in (a, b):
            graphs[L].replay()
    torch.cuda.synchronize()
    for L in (a, b):
        assert torch.equal(L.out, want[L])
    a.x.mul_(-0.5)
    a.ids.copy_((a.ids + 1) % 8)
    graphs[a].replay()
    torch.cuda.synchronize()
    got = a.out.clone()
    assert torch.equal(got, a.run())


def test_large_permutes_captured_and_on_two_streams(pkg, dev):
    """Permutes of many pairs (a sort and a copy): two captured graphs replayed in turns, and two streams at once, keep apart."""
    cases = []
    for i, (T, k, E, H) in enumerate(((700, 4, 30, 64), (3000, 2, 256, 40))):
        g = gen(40 + i)
        ids = routing(g, T, k, E, 0.1)
        x = torch.randn((T, H), generator=g).to(torch.bfloat16)
        cases.append((x.to(dev), ids.int().to(dev), E, torch.zeros((T * k, H), dtype=torch.bfloat16, device=dev)) + route_ref(ids, E))
    run = lambda c: pkg.moe_token_permute(c[0], c[1], c[2], out=c[3])
    check = lambda c, got: torch.equal(got[1].cpu(), c[4]) and torch.equal(got[2].cpu(), c[5]) and all(
        torch.equal(got[0][c[4][t, j]].cpu(), c[0][t].cpu()) for t, j in ((0, 0), (5, 1), (-1, -1)) if c[4][t, j] >= 0)
    for c in cases:
        assert check(c, run(c))
    torch.cuda.synchronize()
    graphs = []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = run(c)
        graphs.append((g, got))
    for _ in range(3):
        for c in cases:
            c[3].zero_()
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(check(c, got) for c, (_, got) in zip(cases, graphs))
    streams = [torch.cuda.Stream(dev) for _ in cases]
    for _ in range(4):
        outs = []
        for c, s in zip(cases, streams):
            s.wait_stream(torch.cuda.current_stream(dev))
            with torch.cuda.stream(s):
                outs.append(run(c))
        torch.cuda.synchronize()
        assert all(check(c, got) for c, got in zip(cases, outs))


@pytest.mark.parametrize("dims", [(3, 2, 4, 256, 384), (40, 8, 16, 1024, 512), (700, 4, 8, 512, 512)])
def test_layers_back_to_back(pkg, dev, dims):
    """Kernels start while the one before them drains: layers one behind the other, whose buffers change hands between them,
    give the bits of layers run one at a time."""
    L = Layer(pkg, dev, *dims, seed=21, away=0.1)
    g = gen(22)
    xs = [torch.randn(tuple(L.x.shape), generator=g).to(device=dev, dtype=L.x.dtype) for _ in range(12)]
    dout = [torch.randn(tuple(L.x.shape), generator=g).to(device=dev, dtype=L.x.dtype) for _ in range(12)]

    def one(x, d):
        L.x = x
        out = L.run()
        dy, dp = pkg.moe_token_unpermute_grad(d, L.y, L.place, L.probs)
        return out, dp, pkg.moe_token_permute_grad(dy, L.place)

    want = []
    for x, d in zip(xs, dout):
        torch.cuda.synchronize()
        want.append([t.clone() for t in one(x, d)])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()                          # without the host's time between the kernels
    with torch.cuda.graph(graph):
        got = [one(x, d) for x, d in zip(xs, dout)]
    for _ in range(20):
        for outs in got:
            for t in outs:
                t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_two_streams_at_once(pkg, dev):
    """Two layers on two streams at the same time: nothing is shared between calls."""
    layers = [Layer(pkg, dev, 64, 4, 8, 512, 384, seed=5 + i) for i in range(2)]
    want = [L.run().clone() for L in layers]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(dev) for _ in layers]
    for _ in range(5):
        outs = []
        for L, s in zip(layers, streams):
            s.wait_stream(torch.cuda.current_stream(dev))
            with torch.cuda.stream(s):
                outs.append(L.run())
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w)


def test_results_repeat_bit_for_bit(pkg, dev):
    L = Layer(pkg, dev, 100, 8, 32, 640, 512, seed=9)
    first = [t.clone() for t in (L.run(), L.h, L.y, L.place)]
    for _ in range(4):
        for t, w in zip((L.run(), L.h, L.y, L.place), first):
            assert torch.equal(t, w)
    dout = torch.randn((100, 640), device=dev).to(torch.bfloat16)
    g0 = pkg.moe_token_unpermute_grad(dout, L.y, L.place, L.probs)
    for _ in range(3):
        assert all(torch.equal(u, v) for u, v in zip(g0, pkg.moe_token_unpermute_grad(dout, L.y, L.place, L.probs)))


def test_offsets_beyond_32_bits(pkg, dev):
    """More than 2^32 bytes, and more than 2^31 elements, behind every tensor that can be so long: the last rows are right."""
    def random_codes(*shape):
        q = torch.empty(shape, dtype=torch.uint8, device=dev)
        q.random_(0, 120)                                   # no NaN codes
        return q.view(F8)

    D, rows = 4096, (1 << 19) + 1029                        # quantiser, on 2^31 and more elements
    x = torch.zeros((rows, D), dtype=torch.bfloat16, device=dev)
    last = activations(gen(31), (3, D), torch.bfloat16)
    x[-3:] = last.to(dev)
    q, s = pkg.block_quant_fp8(x)
    rq, rs = quant_ref(last, F8)
    assert torch.equal(s[-3:].cpu(), rs) and torch.equal(q[-3:].view(torch.uint8).cpu(), rq)
    # the same rows sorted, all but the last behind one expert, and summed again
    ids = torch.zeros((rows, 1), dtype=torch.int32, device=dev)
    ids[-2] = 1
    r, place, counts = pkg.moe_token_permute(x, ids, 3)
    assert counts.tolist() == [rows - 1, 1, 0] and place[-3:, 0].tolist() == [rows - 3, rows - 1, rows - 2]
    assert torch.equal(r[-3:], x[[-3, -1, -2]])
    assert torch.equal(pkg.moe_token_unpermute(r, place)[-3:], x[-3:])
    assert torch.equal(pkg.moe_token_permute_grad(r, place)[-3:], x[-3:])
    probs = torch.full((rows, 1), 0.5, device=dev)
    dr, dp = pkg.moe_token_unpermute_grad(x, r, place, probs, out=torch.empty_like(x))
    assert torch.equal(dr[-3:], 0.5 * x[[-3, -1, -2]])
    sq = (last.double() ** 2).sum(1, keepdim=True)
    within(dp[-3:], sq, sq * D * 2.0 ** -23)
    del x, q, s, r, dr, ids, place
    M, N, K = 70003, 32768, 144                             # product: the output, for many and for few rows
    xq, wq = random_codes(M, K), random_codes(N, K)
    xs, ws = torch.rand((M, 2), device=dev), torch.rand((N // 128, 2), device=dev)
    out = pkg.block_quant_matmul(xq, xs, wq, ws, transposed=True)
    want, mag = mm_ref(xq[-2:].cpu(), xs[-2:].cpu(), wq.cpu(), ws.cpu(), True)
    within(out[-2:], want, mm_tol(want, mag, K, torch.bfloat16))
    del out, wq
    E, K, N = 1024, 2048, 2064                              # and the experts' weights
    for nk in (True, False):
        w = random_codes(E, N, K) if nk else random_codes(E, K, N)
        ws = torch.rand((E, 17, 16) if nk else (E, 16, 17), device=dev)
        for M in (9, 400):
            xq, xs = random_codes(M, K), torch.rand((M, 16), device=dev)
            counts = torch.zeros(E, dtype=torch.int64, device=dev)
            counts[-1], counts[3] = M - 2, 2
            out = pkg.block_quant_grouped_matmul(xq, xs, w, ws, counts, transposed=nk)
            for lo, hi, e in ((0, 2, 3), (2, M, E - 1)):
                want, mag = mm_ref(xq[lo:hi].cpu(), xs[lo:hi].cpu(), w[e].cpu(), ws[e].cpu(), nk)
                within(out[lo:hi], want, mm_tol(want, mag, K, torch.bfloat16), f"{nk} {M} {e}")
        del w


def test_two_phase_entries(pkg, dev):
    """Every operator through its own two phases gives the bits of the one-call form behind the wrappers."""
    L = Layer(pkg, dev, 20, 2, 4, 256, 384, seed=13)
    L.run()
    A, i64, cbool = pkg.AclTensor, ctypes.c_int64, ctypes.c_bool
    new = lambda t: torch.zeros_like(t, dtype=torch.uint8).view(t.dtype) if t.element_size() == 1 else torch.zeros_like(t)
    same = lambda a, b: torch.equal(a.view(torch.uint8), b.view(torch.uint8))

    def check(name, ins, outs, *rest):
        got = [new(t) for t in outs]
        pkg.call(name, *ins, *[A(t) for t in got], *rest)
        assert all(same(a, b) for a, b in zip(got, outs)), name

    q, s = new(L.q), new(L.s)
    pkg.call("aclnnB200BlockQuantFp8", A(L.x), i64(1), A(q), A(s))
    assert same(q, L.q) and same(s, L.s)
    check("aclnnB200SwiGluBlockQuantFp8", [A(L.h)], [L.q2, L.s2q])
    ids = A(L.ids)
    rows, rs, place, counts = new(L.rows), new(L.rs), new(L.place), new(L.counts)
    pkg.call("aclnnB200MoeTokenPermute", A(L.q), ids, A(L.s), A(rows), A(rs), A(place), A(counts))
    assert same(rows, L.rows) and same(rs, L.rs) and same(place, L.place) and same(counts, L.counts)
    check("aclnnB200BlockQuantGroupedMatmul", [A(L.rows), A(L.rs), A(L.w1), A(L.s1), A(L.counts), cbool(True)], [L.h])
    one = pkg.block_quant_matmul(L.q, L.s, L.w1[0], L.s1[0], transposed=True)
    check("aclnnB200BlockQuantMatmul", [A(L.q), A(L.s), A(L.w1[0]), A(L.s1[0]), cbool(True)], [one])
    check("aclnnB200MoeTokenUnpermute", [A(L.y), A(L.place), A(L.probs)], [L.out])
    check("aclnnB200MoeTokenPermuteGrad", [A(L.y), A(L.place)], [pkg.moe_token_permute_grad(L.y, L.place)])
    dy, dp = pkg.moe_token_unpermute_grad(L.x, L.y, L.place, L.probs)
    check("aclnnB200MoeTokenUnpermuteGrad", [A(L.x), A(L.y), A(L.place), A(L.probs)], [dy, dp])


def test_refusals_on_the_device(pkg, dev):
    x = torch.zeros((4, 256), dtype=torch.bfloat16, device=dev)
    with pytest.raises(ValueError):
        pkg.block_quant_fp8(x.t())
    with pytest.raises(RuntimeError):
        pkg.block_quant_fp8(x, row_block=64)
    with pytest.raises(RuntimeError):
        pkg.moe_token_permute(x, torch.zeros((4, 2), dtype=torch.int32, device=dev), 2000)
    with pytest.raises(RuntimeError):
        pkg.moe_token_unpermute(x, torch.zeros((4, 2), dtype=torch.int64, device=dev))
    rows = torch.zeros((8, 256), dtype=torch.bfloat16, device=dev)
    with pytest.raises(RuntimeError):                        # gradient over its own input
        pkg.moe_token_unpermute_grad(x, rows, torch.zeros((4, 2), dtype=torch.int32, device=dev), torch.zeros((4, 2), device=dev), out=rows)
    torch.cuda.synchronize()


def test_no_wait_gave_up(pkg, dev):
    torch.cuda.synchronize()
    lib = pkg.load()
    lib.aclnnB200DeviceStatus.restype = ctypes.c_uint32
    assert lib.aclnnB200DeviceStatus() == 0
