"""The 8-bit linear layer (b200_quantize_i8, b200_rms_norm_i8, b200_gemm_i8) through its binding: refusals on the
CPU, results on the GPU against the formulas in 64 bits.

Integer results are held to equality.  q = round_half_even(127 t / m) is compared with the quotient in 64 bits:
t and m are f32 values, so a quotient is a border between two integers exactly or differs from it by more than
2^-33 (254 t and (2k + 1) m are integers of at most 32 bits times a power of two), far above 2^-53.
f32 results: each rounding is off by at most 2^-24 relative."""
import math

import pytest

F16, F32, BF16, S32 = 10, 11, 13, 4
U32 = 2.0 ** -24


@pytest.fixture(scope="module")
def k(lib_path):
    from pjrt_b200 import kernels
    return kernels.Kernels(lib_path)


# ------------------------------------------------------------------------------------------ refusals (no GPU)
P = 1 << 20          # an address that no call below comes to use


def refused(call, code=-1):
    from pjrt_b200.kernels import KernelError
    with pytest.raises(KernelError) as e:
        call()
    assert e.value.code == code


@pytest.mark.parametrize("change", [dict(dtype=S32), dict(rows=-1), dict(cols=-1), dict(ldx=15), dict(ldq=15), dict(x=None),
                                    dict(q=None), dict(scale=None), dict(x=P + 1), dict(scale=P + 2), dict(rows=1 << 31),
                                    dict(cols=1 << 31, ldx=1 << 31, ldq=1 << 31)])
def test_quantize_refusals(k, change):
    a = dict(x=P, ldx=16, q=P, ldq=16, scale=P, rows=4, cols=16, dtype=BF16)
    refused(lambda: k.quantize_i8(**{**a, **change}))


@pytest.mark.parametrize("change", [dict(dtype=S32), dict(weight_dtype=S32), dict(rows=-1), dict(cols=0), dict(ldx=15), dict(ldr=15),
                                    dict(ldh=15), dict(ldq=15), dict(x=None), dict(weight=None), dict(q=None), dict(scale=None),
                                    dict(residual=None), dict(eps=0.0), dict(eps=-1.0), dict(eps=math.nan), dict(eps=math.inf),
                                    dict(residual=P + 1), dict(h=P + 1), dict(weight=P + 2), dict(ldh=24),
                                    dict(h=2 * P, residual=2 * P, ldr=24)])
def test_rms_norm_refusals(k, change):
    a = dict(x=P, ldx=16, residual=P, ldr=16, weight=P, h=P, ldh=16, q=P, ldq=16, scale=P, rows=4, cols=16, dtype=BF16,
             weight_dtype=F32, eps=1e-5)
    refused(lambda: k.rms_norm_i8(**{**a, **change}))


@pytest.mark.parametrize("change", [dict(out_type=2), dict(m=-1), dict(n=-1), dict(k=-1), dict(lda=31), dict(ldb=31), dict(ldc=15),
                                    dict(k=131072, lda=131072, ldb=131072), dict(a=None), dict(b=None), dict(c=None), dict(c=P + 1),
                                    dict(a_scale=P + 2), dict(b_scale=P + 2), dict(bias=P + 2), dict(act=2), dict(act=-1),
                                    dict(out_type=S32), dict(out_type=S32, a_scale=None, b_scale=None, bias=None, act=1)])
def test_gemm_refusals(k, change):
    a = dict(a=P, lda=32, b=P, ldb=32, a_scale=P, b_scale=P, bias=P, c=P, ldc=16, m=8, n=16, k=32, out_type=BF16)
    refused(lambda: k.gemm_i8(**{**a, **change}))


@pytest.mark.parametrize("change,need", [({}, 0), (dict(a=P + 1), 100 * 48), (dict(lda=33), 100 * 48), (dict(b=P + 8), 1000 * 48),
                                         (dict(lda=33, ldb=34), 1100 * 48), (dict(lda=33, ldb=34, m=2), 0)])
def test_gemm_scratch(k, change, need):
    """Operands that do not lie 16-byte aligned need room for copies, each rounded up to 256 bytes; one or two tokens
    are multiplied where they lie."""
    a = {**dict(a=P, lda=48, b=P, ldb=48, m=100, n=1000, k=33), **change}
    moved = [(a["m"], a["a"] % 16 or a["lda"] % 16), (a["n"], a["b"] % 16 or a["ldb"] % 16)] if a["m"] > 2 else []
    room = sum((r * 48 + 255) // 256 * 256 for r, copy in moved if copy)
    assert k.gemm_i8_scratch_bytes(**a) == room >= need
    if room:
        call = dict(a_scale=None, b_scale=None, bias=None, c=P, ldc=1000, out_type=BF16)
        refused(lambda: k.gemm_i8(**a, **call), -4)
        refused(lambda: k.gemm_i8(**a, **call, scratch=P, scratch_bytes=room - 1), -4)
        refused(lambda: k.gemm_i8(**a, **call, scratch=P + 16, scratch_bytes=room + 256), -4)


def test_empty_calls_do_nothing(k):
    k.quantize_i8(None, 16, None, 16, None, 0, 16, BF16)
    k.rms_norm_i8(None, 16, None, 0, None, None, 0, None, 16, None, 0, 16, BF16, F32, 1e-5)
    k.gemm_i8(None, 32, P, 32, None, None, None, None, 16, 0, 16, 32, BF16)
    k.gemm_i8(P, 32, None, 32, None, None, None, None, 0, 8, 0, 32, BF16)


# ------------------------------------------------------------------------------------------ helpers
def types(torch):
    return {F32: torch.float32, BF16: torch.bfloat16, F16: torch.float16}


def stream(torch):
    return torch.cuda.current_stream().cuda_stream


def rows_of(torch, rows, cols, pad, dtype, fill=None, offset=0):
    """[rows, cols] inside a larger array: `pad` elements between rows, `offset` before the first."""
    n = rows * (cols + pad) + offset + 64
    flat = torch.empty(n, device="cuda", dtype=dtype)
    if fill is not None:
        flat.fill_(fill)
    return flat[offset:offset + rows * (cols + pad)].view(rows, cols + pad)[:, :cols], flat


def activations(torch, g, rows, cols, pad, dtype, offset=0):
    v, _ = rows_of(torch, rows, cols, pad, dtype, offset=offset)
    x = torch.randn(rows, cols, device="cuda", generator=g)
    if cols > 8:
        x[:, cols // 3] *= 30.0
    v.copy_(x)
    return v


def rounded(torch, t):
    """(q, m) of t [rows, cols] f32, the quotient in 64 bits."""
    m = t.abs().amax(1) if t.shape[1] else torch.zeros(t.shape[0], device=t.device)
    ok = torch.isfinite(t).all(1)
    d = torch.where(ok & (m > 0), m, 1.0).double()
    q = torch.where(ok[:, None], t, 0.0).double() * 127.0 / d[:, None]
    return torch.where((ok & (m > 0))[:, None], q.round(), 0.0).to(torch.int8), torch.where(ok, m, math.nan)


def close_f32(torch, got, ref, steps):
    """Within `steps` f32 half steps, relative; below the normal range, of the smallest normal value."""
    got, ref = got.double(), ref.double()
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    fine = ~torch.isnan(ref)
    off = (got - ref).abs()[fine]
    assert bool((off <= steps * U32 * ref.abs()[fine].clamp_min(2.0 ** -126)).all()), float(off.max())


SHAPES = [(1, 1), (1, 768), (3, 5), (7, 1003), (5, 1000), (130, 64), (33, 4096), (9, 257), (2, 8200), (3, 32768), (2, 33001)]


# ------------------------------------------------------------------------------------------ quantize
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("pad,qpad,offset", [(0, 0, 0), (8, 8, 8), (3, 5, 1)])
def test_quantize(k, cuda, dtype, rows, cols, pad, qpad, offset):
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(rows * 131 + cols)
    x = activations(torch, g, rows, cols, pad, types(torch)[dtype], offset)
    q, flat = rows_of(torch, rows, cols, qpad, torch.int8, fill=99, offset=offset)
    scale = torch.full((rows + 1,), -5.0, device="cuda")
    k.quantize_i8(x.data_ptr(), cols + pad, q.data_ptr(), cols + qpad, scale.data_ptr(), rows, cols, dtype, stream(torch))
    ref, m = rounded(torch, x.float())
    assert torch.equal(q, ref)
    close_f32(torch, scale[:rows], m.double() / 127.0, 1)
    assert float(scale[rows]) == -5.0
    kept = flat.clone()
    kept[offset:offset + rows * (cols + qpad)].view(rows, cols + qpad)[:, :cols] = 99
    assert bool((kept == 99).all())              # nothing between or behind the rows is written


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [16, 255, 5000, 40000])
def test_quantize_rows_that_are_special(k, cuda, cols):
    """Zeros, infinities, NaN, values at either end of the f32 range, and exact borders."""
    torch = cuda
    x = torch.randn(9, cols, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    x[0] = 0.0
    x[1, cols - 1] = math.inf
    x[2, 3] = math.nan
    x[3] *= 1e-41
    x[4] *= 1e37
    x[5, 0] = -math.inf
    ties = (torch.arange(cols, device="cuda") % 127).float() + 0.5
    x[6] = ties * torch.where(torch.arange(cols, device="cuda") % 2 == 0, 1.0, -1.0)
    x[6, 0] = 127.0
    x[7] = torch.nextafter(x[6], torch.full_like(x[6], 1000.0))
    x[7, 0] = 127.0
    x[8] = torch.nextafter(x[6], torch.full_like(x[6], -1000.0))
    x[8, 0] = 127.0
    x[6:9].clamp_(-127.0, 127.0)
    q, scale = torch.empty(9, cols, device="cuda", dtype=torch.int8), torch.empty(9, device="cuda")
    k.quantize_i8(x.data_ptr(), cols, q.data_ptr(), cols, scale.data_ptr(), 9, cols, F32, stream(torch))
    ref, m = rounded(torch, x)
    assert torch.equal(q, ref)
    close_f32(torch, scale, m.double() / 127.0, 1)


@pytest.mark.gpu
def test_quantize_no_columns(k, cuda):
    torch = cuda
    scale = torch.full((3,), 7.0, device="cuda")
    k.quantize_i8(None, 0, None, 0, scale.data_ptr(), 3, 0, BF16, stream(torch))
    assert scale.tolist() == [0.0, 0.0, 0.0]


@pytest.mark.gpu
def test_quantize_longest_row(k, cuda):
    """The longest row there may be, whose last group of eight ends past 2^31."""
    torch = cuda
    cols = (1 << 31) - 1
    x = torch.empty(cols, device="cuda", dtype=torch.bfloat16).normal_(generator=torch.Generator(device="cuda").manual_seed(6))
    x[cols - 1] = 50.0
    q, scale = torch.full((cols,), 99, device="cuda", dtype=torch.int8), torch.empty(1, device="cuda")
    k.quantize_i8(x.data_ptr(), cols, q.data_ptr(), cols, scale.data_ptr(), 1, cols, BF16, stream(torch))
    for at in range(0, cols, 1 << 27):
        part = x[at:at + (1 << 27)]
        assert torch.equal(q[at:at + (1 << 27)], (part.double() * 127.0 / 50.0).round().to(torch.int8))
    close_f32(torch, scale, torch.full((1,), 50.0, device="cuda").double() / 127.0, 1)


# ------------------------------------------------------------------------------------------ norm
def norm_reference(torch, x, r, w, eps):
    """(h, q, scale) in 64 bits, from h as it is stored."""
    h = (x.float() + r.float()).to(x.dtype) if r is not None else x
    q, m = rounded(torch, h.float() * w.float())
    return h, q, m.double() / 127.0 / (h.double().square().mean(1) + eps).sqrt()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,wtype", [(BF16, BF16), (BF16, F32), (F16, F16), (F32, F32), (F32, BF16)])
@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("pad,offset", [(0, 0), (8, 8), (3, 1)])
@pytest.mark.parametrize("form", ["written", "kept", "none", "over_x", "over_r"])
def test_rms_norm(k, cuda, dtype, wtype, rows, cols, pad, offset, form):
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(rows * 137 + cols)
    t = types(torch)
    x = activations(torch, g, rows, cols, pad, t[dtype], offset)
    r = activations(torch, g, rows, cols, pad, t[dtype], offset) if form != "none" else None
    w = (1.0 + 0.3 * torch.randn(cols, device="cuda", generator=g)).to(t[wtype])
    ref_h, ref_q, ref_scale = norm_reference(torch, x, r, w, 1e-5)
    q, flat = rows_of(torch, rows, cols, pad, torch.int8, fill=99, offset=offset)
    scale = torch.empty(rows, device="cuda")
    h = {"written": rows_of(torch, rows, cols, pad, t[dtype], fill=3.0, offset=offset)[0], "over_x": x, "over_r": r}.get(form)
    k.rms_norm_i8(x.data_ptr(), cols + pad, None if r is None else r.data_ptr(), cols + pad, w.data_ptr(),
                  None if h is None else h.data_ptr(), cols + pad, q.data_ptr(), cols + pad, scale.data_ptr(), rows, cols, dtype,
                  wtype, 1e-5, stream(torch))
    if h is not None:
        assert torch.equal(h, ref_h)
    assert torch.equal(q, ref_q)
    # a sum of `cols` squares adds at most log2(cols) + 32 roundings (32 in a thread, then in pairs; a long
    # row: cols / 1024 in a thread), halved by the root, and the scale four of its own
    close_f32(torch, scale, ref_scale, (math.log2(cols) + 34) / 2 + 4)
    kept = flat.clone()
    kept[offset:offset + rows * (cols + pad)].view(rows, cols + pad)[:, :cols] = 99
    assert bool((kept == 99).all())


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [16, 1001, 6000, 40000])
def test_rms_norm_rows_that_are_special(k, cuda, cols):
    """Zero rows, infinities, NaN, squares that overflow or vanish, sums that overflow."""
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(2)
    x, r = (torch.randn(8, cols, device="cuda", generator=g) for _ in range(2))
    x[0] = 0.0
    r[0] = 0.0
    x[1, 5] = math.nan
    r[2, cols - 1] = math.inf
    x[3] *= 1e25
    r[3] *= 1e25
    x[4] *= 1e-30
    r[4] *= 1e-30
    x[5, 1] = r[5, 1] = 3e38
    x[6] = -r[6]
    x[7] *= 2e36
    w = 1.0 + 0.1 * torch.randn(cols, device="cuda", generator=g)
    h, q, scale = torch.empty_like(x), torch.empty(8, cols, device="cuda", dtype=torch.int8), torch.empty(8, device="cuda")
    ref_h, ref_q, ref_scale = norm_reference(torch, x, r, w, 1e-6)
    k.rms_norm_i8(x.data_ptr(), cols, r.data_ptr(), cols, w.data_ptr(), h.data_ptr(), cols, q.data_ptr(), cols, scale.data_ptr(), 8,
                  cols, F32, F32, 1e-6, stream(torch))
    assert torch.equal(torch.nan_to_num(h, 1.5), torch.nan_to_num(ref_h, 1.5))
    assert torch.equal(q, ref_q)
    close_f32(torch, scale, ref_scale, (math.log2(cols) + 34) / 2 + 4)


def check_norm_f32(torch, k, x, w, eps):
    """A norm of f32 rows whose residual is zero, q and h equal and the scale within the roundings of a sum of squares
    (as in test_rms_norm)."""
    rows, cols = x.shape
    r = torch.zeros_like(x)
    h, q, scale = torch.empty_like(x), torch.empty(rows, cols, device="cuda", dtype=torch.int8), torch.empty(rows, device="cuda")
    ref_h, ref_q, ref_scale = norm_reference(torch, x, r, w, eps)
    k.rms_norm_i8(x.data_ptr(), cols, r.data_ptr(), cols, w.data_ptr(), h.data_ptr(), cols, q.data_ptr(), cols, scale.data_ptr(), rows,
                  cols, F32, F32, eps, stream(torch))
    assert torch.equal(h, ref_h) and torch.equal(q, ref_q)
    close_f32(torch, scale, ref_scale, (math.log2(cols) + 34) / 2 + 4)


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [16, 1001, 6000, 40000])
def test_rms_norm_large_eps(k, cuda, cols):
    """An eps of the size of squares whose sum overflows, and beside smaller ones."""
    torch = cuda
    u = 0.5 + torch.rand(2, cols, device="cuda", generator=torch.Generator(device="cuda").manual_seed(8))
    check_norm_f32(torch, k, u * torch.tensor([[1.5e19], [1e18]], device="cuda"), torch.ones(cols, device="cuda"), 3e38)


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [16, 1001, 6000, 40000])
def test_rms_norm_small_products(k, cuda, cols):
    """Values and weights whose products leave the normal range, under an eps that brings the scale back into it."""
    torch = cuda
    u = 0.5 + torch.rand(3, cols, device="cuda", generator=torch.Generator(device="cuda").manual_seed(9))
    check_norm_f32(torch, k, u * torch.tensor([[1e-35], [1e-36], [1e-33]], device="cuda"), torch.full((cols,), 1e-4, device="cuda"), 1e-30)


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [200000, 3000001])
def test_rms_norm_long_sums(k, cuda, cols):
    """Equal values: the roundings of a sum in 32 bits would not cancel."""
    torch = cuda
    check_norm_f32(torch, k, torch.tensor([[1.1], [0.3], [1.7], [3e19]], device="cuda").expand(4, cols).contiguous(),
                   torch.ones(cols, device="cuda"), 1e-5)


# ------------------------------------------------------------------------------------------ gemm
def operand(torch, g, rows, cols, pad, offset=0):
    v, _ = rows_of(torch, rows, cols, pad, torch.int8, fill=77, offset=offset)
    v.copy_(torch.randint(-128, 128, (rows, cols), device="cuda", generator=g, dtype=torch.int32))
    return v


def scratch_for(torch, k, a, lda, b, ldb, m, n, kk):
    size = k.gemm_i8_scratch_bytes(a.data_ptr(), lda, b.data_ptr(), ldb, m, n, kk)
    return torch.empty(max(size, 1), device="cuda", dtype=torch.uint8), size


GEMMS = [(1, 1, 1), (1, 2304, 768), (1, 16, 5000), (2, 130, 33), (7, 129, 127), (16, 1000, 128), (17, 64, 4096), (31, 513, 640),
         (64, 768, 768), (65, 2000, 100), (100, 100, 2049), (128, 128, 128), (129, 257, 129), (200, 1000, 4112), (256, 256, 64),
         (300, 520, 1000), (513, 1025, 257), (1000, 2304, 768), (2050, 700, 1536)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,kk", GEMMS)
@pytest.mark.parametrize("pad,offset", [(0, 0), (16, 16), (1, 3)])
def test_gemm_sums(k, cuda, m, n, kk, pad, offset):
    """The raw sums, over the whole range of 8-bit integers, equal those in 64 bits (below 2^53 exact)."""
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(m * 31 + n * 7 + kk)
    a, b = operand(torch, g, m, kk, pad, offset), operand(torch, g, n, kk, pad, offset)
    c, flat = rows_of(torch, m, n, pad, torch.int32, fill=123456789, offset=offset)
    s, size = scratch_for(torch, k, a, kk + pad, b, kk + pad, m, n, kk)
    k.gemm_i8(a.data_ptr(), kk + pad, b.data_ptr(), kk + pad, None, None, None, c.data_ptr(), n + pad, m, n, kk, S32, 0, s.data_ptr(),
              size, stream(torch))
    assert torch.equal(c.double(), a.double() @ b.double().t())
    kept = flat.clone()
    kept[offset:offset + m * (n + pad)].view(m, n + pad)[:, :n] = 123456789
    assert bool((kept == 123456789).all())


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["pair", "0x1", "0x2", "0x4", "0x8", "32x1", "32x3", "32x8", "64x1", "64x4", "64x7", "128x1", "128x2", "128x5", "128x8"])
@pytest.mark.parametrize("m,n,kk", [(1, 300, 1500), (2, 77, 4113), (3, 515, 768), (6, 129, 200), (8, 64, 999), (70, 130, 1024), (300, 520, 1000), (515, 1031, 1280)])
@pytest.mark.parametrize("npad", [0, 3])
def test_gemm_every_form(k, cuda, monkeypatch, form, m, n, kk, npad):
    """CTA pairs, single tiles of 32 to 128 tokens with K cut over up to 8 CTAs, whatever the size, and (0x: up to 8
    tokens) sums in registers with K cut over warps."""
    torch = cuda
    monkeypatch.setenv("B200_GEMM_I8_FORM", form)
    g = torch.Generator(device="cuda").manual_seed(m + n + kk)
    a, b = operand(torch, g, m, kk, 0), operand(torch, g, n, kk, 0)
    s, size = scratch_for(torch, k, a, kk, b, kk, m, n, kk)
    sa, sb = torch.rand(m, device="cuda", generator=g) * 0.01, torch.rand(n, device="cuda", generator=g) * 0.01
    bias = torch.randn(n, device="cuda", generator=g)
    for out_type in (S32, F32, BF16, F16):
        dtype = torch.int32 if out_type == S32 else types(torch)[out_type]
        c, flat = rows_of(torch, m, n, npad, dtype, fill=99)
        ptrs = [None] * 3 if out_type == S32 else [t.data_ptr() for t in (sa, sb, bias)]
        k.gemm_i8(a.data_ptr(), kk, b.data_ptr(), kk, *ptrs, c.data_ptr(), n + npad, m, n, kk, out_type, 0, s.data_ptr(), size,
                  stream(torch))
        if out_type == S32:
            assert torch.equal(c.double(), a.double() @ b.double().t())
        else:
            check_gemm(torch, c, *gemm_reference(torch, a, b, sa, sb, bias, False), out_type, False)
        kept = flat.clone()
        kept[:m * (n + npad)].view(m, n + npad)[:, :n] = 99
        assert bool((kept == 99).all())


def gemm_reference(torch, a, b, sa, sb, bias, gelu):
    c = a.double() @ b.double().t()
    if sa is not None:
        c = c * sa.double()[:, None]
    if sb is not None:
        c = c * sb.double()
    v = c if bias is None else c + bias.double()
    size = c.abs() if bias is None else c.abs() + bias.double().abs()
    if gelu:
        v = v / (1.0 + torch.exp(-2.0 * math.sqrt(2.0 / math.pi) * (v + 0.044715 * v ** 3)))
    return v, size


def check_gemm(torch, got, ref, size, out_type, gelu):
    """The sum's conversion, two products and the bias: four roundings of at most `size` each.  GELU: its slope is
    below 1.13; its own f32 operations leave 2^-19 of the result (the exponent's argument, of magnitude u, carries
    4 half steps of u: below u = 10 the sigmoid is then off by 40 * 2^-24 relative, and beyond that the result is v
    or vanishes, to below 2^-20 in absolute terms)."""
    half = {F32: U32, BF16: 2.0 ** -8, F16: 2.0 ** -11}[out_type]
    off = 4 * U32 * size * (1.13 if gelu else 1.0) + (2.0 ** -18 * ref.abs() + 2.0 ** -20 if gelu else 0.0)
    off = off + half * (ref.abs() + off) + (2.0 ** -25 if out_type == F16 else 0.0)
    d = (got.double() - ref).abs()
    assert bool((d <= off).all()), float((d - off).max())


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,kk", GEMMS)
@pytest.mark.parametrize("out_type", [BF16, F16, F32])
@pytest.mark.parametrize("form", ["scales", "bias", "gelu", "bare"])
def test_gemm_scaled(k, cuda, m, n, kk, out_type, form):
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(m * 37 + n * 11 + kk)
    pad = {"scales": 0, "bias": 5, "gelu": 16, "bare": 0}[form]
    a, b = operand(torch, g, m, kk, pad), operand(torch, g, n, kk, 0)
    unit = 1.0 / (5000.0 * math.sqrt(kk))
    sa = (0.5 + torch.rand(m, device="cuda", generator=g)) * 0.05 if form != "bare" else None
    sb = (0.5 + torch.rand(n, device="cuda", generator=g)) * unit * 20 if form != "bare" else None
    bias = torch.randn(n, device="cuda", generator=g) if form in ("bias", "gelu") else None
    if form == "bare":
        a.clamp_(-3, 3)
        b.clamp_(-3, 3)                          # the sums stay inside f16
    c, flat = rows_of(torch, m, n, pad, types(torch)[out_type], fill=-7.0)
    s, size = scratch_for(torch, k, a, kk + pad, b, kk, m, n, kk)
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    k.gemm_i8(a.data_ptr(), kk + pad, b.data_ptr(), kk, ptr(sa), ptr(sb), ptr(bias), c.data_ptr(), n + pad, m, n, kk, out_type,
              1 if form == "gelu" else 0, s.data_ptr(), size, stream(torch))
    ref, big = gemm_reference(torch, a, b, sa, sb, bias, form == "gelu")
    check_gemm(torch, c, ref, big, out_type, form == "gelu")
    kept = flat.clone()
    kept[:m * (n + pad)].view(m, n + pad)[:, :n] = -7.0
    assert bool((kept == -7.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("m", [3, 300])
def test_gemm_no_depth_and_special_scales(k, cuda, m):
    torch = cuda
    n = 70
    bias = torch.randn(n, device="cuda")
    c = torch.full((m, n), 9.0, device="cuda")
    k.gemm_i8(None, 0, None, 0, None, None, bias.data_ptr(), c.data_ptr(), n, m, n, 0, F32, 0, None, 0, stream(torch))
    assert torch.equal(c, bias.expand(m, n))
    z = torch.full((m, n), 9, device="cuda", dtype=torch.int32)
    k.gemm_i8(None, 0, None, 0, None, None, None, z.data_ptr(), n, m, n, 0, S32, 0, None, 0, stream(torch))
    assert int(z.abs().max()) == 0
    # a token whose scale is NaN (its row held no numbers) gives NaN, the others stay as they are
    a, b = torch.ones(m, 64, device="cuda", dtype=torch.int8), torch.ones(n, 64, device="cuda", dtype=torch.int8)
    a[1] = 0
    sa, sb = torch.ones(m, device="cuda"), torch.ones(n, device="cuda")
    sa[1] = math.nan
    k.gemm_i8(a.data_ptr(), 64, b.data_ptr(), 64, sa.data_ptr(), sb.data_ptr(), None, c.data_ptr(), n, m, n, 64, F32, 0, None, 0,
              stream(torch))
    assert bool(torch.isnan(c[1]).all()) and bool((c[[0] + list(range(2, m))] == 64.0).all())


@pytest.mark.gpu
def test_gemm_deepest_sum(k, cuda):
    """-128 * -128 over the deepest K: the sum next to 2^31."""
    torch = cuda
    kk = 131071
    a = torch.full((2, kk), -128, device="cuda", dtype=torch.int8)
    b = torch.full((130, kk), -128, device="cuda", dtype=torch.int8)
    b[1::2] = 127
    c = torch.empty(2, 130, device="cuda", dtype=torch.int32)
    s, size = scratch_for(torch, k, a, kk, b, kk, 2, 130, kk)
    k.gemm_i8(a.data_ptr(), kk, b.data_ptr(), kk, None, None, None, c.data_ptr(), 130, 2, 130, kk, S32, 0, s.data_ptr(), size,
              stream(torch))
    assert bool((c[:, ::2] == 16384 * kk).all()) and bool((c[:, 1::2] == -128 * 127 * kk).all())


# ------------------------------------------------------------------------------------------ together
def layer(torch, k, s):
    """norm -> hidden product with GELU -> quantize -> product back to the width: a block's MLP in 8 bits."""
    st = stream(torch)
    t, d, f = s["tokens"], s["width"], s["hidden"]
    k.rms_norm_i8(s["x"].data_ptr(), d, s["r"].data_ptr(), d, s["w"].data_ptr(), s["h"].data_ptr(), d, s["q1"].data_ptr(), d,
                  s["s1"].data_ptr(), t, d, BF16, F32, 1e-5, st)
    k.gemm_i8(s["q1"].data_ptr(), d, s["w1"].data_ptr(), d, s["s1"].data_ptr(), s["sw1"].data_ptr(), s["b1"].data_ptr(),
              s["y"].data_ptr(), f, t, f, d, BF16, 1, None, 0, st)
    k.quantize_i8(s["y"].data_ptr(), f, s["q2"].data_ptr(), f, s["s2"].data_ptr(), t, f, BF16, st)
    k.gemm_i8(s["q2"].data_ptr(), f, s["w2"].data_ptr(), f, s["s2"].data_ptr(), s["sw2"].data_ptr(), None, s["z"].data_ptr(), d, t, d,
              f, BF16, 0, None, 0, st)


def layer_state(torch, k, tokens, width=768, hidden=2048):
    g = torch.Generator(device="cuda").manual_seed(tokens)
    new = lambda dtype, *shape: torch.zeros(*shape, device="cuda", dtype=dtype)  # noqa: E731
    s = dict(tokens=tokens, width=width, hidden=hidden)
    s["x"], s["r"] = (torch.randn(tokens, width, device="cuda", generator=g).bfloat16() for _ in range(2))
    s["w"] = 1.0 + 0.1 * torch.randn(width, device="cuda", generator=g)
    s["b1"] = 0.1 * torch.randn(hidden, device="cuda", generator=g)
    for name, n, d in (("w1", hidden, width), ("w2", width, hidden)):
        s["f" + name] = torch.randn(n, d, device="cuda", generator=g) / math.sqrt(d)
        s[name], s["s" + name] = new(torch.int8, n, d), new(torch.float32, n)
        k.quantize_i8(s["f" + name].data_ptr(), d, s[name].data_ptr(), d, s["s" + name].data_ptr(), n, d, F32, stream(torch))
    s["h"], s["y"], s["z"] = new(torch.bfloat16, tokens, width), new(torch.bfloat16, tokens, hidden), new(torch.bfloat16, tokens, width)
    s["q1"], s["q2"] = new(torch.int8, tokens, width), new(torch.int8, tokens, hidden)
    s["s1"], s["s2"] = new(torch.float32, tokens), new(torch.float32, tokens)
    return s


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 5, 64, 333, 1024])
def test_layer(k, cuda, tokens):
    """The chain against its steps in 64 bits on what each step was given, and against the layer without 8 bits:
    a value rounded to 8 bits is off by half of m / 127, for normal rows about 1% of a value's size, and errors of
    many values add up like their roots: 3% of the result covers four such roundings."""
    torch = cuda
    s = layer_state(torch, k, tokens)
    layer(torch, k, s)
    h, q1, s1 = norm_reference(torch, s["x"], s["r"], s["w"], 1e-5)
    assert torch.equal(s["h"], h) and torch.equal(s["q1"], q1)
    y, big = gemm_reference(torch, s["q1"], s["w1"], s["s1"], s["sw1"], s["b1"], True)
    check_gemm(torch, s["y"], y, big, BF16, True)
    assert torch.equal(s["q2"], rounded(torch, s["y"].float())[0])
    z, big = gemm_reference(torch, s["q2"], s["w2"], s["s2"], s["sw2"], None, False)
    check_gemm(torch, s["z"], z, big, BF16, False)
    n = h.double() * s["w"].double() / (h.double().square().mean(1, keepdim=True) + 1e-5).sqrt()
    v = n @ s["fw1"].double().t() + s["b1"].double()
    v = v / (1.0 + torch.exp(-2.0 * math.sqrt(2.0 / math.pi) * (v + 0.044715 * v ** 3)))
    full = v @ s["fw2"].double().t()
    assert float((s["z"].double() - full).norm() / full.norm()) <= 0.03


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [3, 300])
def test_layer_captured_and_on_another_stream(k, cuda, tokens):
    torch = cuda
    s = layer_state(torch, k, tokens)
    layer(torch, k, s)
    want = s["z"].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s["z"].zero_()
        layer(torch, k, s)
    side.synchronize()
    assert torch.equal(s["z"], want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer(torch, k, s)
    x = s["x"].clone()
    s["x"].copy_(torch.flip(x, [1]))
    layer(torch, k, s)
    flipped = s["z"].clone()
    for inputs, out in ((x, want), (torch.flip(x, [1]), flipped)):
        s["x"].copy_(inputs)
        s["z"].zero_()
        graph.replay()
        assert torch.equal(s["z"], out)


@pytest.mark.gpu
def test_two_streams_at_once(k, cuda):
    """Calls that overlap on the GPU share nothing: the results are those of calls one after the other."""
    torch = cuda
    states = [layer_state(torch, k, t) for t in (40, 700)]
    want = []
    for s in states:
        layer(torch, k, s)
        want.append(s["z"].clone())
        s["z"].zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    for _ in range(5):
        for s, side in zip(states, streams):
            with torch.cuda.stream(side):
                layer(torch, k, s)
    torch.cuda.synchronize()
    for s, w in zip(states, want):
        assert torch.equal(s["z"], w)


@pytest.mark.gpu
def test_offsets_past_32_bits(k, cuda):
    """Arrays of more than 2^31 elements: the rows on either side of that place and the last ones."""
    torch = cuda
    rows, cols = 270000, 8000
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.empty(rows, cols, device="cuda", dtype=torch.bfloat16)
    x.normal_(generator=g)
    q, scale = torch.empty(rows, cols, device="cuda", dtype=torch.int8), torch.empty(rows, device="cuda")
    k.quantize_i8(x.data_ptr(), cols, q.data_ptr(), cols, scale.data_ptr(), rows, cols, BF16, stream(torch))
    at = torch.tensor([0, (1 << 31) // cols - 1, (1 << 31) // cols, rows - 2, rows - 1], device="cuda")
    ref, m = rounded(torch, x[at].float())
    assert torch.equal(q[at], ref)
    close_f32(torch, scale[at], m.double() / 127.0, 1)
    del x
    b = operand(torch, g, cols, 48, 0)
    c = torch.empty(rows, cols, device="cuda", dtype=torch.bfloat16)
    k.gemm_i8(q.data_ptr(), cols, b.data_ptr(), 48, scale.data_ptr(), None, None, c.data_ptr(), cols, rows, cols, 48, BF16, 0, None, 0,
              stream(torch))
    check_gemm(torch, c[at], *gemm_reference(torch, q[at][:, :48], b, scale[at], None, None, False), BF16, False)


COUNT_READS = """
import ctypes, sys
import torch
from torch.profiler import ProfilerActivity, profile
sys.path.insert(0, sys.argv[2])
from pjrt_b200 import kernels
lib, k = ctypes.CDLL(sys.argv[1]), kernels.Kernels(sys.argv[1])
a = torch.ones(300, 64, device="cuda", dtype=torch.int8)
c = torch.empty(300, 300, device="cuda", dtype=torch.int32)
def reads():
    with profile(activities=[ProfilerActivity.CUDA]) as p:
        assert lib.b200_take_device_error() == 0
        torch.cuda.synchronize()
    return sum("Memcpy DtoH" in e.name for e in p.events())
reads()
before = reads()
k.gemm_i8(a.data_ptr(), 64, a.data_ptr(), 64, None, None, None, c.data_ptr(), 300, 300, 300, 64, 4)
print("reads", before, reads())
"""


@pytest.mark.gpu
def test_error_flag_read_only_behind_products(lib_path, cuda):
    """b200_take_device_error copies the 8-bit product's flag from the device once a product has been launched, and
    before that the four flags of the other kernels alone."""
    import subprocess
    import sys
    from conftest import PKG
    r = subprocess.run([sys.executable, "-c", COUNT_READS, lib_path, PKG], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    before, after = (int(n) for n in r.stdout.split("reads")[1].split())
    if not after:
        pytest.skip("copies are not recorded here")
    assert (before, after) == (4, 5)


# ------------------------------------------------------------------------------------------ every launch form
def row_pitch(cols, aligned):
    """Rows 16-byte aligned, or at odd places."""
    return (cols + 15) // 8 * 8 if aligned else cols + 1 + cols % 2


# with 1200 rows and with three: rows in 1 to 4 groups of eight a lane, in blocks of up to 256, 512 and 1024 threads
WIDTHS = [301, 701, 1003, 1501, 2041, 3501, 5003, 12005, 20011]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows", [3, 1200])
@pytest.mark.parametrize("cols", WIDTHS)
@pytest.mark.parametrize("aligned", [True, False])
def test_quantize_every_form(k, cuda, dtype, rows, cols, aligned):
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(rows * 139 + cols)
    ld = row_pitch(cols, aligned)
    x = activations(torch, g, rows, cols, ld - cols, types(torch)[dtype])
    q, flat = rows_of(torch, rows, cols, ld - cols, torch.int8, fill=99)
    scale = torch.empty(rows, device="cuda")
    k.quantize_i8(x.data_ptr(), ld, q.data_ptr(), ld, scale.data_ptr(), rows, cols, dtype, stream(torch))
    ref, m = rounded(torch, x.float())
    assert torch.equal(q, ref)
    close_f32(torch, scale, m.double() / 127.0, 1)
    flat[:rows * ld].view(rows, ld)[:, :cols] = 99
    assert bool((flat == 99).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,wtype", [(BF16, BF16), (F16, F32), (F32, F32)])
@pytest.mark.parametrize("rows", [3, 1200])
@pytest.mark.parametrize("cols", WIDTHS)
@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("form", ["written", "over_x"])
def test_rms_norm_every_form(k, cuda, dtype, wtype, rows, cols, aligned, form):
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(rows * 149 + cols)
    t, ld = types(torch), row_pitch(cols, aligned)
    x, r = (activations(torch, g, rows, cols, ld - cols, t[dtype]) for _ in range(2))
    w = (1.0 + 0.3 * torch.randn(cols, device="cuda", generator=g)).to(t[wtype])
    ref_h, ref_q, ref_scale = norm_reference(torch, x, r, w, 1e-5)
    h = x if form == "over_x" else rows_of(torch, rows, cols, ld - cols, t[dtype])[0]
    q, flat = rows_of(torch, rows, cols, ld - cols, torch.int8, fill=99)
    scale = torch.empty(rows, device="cuda")
    k.rms_norm_i8(x.data_ptr(), ld, r.data_ptr(), ld, w.data_ptr(), h.data_ptr(), ld, q.data_ptr(), ld, scale.data_ptr(), rows, cols,
                  dtype, wtype, 1e-5, stream(torch))
    assert torch.equal(h, ref_h) and torch.equal(q, ref_q)
    close_f32(torch, scale, ref_scale, (math.log2(cols) + 34) / 2 + 4)
    flat[:rows * ld].view(rows, ld)[:, :cols] = 99
    assert bool((flat == 99).all())


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [16, 1001, 6000, 40000])
def test_rms_norm_large_values_and_weights(k, cuda, cols):
    """Squares that overflow beside weights as large: the scale is finite, and no step on the way to it overflows."""
    torch = cuda
    u = 0.5 + 0.5 * torch.rand(1, cols, device="cuda", generator=torch.Generator(device="cuda").manual_seed(7))
    check_norm_f32(torch, k, 1e20 * u, torch.full((cols,), 1e18, device="cuda"), 1e-5)


def check_every_result(torch, k, m, n, kk, pad, npad):
    """The product in every type, with and without GELU and in raw sums: all of C, and what lies between its rows."""
    g = torch.Generator(device="cuda").manual_seed(m * 41 + n * 13 + kk)
    a, b = operand(torch, g, m, kk, pad), operand(torch, g, n, kk, pad)
    s, size = scratch_for(torch, k, a, kk + pad, b, kk + pad, m, n, kk)
    sa = (0.5 + torch.rand(m, device="cuda", generator=g)) * 0.05
    sb = (0.5 + torch.rand(n, device="cuda", generator=g)) * 20 / (5000.0 * math.sqrt(kk))
    bias = torch.randn(n, device="cuda", generator=g)
    for out_type, act in ((S32, 0), (F32, 0), (F32, 1), (BF16, 0), (BF16, 1), (F16, 0), (F16, 1)):
        c, flat = rows_of(torch, m, n, npad, torch.int32 if out_type == S32 else types(torch)[out_type], fill=99)
        ptrs = [None] * 3 if out_type == S32 else [t.data_ptr() for t in (sa, sb, bias)]
        k.gemm_i8(a.data_ptr(), kk + pad, b.data_ptr(), kk + pad, *ptrs, c.data_ptr(), n + npad, m, n, kk, out_type, act, s.data_ptr(),
                  size, stream(torch))
        if out_type == S32:
            assert torch.equal(c.double(), a.double() @ b.double().t())
        else:
            check_gemm(torch, c, *gemm_reference(torch, a, b, sa, sb, bias, bool(act)), out_type, bool(act))
        flat[:m * (n + npad)].view(m, n + npad)[:, :n] = 99
        assert bool((flat == 99).all())


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,kk,pad", [(4500, 4096, 1000, 8), (4500, 4100, 1000, 0), (8192, 2301, 768, 0), (5000, 4104, 130, 14)])
@pytest.mark.parametrize("npad", [0, 8, 3])
def test_gemm_many_tiles_a_pair(k, cuda, monkeypatch, m, n, kk, pad, npad):
    """Pairs of CTAs that work on three and more tiles each, with K in more blocks than a tile has stages and in fewer,
    rows of C that TMA can write and that it cannot."""
    monkeypatch.setenv("B200_GEMM_I8_FORM", "pair")
    check_every_result(cuda, k, m, n, kk, pad, npad)


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["pair", "0x1", "0x4", "32x1", "32x6", "64x1", "64x2", "128x1", "128x3"])
@pytest.mark.parametrize("m,n,kk", [(1, 300, 1500), (7, 515, 768), (70, 130, 1024), (300, 520, 1000)])
def test_gemm_every_form_and_result(k, cuda, monkeypatch, form, m, n, kk):
    monkeypatch.setenv("B200_GEMM_I8_FORM", form)
    check_every_result(cuda, k, m, n, kk, 0, 3)


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["pair", "0x8", "32x1", "32x8", "64x4", "128x1"])
@pytest.mark.parametrize("m", [4, 100])
def test_gemm_deepest_sum_in_every_form(k, cuda, monkeypatch, form, m):
    torch = cuda
    monkeypatch.setenv("B200_GEMM_I8_FORM", form)
    kk, n = 131071, 130
    a = torch.full((m, kk), -128, device="cuda", dtype=torch.int8)
    b = torch.full((n, kk), -128, device="cuda", dtype=torch.int8)
    b[1::2] = 127
    c = torch.empty(m, n, device="cuda", dtype=torch.int32)
    s, size = scratch_for(torch, k, a, kk, b, kk, m, n, kk)
    k.gemm_i8(a.data_ptr(), kk, b.data_ptr(), kk, None, None, None, c.data_ptr(), n, m, n, kk, S32, 0, s.data_ptr(), size, stream(torch))
    assert bool((c[:, ::2] == 16384 * kk).all()) and bool((c[:, 1::2] == -128 * 127 * kk).all())


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["pair", "0x1", "32x1", "64x1", "128x1"])
@pytest.mark.parametrize("m,n,kk", [(1, 1, 1), (5, 1, 1), (100, 1, 17), (3, 7, 1), (300, 1, 256)])
def test_gemm_smallest_in_every_form(k, cuda, monkeypatch, form, m, n, kk):
    monkeypatch.setenv("B200_GEMM_I8_FORM", form)
    check_every_result(cuda, k, m, n, kk, 0, 0)
