"""The 8-bit serving path: block quantisation, the block-scaled product, the residual norm that feeds it, against plain
64-bit implementations on the same stored inputs; refusals on the CPU.

Bounds (u = 2^-24, an fp32 rounding; half a step of a type t is finfo(t).eps / 2):
  quantisation      scale is one fp32 division of an exact maximum, the value one fp32 division and one conversion:
                    bit-equal to the same three operations in torch.
  product           a sum of up to 128 products per block (each exact in fp32) and a sum over blocks; an adder that
                    truncates loses at most 2u of the magnitudes per addition, so the error is at most
                    (2*128 + 2*blocks + 8) u * sum |x w s|, plus half a step of the output type.
  residual norm     h is bit-equal to torch's sum and rounding.  The sum of squares adds H/256 + 48 terms in a row at
                    most on any path, its root halves the relative error; three more roundings:
                    |y - ref| <= (half step + (H/256 + 64) u) |ref|.
  its e4m3 form     |q s - ref| <= half a step of e4m3 (2^-4 of the value, or 2^-10 scales below the normal range),
                    plus the fp32 error above; the factor 1 + 2^-8 covers a tie decided the other way.
  its backward      sums of terms a_i: error <= c u * sum |a_i| with c = the longest chain of additions.
"""
import math

import pytest
import torch

from quick_ssm_b200 import _lib, fp8
from quick_ssm_b200.norm import add_rms_norm, add_rms_norm_fp8

gpu = pytest.mark.gpu
U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
ids = lambda v: {F32: "fp32", F16: "fp16", BF16: "bf16"}.get(v) if isinstance(v, torch.dtype) else None  # noqa: E731


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


# ------------------------------------------------------------------------------------------------
# plain forms
# ------------------------------------------------------------------------------------------------
def plain_quantize(v, block_rows):
    """fp32 [rows, K] on the CPU -> (e4m3, scales), block by block."""
    rows, K = v.shape
    q = torch.empty(rows, K, dtype=torch.float8_e4m3fn)
    scales = torch.empty(-(-rows // block_rows), -(-K // 128))
    for i in range(scales.shape[0]):
        for j in range(scales.shape[1]):
            b = v[i * block_rows:(i + 1) * block_rows, j * 128:(j + 1) * 128]
            s = b.abs().max().clamp_min(2.0 ** -100) / 448.0
            scales[i, j] = s
            q[i * block_rows:(i + 1) * block_rows, j * 128:(j + 1) * 128] = (b / s).clamp(-448, 448).to(torch.float8_e4m3fn)
    return q, scales


def wide(q, scales, block_rows):
    rows, K = q.shape
    per = scales.double().repeat_interleave(block_rows, 0)[:rows].repeat_interleave(128, 1)[:, :K]
    return q.float().double() * per


def plain_norm(x, res, w, eps):
    """64-bit y, h as stored (64-bit), 1/rms."""
    h = x if res is None else (x.float() + res.float()).to(res.dtype)
    hd = h.double()
    r = 1.0 / torch.sqrt(hd.square().mean(-1, keepdim=True) + eps)
    return hd * r * w.double(), h, r


def bits(q):
    """e4m3 bytes; both of its NaNs (0x7f, 0xff: a NaN has no sign to compare) as one."""
    b = q.contiguous().view(torch.uint8)
    return torch.where((b & 0x7F) == 0x7F, torch.full_like(b, 0x7F), b)


def norm_inputs(rows, H, xd, rd, seed=0):
    g = torch.Generator().manual_seed(seed + rows * 7 + H)
    x = torch.randn(rows, H, generator=g).mul(torch.randn(H, generator=g).exp()).to(xd)
    res = torch.randn(rows, H, generator=g).mul(3).to(rd)
    w = 1 + 0.3 * torch.randn(H, generator=g)
    return x, res, w, g


# ------------------------------------------------------------------------------------------------
# refusals (CPU)
# ------------------------------------------------------------------------------------------------
def test_operands_check_their_shapes_and_types():
    v = torch.zeros(3, 200, dtype=torch.uint8).view(torch.float8_e4m3fn)
    fp8.Fp8Rows(v, torch.ones(3, 2))
    fp8.Fp8Weight(v, torch.ones(1, 2))
    for bad in (torch.ones(3, 1), torch.ones(2, 2), torch.ones(6), torch.ones(1, 3, 2)):
        with pytest.raises(ValueError):
            fp8.Fp8Rows(v, bad)
    with pytest.raises(ValueError):
        fp8.Fp8Weight(v, torch.ones(2, 2))
    with pytest.raises(TypeError):
        fp8.Fp8Rows(v, torch.ones(3, 2, dtype=F16))
    with pytest.raises(TypeError):
        fp8.Fp8Weight(v.view(torch.uint8), torch.ones(1, 2))


def test_cpu_tensors_are_refused():
    x, w = torch.randn(4, 128), torch.ones(128)
    q = fp8.Fp8Rows(torch.zeros(4, 128, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.ones(4, 1))
    qw = fp8.Fp8Weight(q.values, torch.ones(1, 1))
    for call in (lambda: add_rms_norm(x, x, w), lambda: add_rms_norm_fp8(x, None, w), lambda: fp8.quantize_rows(x),
                 lambda: fp8.quantize_weight(x), lambda: fp8.matmul_fp8(q, qw)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_c_entries_check_arguments_without_gpu():
    import ctypes
    lib = _lib.load()
    one, odd = ctypes.c_void_p(256), ctypes.c_void_p(264)
    mm = lambda x=one, xs=64, M=4, N=4, K=64, ys=4, out=2, bias=None: lib.qssm_matmul_fp8(  # noqa: E731
        x, one, one, one, bias, one, M, N, K, xs, 1, M, 64, 1, 1, ys, out, 0, None, None)
    assert mm(M=0) == 0 and mm(N=0) == 0
    assert mm(M=-1) == -2 and mm(out=5) == -3 and mm(x=None) == -1
    assert mm(K=0) == -2 and mm(M=2 ** 31) == -2
    assert mm(x=odd) == -4 and mm(xs=72) == -4 and mm(xs=48) == -4 and mm(ys=3) == -4
    norm = lambda rows=2, xd=2, rd=2, x=one, ys=8: lib.qssm_add_rmsnorm_fwd(  # noqa: E731
        x, one, one, one, one, None, rows, 8, 8, 8, ys, 8, 1e-5, xd, rd, 0, None)
    assert norm(rows=0) == 0 and norm(rows=-1) == -2 and norm(xd=9) == -3 and norm(rd=1) == -3
    assert norm(x=None) == -1 and norm(ys=7) == -4
    assert lib.qssm_add_rmsnorm_fp8(one, one, one, one, one, None, 2, 8, 8, 8, 16, 8, 1, 2, 1e-5, 2, 2, 0, None) == -1
    bwd = lambda ws, nbytes: lib.qssm_add_rmsnorm_bwd(  # noqa: E731
        one, one, one, None, one, one, None, one, ws, nbytes, 2, 8, 8, 8, 0, 8, 0, 0, 0, 0, None)
    assert bwd(None, 64) == -1 and bwd(one, 63) == -6 and bwd(ctypes.c_void_p(8), 64) == -6
    assert lib.qssm_add_rmsnorm_workspace_bytes(2, 8) == 64 and lib.qssm_add_rmsnorm_workspace_bytes(0, 8) == 0
    assert lib.qssm_quant_fp8_rows(one, one, one, 2, 8, 8, 7, 1, 2, 0, None) == -4
    assert lib.qssm_quant_fp8_blocks(one, None, one, 2, 8, 8, 8, 1, 2, 0, None) == -1
    assert lib.qssm_quant_fp8_blocks(one, one, one, 0, 8, 8, 8, 1, 2, 0, None) == 0


# ------------------------------------------------------------------------------------------------
# quantisation
# ------------------------------------------------------------------------------------------------
SIZES = [(1, 1), (3, 17), (2, 128), (5, 129), (130, 300), (7, 1000), (64, 2050), (300, 256), (2, 5000)]


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=ids)
@pytest.mark.parametrize("shape", SIZES, ids=str)
def test_quantisation_is_bit_equal_to_torch(shape, dtype):
    g = torch.Generator().manual_seed(shape[0] * 31 + shape[1])
    x = (torch.randn(*shape, generator=g) * torch.randn(shape[1], generator=g).mul(3).exp()).to(dtype)
    for fn, rows in ((fp8.quantize_rows, 1), (fp8.quantize_weight, 128)):
        q, s = plain_quantize(x.float(), rows)
        got = fn(x.cuda())
        assert got.values.stride(0) % 16 == 0
        assert torch.equal(got.scales.cpu(), s) and torch.equal(bits(got.values.cpu()), bits(q))


@gpu
def test_quantisation_of_blocks_of_zeros_tiny_values_and_non_finite_ones():
    x = torch.zeros(5, 384)
    x[1] = 1e-38
    x[2, 130] = math.inf
    x[2, 131] = 1.0
    x[3, 5] = math.nan
    x[4] = 3e38
    for dt in (F32, BF16):
        got = fp8.quantize_rows(x.cuda().to(dt))
        v, s = got.values.float().cpu(), got.scales.cpu()
        assert (v[:2] == 0).sum() >= 384 and torch.isfinite(s[:2]).all() and (s[:2] > 0).all()
        assert (v[1] == 0).all()  # 1e-38 is far below the floor's smallest step
        assert s[2, 1] == math.inf and torch.isnan(v[2, 130]) and v[2, 131] == 0 and s[2, 0] > 0
        assert torch.isnan(s[3, 0]) and torch.isnan(v[3, :128]).all() and (v[3, 128:] == 0).all()
        assert (v[4] == 448).all()
        for bad in (2, 3):  # and what such a block gives in a product is NaN, in its own row only
            w = fp8.quantize_weight(torch.ones(16, 384).cuda())
            y = fp8.matmul_fp8(got, w)
            assert torch.isnan(y[bad]).all() and torch.isfinite(y[0]).all()


@gpu
def test_quantisation_of_strided_and_nested_inputs():
    g = torch.Generator().manual_seed(4)
    base = torch.randn(6, 9, 600, generator=g).cuda()
    for x in (base[:, :, 7:320], base[:, ::2, :256], base.transpose(0, 1), base[..., ::3], base[2], base[0, 0], base.expand(2, 6, 9, 600),
              base[:0], base[..., :0]):
        got = fp8.quantize_rows(x)
        assert got.shape == x.shape and got.scales.shape == (*x.shape[:-1], -(-x.shape[-1] // 128))
        if x.numel():
            q, s = plain_quantize(x.reshape(-1, x.shape[-1]).cpu(), 1)
            assert torch.equal(got.scales.reshape(-1, s.shape[1]).cpu(), s)
            assert torch.equal(bits(got.values.reshape(-1, x.shape[-1]).cpu()), bits(q))
    assert torch.equal(fp8.quantize_weight(base[0].t()).scales.cpu(), plain_quantize(base[0].t().cpu(), 128)[1])


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16], ids=ids)
@pytest.mark.parametrize("K", [1, 7, 9, 130, 255])
@pytest.mark.parametrize("blocks", [False, True], ids=["rows", "weight"])
def test_quantisation_at_every_offset_leaves_the_neighbours_alone(K, blocks, dtype):
    """Sources and values that start at each element of a 16-byte word, NaN around the source, marks around the values."""
    rows, pitch = 131, K + 3
    g = torch.Generator().manual_seed(K)
    data = (torch.randn(rows, K, generator=g) * 3).to(dtype)
    q, s = plain_quantize(data.float(), 128 if blocks else 1)
    for off in range(8):
        room = torch.full((off + rows * pitch + 16,), math.nan, dtype=dtype, device="cuda")
        x = room[off:off + rows * pitch].view(rows, pitch)[:, :K]
        x.copy_(data)
        out = torch.full((off + rows * pitch + 16,), 0x55, dtype=torch.uint8, device="cuda")
        values = out[off:off + rows * pitch].view(rows, pitch)
        scales = torch.empty_like(s, device="cuda")
        _lib.quant_fp8(x, values[:, :K], scales, blocks)
        assert torch.equal(scales.cpu(), s) and torch.equal(values[:, :K].cpu(), q.view(torch.uint8))
        assert (out[:off] == 0x55).all() and (values[:, K:] == 0x55).all() and (out[off + rows * pitch:] == 0x55).all()


# ------------------------------------------------------------------------------------------------
# the product
# ------------------------------------------------------------------------------------------------
def operands(M, N, K, seed=0):
    g = torch.Generator().manual_seed(seed + M * 5 + N * 3 + K)
    x = fp8.quantize_rows((torch.randn(M, K, generator=g) * torch.randn(K, generator=g).exp()).cuda())
    w = fp8.quantize_weight((torch.randn(N, K, generator=g) * K ** -0.5).cuda())
    return x, w, torch.randn(N, generator=g)


def check_product(y, x, w, bias, name=""):
    K = x.shape[-1]
    xd, wd = wide(x.values.cpu(), x.scales.cpu(), 1), wide(w.values.cpu(), w.scales.cpu(), 128)
    ref, mag = xd @ wd.t(), xd.abs() @ wd.abs().t()
    if bias is not None:
        ref, mag = ref + bias.double(), mag + bias.double().abs()
    bound = (2 * 128 + 2 * (-(-K // 128)) + 8) * U * mag + half_step(y.dtype) * ref.abs() * (1 + 2 ** -8)
    off = (y.double().cpu() - ref).abs()
    if y.dtype == F16:
        bound = bound + 2.0 ** -25  # half of its smallest subnormal
    assert torch.isfinite(y).all() and (off <= bound).all(), \
        f"{name}: {(off > bound).sum()} of {off.numel()} off, worst {(off / bound).max():.3g} bounds"


# both sides of every tile boundary, rows for one to many tokens, short and long sums, odd sizes
PRODUCTS = [(1, 1, 1), (1, 16, 16), (1, 128, 128), (2, 130, 100), (7, 1000, 257), (16, 256, 1024), (17, 129, 640),
            (33, 512, 4096), (64, 1024, 384), (65, 300, 1100), (127, 128, 128), (128, 256, 512), (129, 257, 129),
            (200, 2500, 1100), (256, 256, 256), (257, 513, 130), (1000, 130, 48), (1537, 700, 260), (300, 8, 2000),
            (2100, 2500, 260), (129, 19001, 129), (9600, 514, 400), (4700, 1030, 16)]


@gpu
@pytest.mark.parametrize("shape", PRODUCTS, ids=str)
def test_product_matches_the_formula(shape):
    M, N, K = shape
    x, w, bias = operands(M, N, K)
    for dt, b in ((BF16, None), (F32, bias), (F16, bias.to(BF16)), (BF16, bias.to(F16))):
        y = fp8.matmul_fp8(x, w, None if b is None else b.cuda(), out_dtype=dt)
        check_product(y, x, w, b, f"{shape} {dt}")
    _lib.check_device_status(synchronize=True)


@gpu
def test_product_of_foreign_layouts_and_nested_rows():
    """Row-major scales, values on odd addresses and pitches, leading axes, empty extents."""
    x, w, bias = operands(24, 40, 300)
    y = fp8.matmul_fp8(x, w, out_dtype=F32)
    u8 = lambda t: t.view(torch.uint8)  # noqa: E731
    room = torch.zeros(24 * 301 + 5, dtype=torch.uint8, device="cuda")
    odd = room[5:].view(24, 301)[:, :300]
    odd.copy_(u8(x.values))
    assert torch.equal(fp8.matmul_fp8(fp8.Fp8Rows(odd.view(torch.float8_e4m3fn), x.scales.contiguous()), w, out_dtype=F32), y)
    wodd = torch.empty(300, 40, dtype=torch.uint8, device="cuda").t()
    wodd.copy_(u8(w.values))
    ws = w.scales.t().contiguous().t()
    assert torch.equal(fp8.matmul_fp8(x, fp8.Fp8Weight(wodd.view(torch.float8_e4m3fn), ws), out_dtype=F32), y)
    nested = fp8.Fp8Rows(x.values.unflatten(0, (2, 3, 4)), x.scales.unflatten(0, (2, 3, 4)))
    assert torch.equal(fp8.matmul_fp8(nested, w, out_dtype=F32), y.view(2, 3, 4, 40))
    one = fp8.Fp8Rows(x.values[3], x.scales[3])
    assert fp8.matmul_fp8(one, w, out_dtype=F32).shape == (40,)
    check_product(fp8.matmul_fp8(one, w, out_dtype=F32)[None], fp8.Fp8Rows(x.values[3:4], x.scales[3:4]), w, None)
    assert fp8.matmul_fp8(fp8.Fp8Rows(x.values[:0], x.scales[:0]), w).shape == (0, 40)
    none = fp8.quantize_rows(torch.zeros(3, 0, device="cuda"))
    y0 = fp8.matmul_fp8(none, fp8.quantize_weight(torch.zeros(40, 0, device="cuda")), bias.cuda(), out_dtype=F32)
    assert torch.equal(y0.cpu(), bias.expand(3, 40))
    with pytest.raises(ValueError, match="columns"):
        fp8.matmul_fp8(none, w)
    with pytest.raises(ValueError, match="bias"):
        fp8.matmul_fp8(x, w, bias[:-1].cuda())
    with pytest.raises(TypeError):
        fp8.matmul_fp8(x, w, out_dtype=torch.float64)
    with pytest.raises(RuntimeError, match="CUDA"):
        fp8.matmul_fp8(x, w, bias)


@gpu
def test_product_is_deterministic_and_leaves_its_neighbours_alone():
    """The same call twice gives the same bits, from any stream; rows are independent of the rows beside them."""
    for M, N, K in ((5, 1024, 4096), (100, 1024, 2048), (600, 384, 512)):
        x, w, _ = operands(M, N, K)
        a = fp8.matmul_fp8(x, w)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            b = fp8.matmul_fp8(x, w)
        side.synchronize()
        assert torch.equal(a, b)
        same = fp8.Fp8Rows(x.values.clone().contiguous(), x.scales.clone())
        u = same.values.view(torch.uint8)
        u[0] = 0x7F  # NaN in one row stays there
        y = fp8.matmul_fp8(same, w)
        assert torch.isnan(y[0]).all() and torch.equal(y[1:], a[1:])


@gpu
def test_product_of_more_rows_than_a_grid_has_in_one_direction():
    M, N, K = 8_400_000, 1, 16
    x = fp8.quantize_rows(torch.randn(M, K, device="cuda"))
    w = fp8.quantize_weight(torch.randn(N, K, device="cuda"))
    y = fp8.matmul_fp8(x, w, out_dtype=F32)
    at = torch.cat([torch.arange(0, M, 4099), torch.arange(M - 300, M)])
    part = fp8.Fp8Rows(x.values[at.cuda()], x.scales[at.cuda()])
    check_product(y[at.cuda()], part, w, None)
    assert torch.isfinite(y).all()


@gpu
def test_scales_shared_by_broadcasting():
    """One scale for a whole operand, expanded: strides of zero."""
    x, w, _ = operands(300, 520, 700)
    xs, ws = torch.full((1, 1), 0.25, device="cuda").expand(300, 6), torch.full((1, 1), 0.5, device="cuda").expand(5, 6)
    for rows in (3, 300):
        part = fp8.Fp8Rows(x.values[:rows], xs[:rows])
        check_product(fp8.matmul_fp8(part, fp8.Fp8Weight(w.values, ws), out_dtype=F32), part, fp8.Fp8Weight(w.values, ws), None)


# ------------------------------------------------------------------------------------------------
# residual norm
# ------------------------------------------------------------------------------------------------
TYPES = [(F32, F32), (BF16, BF16), (F16, F16), (BF16, F32), (F16, F32)]
NORMS = [(1, 1), (1, 1024), (3, 17), (5, 128), (33, 250), (9, 257), (4, 1000), (70, 1024), (2500, 64), (2400, 1000),
         (2400, 1023), (6, 2050), (3, 4096), (5, 8192), (2, 8200), (3, 10001), (2, 17000)]


@gpu
@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(map(ids, t)))
@pytest.mark.parametrize("shape", NORMS, ids=str)
def test_residual_norm_forward_and_8bit(shape, types):
    (rows, H), (xd, rd) = shape, types
    x, res, w, _ = norm_inputs(rows, H, xd, rd)
    ref, h, _ = plain_norm(x, res, w, 1e-5)
    rel = (H / 256 + 64) * U
    y, got_h = add_rms_norm(x.cuda(), res.cuda(), w.cuda())
    assert y.dtype == xd and got_h.dtype == rd and torch.equal(got_h.cpu(), h)
    tiny = 2.0 ** -25 if xd == F16 else 0.0
    assert ((y.double().cpu() - ref).abs() <= (half_step(xd) + rel) * (1 + 2 ** -8) * ref.abs() + tiny).all()
    q, got_h = add_rms_norm_fp8(x.cuda(), res.cuda(), w.cuda())
    assert torch.equal(got_h.cpu(), h) and q.values.stride(0) % 16 == 0
    pad = torch.nn.functional.pad(ref, (0, -H % 128)).view(rows, -1, 128)
    s = pad.abs().amax(-1).clamp_min(2.0 ** -100) / 448
    assert ((q.scales.double().cpu() - s).abs() <= (rel + 2 * U) * s).all()
    per = q.scales.double().cpu().repeat_interleave(128, 1)[:, :H]
    off = (q.values.float().double().cpu() * per - ref).abs()
    assert (off <= torch.maximum(2.0 ** -4 * ref.abs(), 2.0 ** -10 * per) * (1 + 2 ** -8) + rel * ref.abs()).all()


@gpu
@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(map(ids, t)))
@pytest.mark.parametrize("shape", NORMS, ids=str)
def test_residual_norm_backward(shape, types):
    (rows, H), (xd, rd) = shape, types
    x, res, w, g = norm_inputs(rows, H, xd, rd)
    dy, dh = torch.randn(rows, H, generator=g).to(xd), torch.randn(rows, H, generator=g).to(rd)
    _, h, r = plain_norm(x, res, w, 1e-5)
    hd, gw = h.double(), dy.double() * w.double()
    k = r ** 3 * (hd * gw).mean(-1, keepdim=True)
    ref = dh.double() + r * gw - hd * k
    mag = dh.double().abs() + r * gw.abs() + hd.abs() * r ** 3 * (hd * gw).abs().mean(-1, keepdim=True)
    c = (H / 256 + 64 + 3 * (H / 512 + 32)) * U
    dw, dw_mag = (dy.double() * hd * r).sum(0), (dy.double() * hd * r).abs().sum(0)
    for use_dh in (True, False):
        leaves = [t.cuda().requires_grad_() for t in (x, res, w)]
        y, got_h = add_rms_norm(*leaves)
        torch.autograd.backward((y, got_h) if use_dh else (y,), (dy.cuda(), dh.cuda()) if use_dh else (dy.cuda(),))
        want, m = (ref, mag) if use_dh else (ref - dh.double(), mag - dh.double().abs())
        for leaf, dt in ((leaves[0], xd), (leaves[1], rd)):
            off = (leaf.grad.double().cpu() - want).abs()
            tiny = 2.0 ** -25 if dt == F16 else 0.0
            assert leaf.grad.dtype == dt and (off <= half_step(dt) * (1 + 2 ** -8) * want.abs() + c * m + tiny).all()
        assert ((leaves[2].grad.double().cpu() - dw).abs() <= (rows + H / 256 + 96) * U * dw_mag + 1e-30).all()


@gpu
@pytest.mark.parametrize("types", [(F32, F32), (BF16, BF16), (BF16, F32)], ids=lambda t: "-".join(map(ids, t)))
@pytest.mark.parametrize("shape", [(1300, 8200), (900, 10001), (700, 20480)], ids=str)
def test_weight_gradient_of_long_rows_over_many_rows_per_cta(shape, types):
    """Rows too long for registers, more of them than CTAs: the sums of dw that a CTA keeps in shared memory or scratch."""
    (rows, H), (xd, rd) = shape, types
    x, res, w, g = norm_inputs(rows, H, xd, rd)
    dy = torch.randn(rows, H, generator=g).to(xd)
    _, h, r = plain_norm(x, res, w, 1e-5)
    terms = dy.double() * h.double() * r
    dw, dw_mag = terms.sum(0), terms.abs().sum(0)
    leaves = [t.cuda().requires_grad_() for t in (x, res, w)]
    for _ in range(2):
        grad, = torch.autograd.grad(add_rms_norm(*leaves)[0], leaves[2], dy.cuda())
        assert ((grad.double().cpu() - dw).abs() <= (rows + H / 256 + 96) * U * dw_mag + 1e-30).all()


@gpu
def test_residual_norm_gradient_against_differences():
    """The kernel's gradient against differences of the 64-bit formula, with shared and broadcast inputs: one residual
    row for all, and x used as its own residual."""
    g = torch.Generator().manual_seed(8)
    x, res, w, dy, dh = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((6, 40), (1, 40), (40,), (6, 40), (6, 40)))

    def loss(x, res, w):
        h = x + res.expand(6, 40)
        y = h / torch.sqrt(h.square().mean(-1, keepdim=True) + 1e-5) * w
        return (y * dy).sum() + (h * dh).sum()

    leaves = [t.float().cuda().requires_grad_() for t in (x, res, w)]
    x, res, w = (t.float().double() for t in (x, res, w))
    y, h = add_rms_norm(leaves[0], leaves[1].expand(6, 40), leaves[2])
    torch.autograd.backward((y, h), (dy.float().cuda(), dh.float().cuda()))
    step = 1e-5
    for n, (leaf, at) in enumerate(((leaves[0], (2, 5)), (leaves[1], (0, 17)), (leaves[2], (39,)))):
        v = [x.clone(), res.clone(), w.clone()]
        v[n][at] += step
        up = loss(*v)
        v[n][at] -= 2 * step
        num = (up - loss(*v)) / (2 * step)
        # central differences are good to step^2, the fp32 gradient to a few u of sums of about ten
        assert abs(leaf.grad.double().cpu()[at] - num) <= 1e-5 * max(1.0, abs(num))
    a = torch.randn(4, 64, device="cuda", requires_grad=True)
    one = torch.ones(64, device="cuda")
    y, h = add_rms_norm(a, a, one)
    h.sum().backward()
    assert torch.equal(a.grad, torch.full_like(a, 2.0))  # y unused: h's gradient alone, to both


@gpu
@pytest.mark.parametrize("wd", [BF16, F16], ids=ids)
def test_residual_norm_weight_types_and_partial_gradients(wd):
    x, res, w, g = norm_inputs(40, 300, BF16, F32)
    w = w.to(wd)
    ref, _, r = plain_norm(x, res, w, 1e-5)
    y, _ = add_rms_norm(x.cuda(), res.cuda(), w.cuda())
    assert ((y.double().cpu() - ref).abs() <= (half_step(BF16) + 66 * U) * (1 + 2 ** -8) * ref.abs()).all()
    dy = torch.randn(40, 300, generator=g).to(BF16)
    full = [t.cuda().requires_grad_() for t in (x, res, w)]
    add_rms_norm(*full)[0].backward(dy.cuda())
    assert full[2].grad.dtype == wd
    for keep in range(3):  # only one input needs its gradient: the same values
        part = [t.cuda().requires_grad_(i == keep) for i, t in enumerate((x, res, w))]
        add_rms_norm(*part)[0].backward(dy.cuda())
        assert torch.equal(part[keep].grad, full[keep].grad)
        assert all(p.grad is None for i, p in enumerate(part) if i != keep)


@gpu
def test_residual_norm_layouts_streams_and_refusals():
    g = torch.Generator().manual_seed(2)
    base = torch.randn(5, 8, 700, generator=g).cuda()
    w = (1 + torch.rand(300, generator=g)).cuda()
    views = [(base[..., 1:301], base[..., 400:700]), (base[:, ::2, :300], base[:, 1::2, 3:303]),
             (base[0, 0, :300], base[1, 1, :300]), (base[:0, :, :300], base[:0, :, 300:600]),
             (base[..., :300], base[:1, :1, :300].expand(5, 8, 300)), (base[..., 0:600:2], base[..., 1:601:2])]
    for x, res in views:
        y, h = add_rms_norm(x, res, w)
        q, h8 = add_rms_norm_fp8(x, res, w)
        assert y.shape == x.shape and q.shape == x.shape and torch.equal(h, x + res) and torch.equal(h8, h)
        if x.numel():  # rows of another alignment are summed in another order: the bound, not the bits
            ref, _, _ = plain_norm(x.reshape(-1, 300).cpu(), res.reshape(-1, 300).cpu(), w.cpu(), 1e-5)
            rel = (300 / 256 + 64) * U
            assert ((y.reshape(-1, 300).double().cpu() - ref).abs() <= (half_step(F32) + rel) * (1 + 2 ** -8) * ref.abs()).all()
            deq = q.dequantize().reshape(-1, 300).double().cpu()
            per = q.scales.reshape(-1, 3).double().cpu().repeat_interleave(128, 1)[:, :300]
            assert ((deq - ref).abs() <= torch.maximum(2.0 ** -4 * ref.abs(), 2.0 ** -10 * per) * (1 + 2 ** -8) + rel * ref.abs()).all()
    q, h = add_rms_norm_fp8(base, None, torch.ones(700, device="cuda"))
    assert h is base
    x = base[..., :300]
    with pytest.raises(ValueError):
        add_rms_norm(x, x[:1], w)
    with pytest.raises(ValueError):
        add_rms_norm(x, None, w)
    with pytest.raises(ValueError):
        add_rms_norm(x, x, w[:-1])
    with pytest.raises(TypeError):
        add_rms_norm(x, x.half(), w)
    with pytest.raises(TypeError):
        add_rms_norm(x.double(), x.double(), w)
    with pytest.raises(RuntimeError):
        add_rms_norm(x, x, w.cpu())
    y, h = add_rms_norm(x.clone().requires_grad_(), x, w)
    h.add_(1)  # the backward needs h as it was
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()


@gpu
def test_residual_norm_of_nothing_and_gradients_of_one_output():
    w = torch.rand(8, device="cuda", requires_grad=True)
    for shape, wt in (((0, 8), w), ((3, 0), torch.rand(0, device="cuda", requires_grad=True))):
        x, r = (torch.zeros(shape, device="cuda", requires_grad=True) for _ in range(2))
        y, h = add_rms_norm(x, r, wt)
        (y.sum() + h.sum()).backward()
        assert y.shape == h.shape == x.grad.shape == r.grad.shape == shape and (wt.grad == 0).all()
    x = torch.randn(4, 8, device="cuda").to(BF16).requires_grad_()
    r = torch.randn(4, 8, device="cuda", requires_grad=True)
    y, h = add_rms_norm(x, r, w)
    h.sum().backward()  # only the sum was used: ones to both, each in its own type
    assert x.grad.dtype == BF16 and r.grad.dtype == F32 and (x.grad == 1).all() and (r.grad == 1).all()
    y, h = add_rms_norm(x, r, w)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(y.float().sum(), r, create_graph=True)
    with torch.no_grad():
        y, h = add_rms_norm(x, r, w)
    assert not y.requires_grad and not h.requires_grad


@gpu
def test_calls_on_two_streams_at_once():
    """Products of both kernels, norms and quantisation on two streams without an order between them."""
    jobs = []
    for M, N, K in ((3000, 2000, 700), (9, 3000, 2000)):
        x, w, _ = operands(M, N, K)
        src, res, one = torch.randn(M, K, device="cuda"), torch.randn(M, K, device="cuda"), torch.ones(K, device="cuda")

        def job(x=x, w=w, src=src, res=res, one=one):
            q, h = add_rms_norm_fp8(src, res, one)
            return fp8.matmul_fp8(x, w), fp8.matmul_fp8(q, w), h, fp8.quantize_rows(src).values.view(torch.uint8)

        jobs.append((job, job()))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(jobs[i][0]())
    torch.cuda.synchronize()
    for (_, want), results in zip(jobs, got):
        assert all(torch.equal(a, b) for r in results for a, b in zip(r, want))
    _lib.check_device_status(synchronize=True)


@gpu
def test_non_finite_rows_stay_in_their_rows():
    x, res, w, _ = norm_inputs(6, 512, BF16, BF16)
    x[1, 7], x[4, 100] = math.nan, math.inf
    y, _ = add_rms_norm(x.cuda(), res.cuda(), w.cuda())
    q, _ = add_rms_norm_fp8(x.cuda(), res.cuda(), w.cuda())
    ok = [0, 2, 3, 5]
    assert torch.isfinite(y[ok]).all() and torch.isnan(y[1]).all() and torch.isnan(y[4, 100])
    assert torch.isfinite(q.scales[ok]).all() and torch.isnan(q.scales[1]).all() and torch.isnan(q.scales[4, 0])
