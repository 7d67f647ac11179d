"""Edges of the residual norm and the 8-bit serving path: strides of axes of one, widths of types, sources at the end of
their memory, weights that move between devices.  Bounds as derived in ``test_fp8.py``."""
import copy
import glob
import os
import re
import subprocess

import pytest
import torch

from quick_ssm_b200 import _lib, fp8
from quick_ssm_b200.layers import SSM, SSMFp8, SSMFused, SSMStack, SSMStackFp8
from quick_ssm_b200.norm import _room_like, add_rms_norm, add_rms_norm_fp8
from quick_ssm_b200.streaming import ScanState, scan_chunk

from test_fp8 import BF16, F16, F32, U, check_product, gpu, half_step, ids, operands, plain_norm
from test_fp8_layers import blocks, plain_block, rel


@pytest.mark.parametrize("shape,order", [((1, 8), (1, 0)), ((1, 1, 8), (2, 0, 1)), ((3, 1), (1, 0)), ((1, 5, 8), (1, 0, 2))], ids=str)
def test_outputs_lie_row_by_row_whatever_the_strides_of_axes_of_one(shape, order):
    """One token out of a transposed product has strides (1, 1): its outputs must not."""
    t = torch.zeros([shape[i] for i in order]).permute([order.index(i) for i in range(len(shape))])
    assert t.shape == shape
    for dt in (F32, BF16):
        room = _room_like(t, dt)
        assert room.shape == shape and room.dtype == dt and room.stride() == torch.empty(shape).stride()


@gpu
@pytest.mark.parametrize("rd", [BF16, F32], ids=ids)
@pytest.mark.parametrize("H", [8, 1024], ids=str)
def test_one_token_out_of_a_transposed_product(H, rd):
    """x, residual or both as a column transposed ([1, H] with strides (1, 1)): the results of the ordinary layout, whose
    order of sums they need not share (the bounds of the tests above)."""
    g = torch.Generator().manual_seed(H)
    x, res, dy, dh = (torch.randn(1, H, generator=g).to(dt).cuda() for dt in (BF16, rd, BF16, rd))
    w = (1 + torch.rand(H, generator=g)).cuda()
    turned = lambda t: torch.empty(H, 1, dtype=t.dtype, device="cuda").copy_(t.t()).t()  # noqa: E731
    assert turned(x).stride() == (1, 1)
    ref, _, r = plain_norm(x.cpu(), res.cpu(), w.cpu(), 1e-5)
    lim = (half_step(BF16) + (H / 256 + 64) * U) * (1 + 2 ** -8) * ref.abs()
    hd, gw = (x.float() + res.float()).to(rd).double().cpu(), dy.double().cpu() * w.double().cpu()
    d = dh.double().cpu() + r * gw - hd * r ** 3 * (hd * gw).mean(-1, keepdim=True)
    mag = dh.double().abs().cpu() + r * gw.abs() + hd.abs() * r ** 3 * (hd * gw).abs().mean(-1, keepdim=True)
    c = (H / 256 + 64 + 3 * (H / 512 + 32)) * U
    for a, b in ((turned(x), res), (x, turned(res)), (turned(x), turned(res)), (turned(x)[None], turned(res)[None])):
        a, b = a.detach().requires_grad_(), b.detach().requires_grad_()
        y, h = add_rms_norm(a, b, w)
        torch.autograd.backward((y, h), (turned(dy).view_as(y), turned(dh).view_as(h)))
        assert y.shape == a.shape and torch.equal(h.detach().view(1, H), (x.float() + res.float()).to(rd))
        assert ((y.detach().view(1, H).double().cpu() - ref).abs() <= lim).all()
        for leaf in (a, b):
            assert ((leaf.grad.view(1, H).double().cpu() - d).abs() <= half_step(leaf.dtype) * (1 + 2 ** -8) * d.abs() + c * mag).all()
        q, h8 = add_rms_norm_fp8(a.detach(), b.detach(), w)
        assert q.shape == a.shape and torch.equal(h8, h.detach())
        per = q.scales.view(1, -1).double().cpu().repeat_interleave(128, 1)[:, :H]
        off = (q.dequantize().view(1, H).double().cpu() - ref).abs()
        assert (off <= torch.maximum(2.0 ** -4 * ref.abs(), 2.0 ** -10 * per) * (1 + 2 ** -8) + (H / 256 + 64) * U * ref.abs()).all()


@gpu
@pytest.mark.parametrize("what", ["plain", "branch", "factors", "scan"])
def test_serving_a_block_of_float16_gates_keeps_the_range_of_its_weights(what):
    """The default compute type over fp32 weights: finite block outputs beyond 65504, a gate whose one factor is beyond it,
    and a scan output beyond it.  The bound is that of the bf16 block in ``test_fp8_layers``: what is rounded to bf16 there
    is rounded to fp16 or not at all here."""
    block = blocks(1, 64, 2.0, compute=F16)[0]
    with torch.no_grad():
        if what == "branch":
            block.out_proj.weight.mul_(1e6)
        elif what == "factors":
            block.C_proj_a.weight.mul_(1e6)
            block.C_proj_b.weight.mul_(1e-6)
        elif what == "scan":
            block.B_proj.weight.mul_(1e4)
            block.C_proj_a.weight.mul_(300)
    served = SSMFp8(block)
    torch.manual_seed(11)
    x, r = torch.randn(3, 20, 64), torch.randn(3, 20, 64).mul(2)
    out, h, state = served(x.cuda(), r.cuda())
    want, want_h, want_s = plain_block(served, x, r, torch.zeros(3, 128, dtype=torch.float64))
    if what == "branch":
        assert want.abs().max() > 65504
    assert served.gate_dtype == F16 and out.dtype == F32 and torch.equal(h.double().cpu(), want_h)
    assert rel(out, want) < 0.03 and rel(state.h, want_s) < 0.03
    y, _ = SSMStackFp8([block, block])(x.cuda().to(BF16))
    assert y.dtype == BF16 and torch.isfinite(y).all()
    _lib.check_device_status(synchronize=True)


@gpu
@pytest.mark.parametrize("xd", [F32, BF16, F16], ids=ids)
@pytest.mark.parametrize("compute", [BF16, F16], ids=ids)
def test_serving_blocks_chained_by_hand(compute, xd):
    """Block after block with the residual stream apart, whatever its type: the stack's result."""
    made = blocks(3, 64, 2.0, compute=compute)
    x = torch.randn(2, 9, 64, device="cuda").to(xd)
    want, _ = SSMStackFp8(made)(x)
    y, h = x, None
    for block in made:
        y, h, _ = SSMFp8(block)(y, h)
    assert want.dtype == xd and torch.equal((h + y).to(xd), want)


@gpu
def test_serving_types_follow_the_block():
    for weights, compute, gate, want in ((F32, F16, None, (F16, F32)), (F32, BF16, None, (BF16, BF16)), (F32, F32, None, (BF16, BF16)),
                                         (F16, F16, None, (F16, F16)), (BF16, F16, None, (F16, F32)), (F32, F16, BF16, (BF16, BF16)),
                                         (F32, BF16, F16, (F16, F32))):
        served = SSMFp8(SSM(32, dtype=weights, compute_dtype=compute).cuda(), gate)
        x = torch.randn(2, 5, 32, device="cuda").to(weights)
        out, _, _ = served(x)
        assert (served.gate_dtype, served.act_dtype) == want and out.dtype == want[1] and torch.isfinite(out).all()
    with pytest.raises(TypeError, match="gates"):
        SSMFp8(SSM(32).cuda(), F32)


# ------------------------------------------------------------------------------------------------
# types and arguments of the training blocks
# ------------------------------------------------------------------------------------------------
F64 = torch.float64


@gpu
@pytest.mark.parametrize("weights,xd", [(F32, F32), (F32, BF16), (F32, F16), (F64, F64), (F64, F32), (F64, BF16)], ids=ids)
def test_stack_takes_the_types_that_its_blocks_take(weights, xd):
    """Without autocast the plain blocks promote x to the weights' type.  The fused blocks and the stack do as well: the result
    and the gradients of the plain blocks on x promoted beforehand, 1e-5 of the largest value per block and direction
    (the order of fp32 sums).  x's gradient comes from two uses of x, the residual and the norm: autograd rounds each to x's
    type and then their sum, three half steps of three magnitudes."""
    seq = torch.nn.Sequential(*(SSM(64, 2.0, dtype=weights, compute_dtype=F32) for _ in range(3))).cuda()
    fused = torch.nn.Sequential(*(SSMFused(64, 2.0, dtype=weights, compute_dtype=F32) for _ in range(3))).cuda()
    stack = SSMStack(3, 64, 2.0, dtype=weights, compute_dtype=F32).cuda()
    fused.load_state_dict(seq.state_dict())
    stack.load_state_dict({f"layers.{k}": v for k, v in seq.state_dict().items()})
    x = torch.randn(2, 9, 64, device="cuda").to(xd)
    dy = torch.randn(2, 9, 64, device="cuda").to(weights)
    x0 = x.clone().to(weights).requires_grad_()
    first = seq[0](x0)
    first.retain_grad()  # what the residual passes on
    want = seq[2](seq[1](first))
    want.backward(dy)
    skip, total = first.grad.double(), x0.grad.double()
    rounded = half_step(xd) * (1 + 2 ** -8) * (skip.abs() + (total - skip).abs() + total.abs())
    assert seq(x).dtype == want.dtype
    lim = lambda w: 6e-5 * w.abs().max()  # noqa: E731
    for model, layers in ((fused, fused), (stack, stack.layers)):
        xi = x.clone().requires_grad_()
        got = model(xi)
        got.backward(dy)
        assert got.dtype == want.dtype and (got - want).abs().max() <= lim(want)
        assert xi.grad.dtype == xd
        assert ((xi.grad.double() - total).abs() <= lim(total) + rounded).all()
        for p, q in zip(layers.parameters(), seq.parameters()):
            assert (p.grad - q.grad).abs().max() <= lim(q.grad)
    _lib.check_device_status(synchronize=True)


@gpu
def test_norm_weights_in_float32_beside_16_bit_projections():
    """What the fused blocks take and the plain ones do not: the norm on x as it is."""
    fused, stack = SSMFused(64, dtype=BF16, compute_dtype=BF16).cuda(), SSMStack(2, 64, dtype=BF16, compute_dtype=BF16).cuda()
    x = torch.randn(2, 9, 64, device="cuda").to(BF16)
    same = stack(x), fused(x)
    for layer in (fused, *stack.layers):
        layer.pre_norm.float()  # ones either way
    for got, want in zip((stack(x), fused(x)), same):
        assert got.dtype == BF16 and torch.equal(got, want)


@gpu
def test_stack_takes_the_arguments_that_its_blocks_take():
    stack = SSMStack(2, 32, compute_dtype=F32).cuda()
    x = torch.randn(2, 40, 32, device="cuda")
    want = stack(x)
    for kw in (dict(block_l=16, tile_b=1, tile_d=8), dict(checkpoint=False), dict(backend="torch"), dict(scan_out_dtype=F32)):
        seq = x
        for layer in stack.layers:
            seq = layer(seq, **kw)
        got = stack(x, **kw)
        # fp32 sums in another order, as above
        assert (got - seq).abs().max() <= 4e-5 * seq.abs().max() and (got - want).abs().max() <= 4e-5 * want.abs().max()


@gpu
@pytest.mark.parametrize("L", [1, 40])
def test_scan_continues_from_a_state_in_any_layout(L):
    a, x, b, c = (torch.rand(5, L, 24, device="cuda") for _ in range(4))
    h = torch.randn(5, 24, device="cuda")
    y, end = scan_chunk(x, a, b, c, ScanState(h))
    wide = torch.randn(5, 48, device="cuda")
    wide[:, ::2] = h
    for other in (h.t().contiguous().t(), wide[:, ::2], h[:1].expand(5, 24)):
        want, want_end = (y, end) if torch.equal(other, h) else scan_chunk(x, a, b, c, ScanState(other.clone()))
        got, got_end = scan_chunk(x, a, b, c, ScanState(other))
        assert torch.equal(got, want) and torch.equal(got_end.h, want_end.h)


# ------------------------------------------------------------------------------------------------
# weights that move
# ------------------------------------------------------------------------------------------------
def spaced(block):
    return all(getattr(block, k).stride(0) % 16 == 0 and getattr(block, k).stride(1) == 1 for k in ("in_values", "out_values"))


def test_serving_weights_keep_their_spacing_without_a_gpu():
    """A tensor with gaps between its rows loses them in a move; the block puts them back."""
    block = SSMFp8.__new__(SSMFp8)
    torch.nn.Module.__init__(block)
    for name, (n, k) in (("in", (200, 40)), ("out", (40, 44))):
        values = fp8._values_like(n, k, "cpu")
        values.view(torch.uint8).copy_(torch.randint(0, 120, (n, k), dtype=torch.uint8))
        block._keep(name, fp8.Fp8Weight(values, torch.rand(fp8.n_blocks(n), fp8.n_blocks(k))), torch.rand(n))
    assert spaced(block)
    before = {k: v.clone() for k, v in block.state_dict().items()}
    assert before["in_values"].stride(0) == 40
    at = block.in_values.data_ptr()
    block.load_state_dict(before)
    assert block.in_values.data_ptr() == at  # in place: a captured step still reads it
    stack = torch.nn.Sequential(block)
    for move in (lambda: stack._apply(lambda t: t.clone()), lambda: block.load_state_dict(before, assign=True)):
        move()
        assert spaced(block) and set(block.state_dict()) == set(before)
        assert all(torch.equal(v, before[k]) for k, v in block.state_dict().items())


@gpu
def test_serving_weights_keep_their_spacing():
    made = blocks(1, 72, 1.5)
    x = torch.randn(2, 6, 72, device="cuda")
    first = SSMFp8(made[0])
    want = first(x)[0]
    dense = {k: v.clone() for k, v in first.state_dict().items()}
    moved, loaded = SSMFp8(made[0]).cpu().cuda(), SSMFp8(made[0])
    loaded.load_state_dict(dense, assign=True)
    for block in (first, moved, loaded, copy.deepcopy(first), copy.deepcopy(moved)):
        assert spaced(block)
        at = block.in_values.data_ptr()
        assert torch.equal(block(x)[0], want) and block.in_values.data_ptr() == at
        assert fp8.copyable(block.in_values)[0] is block.in_values


# ------------------------------------------------------------------------------------------------
# sources at the end of their memory
# ------------------------------------------------------------------------------------------------
HOST_SIDE = r"""
#include <stdint.h>
#include <stdio.h>
#include <string.h>
#define __device__
#define __forceinline__ inline
static uintptr_t from, upto;
static long outside = 0;
static void seen(const void* p, size_t n) { if ((uintptr_t)p < from || (uintptr_t)p + n > upto) ++outside; }
struct uint4 {  // what is read is read through its copies
    uint32_t x, y, z, w;
    uint4() : x(0), y(0), z(0), w(0) {}
    uint4(const uint4& o) { seen(&o, 16); memcpy(this, &o, 16); }
    uint4& operator=(const uint4& o) { seen(&o, 16); memcpy(this, &o, 16); return *this; }
};
static uint32_t __funnelshift_r(uint32_t lo, uint32_t hi, uint32_t by) { return (uint32_t)((((uint64_t)hi << 32) | lo) >> (by & 31)); }
%s
int main() {
    alignas(16) static uint16_t room[8192];
    long wrong = 0, by_words = 0, by_each = 0;
    for (int off = 0; off < 8; ++off)
        for (int rows = 1; rows < 140; rows += rows < 4 ? 1 : 126)
            for (int K = 1; K < 300; K += K < 20 ? 1 : 13)
                for (int gap = -1; gap < 4; ++gap) {
                    const long long stride = gap < 0 ? 0 : K + gap, all = (rows - 1) * stride + K;
                    if (off + all + 64 > 8192) continue;
                    for (int i = 0; i < 8192; ++i) room[i] = (uint16_t)(i * 7 + 1);
                    const uint16_t* x = room + 32 + off;
                    from = (uintptr_t)x; upto = (uintptr_t)(x + all);
                    for (long long top = 0; top < rows; top += 128)
                        for (int col0 = 0; col0 < K; col0 += 128) {  // as the kernel's blocks of 128 x 128
                            const int cols = K - col0 < 128 ? K - col0 : 128;
                            const long long bottom = top + 128 < rows ? top + 128 : rows;
                            const bool words = words_inside(top * stride + col0, (bottom - 1) * stride + col0 + cols, all);
                            ++(words ? by_words : by_each);
                            for (long long row = top; row < bottom; ++row)
                                for (int l = 0; l < 16; ++l) {
                                    uint16_t out[8];
                                    const uint16_t* at = x + row * stride + col0 + 8 * l;
                                    if (words) load_any8<uint16_t>(at, cols - 8 * l, out);
                                    else load_each8<uint16_t>(at, cols - 8 * l, out);
                                    for (int i = 0; i < 8; ++i) wrong += out[i] != (8 * l + i < cols ? at[i] : 0);
                                }
                        }
                }
    printf("%%ld %%ld %%d", wrong, outside, by_words > 100 && by_each > 100);
}
"""


def test_reads_of_sources_on_any_boundary_stay_in_the_source(tmp_path):
    """The device functions, compiled for the host, over blocks of sources at every offset in a word: right elements, and no
    16-byte word that reaches over the source's first or last element."""
    with open(os.path.join(os.path.dirname(_lib.LIB_PATH), "csrc", "qssm_elem.cuh")) as f:
        text = f.read()
    functions = text[text.index("template <typename T> __device__ __forceinline__ void load_any8"):text.index("__device__ __forceinline__ float sum_warp(")]
    src, exe = tmp_path / "any8.cpp", tmp_path / "any8"
    src.write_text(HOST_SIDE % functions)
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-fno-strict-aliasing", "-o", str(exe), str(src)])
    assert subprocess.check_output([str(exe)], text=True).split() == ["0", "0", "1"]


# ------------------------------------------------------------------------------------------------
# barriers
# ------------------------------------------------------------------------------------------------
def barriers_without_a_whole_warp(pattern):
    """Lines of inline PTX that match and have no ``__syncwarp();`` in the two lines in front of them."""
    found, loose = 0, []
    for path in sorted(glob.glob(os.path.join(os.path.dirname(_lib.LIB_PATH), "csrc", "*.cu*"))):
        with open(path) as f:
            lines = f.read().splitlines()
        for i, line in enumerate(lines):
            if "asm" in line and re.search(pattern, line):
                found += 1
                if not any("__syncwarp();" in before for before in lines[max(0, i - 2):i]):
                    loose.append(f"{os.path.basename(path)}:{i + 1}")
    return found, loose


def test_cluster_barriers_find_the_warp_whole():
    """The aligned forms are undefined where only some lanes of a warp arrive together, and lanes that left a branch need
    not be together again: sums are joined by the lanes whose column exists, and the barrier behind them keeps those sums alive."""
    found, loose = barriers_without_a_whole_warp(r"barrier\.cluster\.arrive")
    assert found == 1 and not loose


def test_named_barriers_find_the_warp_whole():
    """The same for the barrier of the warps that share a row, behind the store of one lane."""
    found, loose = barriers_without_a_whole_warp(r'"bar\.sync')
    assert found == 1 and not loose


def test_tensor_memory_loads_find_the_warp_whole():
    """Between a branch of one lane and the next aligned load of a product's kernels the warp is put together: from such a
    branch on, the first of ``__syncwarp``, ``__all_sync`` and ``tmem_ld`` (around the loop as well) is no load."""
    with open(os.path.join(os.path.dirname(_lib.LIB_PATH), "csrc", "qssm_fp8mm.cuh")) as f:
        text = f.read()
    loops = [text[text.index("for (int t = pair; ok && t < tiles; t += pairs, ++turn) {\n            const int m0 = (t % p.m_tiles) * MMR_M + (int)rank * 128 + quarter"):text.index("if (lane == 0) tma_wait_all();")],
             text[text.index("for (int j = 0; j < C::ROWS / 2; ++j) acc[j] = make_float2(0.f, 0.f);"):text.index("if (!ok && lane == 0 && p.status", text.index("matmul_fp8_few_kernel"))]]
    for loop in loops:
        marks = re.findall(r"if \(lane == 0|__syncwarp\(\)|__all_sync\(|tmem_ld<", loop)
        assert "tmem_ld<" in marks and "if (lane == 0" in marks
        for i, m in enumerate(marks):
            if m == "if (lane == 0":
                after = next(n for n in marks[i + 1:] + marks if n != "if (lane == 0")
                assert after != "tmem_ld<", loop[:60]


@gpu
@pytest.mark.parametrize("shape", [(1, 1001, 4096), (16, 333, 8192), (40, 97, 4096), (64, 1005, 4096), (100, 300, 16384)], ids=str)
def test_products_joined_over_a_cluster_with_columns_that_end_inside_a_warp(shape):
    """k cut over clusters, N no multiple of 32, launches close behind each other: every one the same, and the formula's."""
    x, w, bias = operands(*shape)
    ys = [fp8.matmul_fp8(x, w, bias.cuda(), out_dtype=F32) for _ in range(40)]
    check_product(ys[0], x, w, bias, str(shape))
    assert all(torch.equal(y, ys[0]) for y in ys)
    _lib.check_device_status(synchronize=True)


# ------------------------------------------------------------------------------------------------
# calls of other kinds
# ------------------------------------------------------------------------------------------------
@gpu
def test_offsets_beyond_32_bits():
    """More than 2^31 elements in a source, an output and a gradient: rows at both ends and around 2^31 against the formulas,
    quantised ones against calls on those rows alone."""
    rows, H = 2_150_000, 1024
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.empty(rows, H, dtype=BF16, device="cuda").normal_(generator=g)
    w = torch.rand(H, device="cuda", generator=g) + 0.5
    at = [0, 1, rows // 2, 2 ** 21 - 1, 2 ** 21, 2 ** 21 + 1, rows - 2, rows - 1]
    few = x[at].contiguous()
    y, h = add_rms_norm(x, x, w)
    # few rows take more warps each, whose sums are joined in another order: the bound of the norm's tests
    ref, want_h, r = plain_norm(few.cpu(), few.cpu(), w.cpu(), 1e-5)
    assert torch.equal(h[at].cpu(), want_h)
    assert ((y[at].double().cpu() - ref).abs() <= (half_step(BF16) + (H / 256 + 64) * U) * (1 + 2 ** -8) * ref.abs()).all()
    rstd = r.float().reshape(-1).cuda()
    full = torch.ones(rows, device="cuda")
    full[at] = rstd
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    _lib.add_rmsnorm_bwd(h, w, x, None, full, dx, None, dw)
    hd, gw = want_h.double(), few.double().cpu() * w.double().cpu()
    rd = rstd.double().cpu()[:, None]
    d = rd * gw - hd * rd ** 3 * (hd * gw).mean(-1, keepdim=True)
    mag = rd * gw.abs() + hd.abs() * rd ** 3 * (hd * gw).abs().mean(-1, keepdim=True)
    c = (H / 256 + 64 + 3 * (H / 512 + 32)) * U
    assert ((dx[at].double().cpu() - d).abs() <= half_step(BF16) * (1 + 2 ** -8) * d.abs() + c * mag).all()
    del y, h, dx, full
    q, small = fp8.quantize_rows(x), fp8.quantize_rows(few)
    assert torch.equal(q.values[at].view(torch.uint8), small.values.view(torch.uint8)) and torch.equal(q.scales[at], small.scales)
    del q
    wide_w = fp8.quantize_weight(x)
    band = fp8.quantize_weight(x[128 * 16700:128 * 16700 + 256].clone())
    assert torch.equal(wide_w.values[128 * 16700:128 * 16700 + 256].view(torch.uint8), band.values.view(torch.uint8))
    assert torch.equal(wide_w.scales[16700:16702], band.scales)
    del wide_w, x
    M, N, K = 110_000, 20_000, 64
    a, b, _ = operands(M, N, K)
    out = fp8.matmul_fp8(a, b)
    tail = [0, M - 300, M - 1]
    part = fp8.Fp8Rows(a.values[tail], a.scales[tail])
    check_product(out[tail], part, b, None)
    _lib.check_device_status(synchronize=True)


@gpu
def test_inference_mode_and_empty_batches():
    stack = SSMStack(2, 64, 2.0, compute_dtype=BF16).cuda()
    x = torch.randn(2, 7, 64, device="cuda")
    want = stack(x)
    served = SSMStackFp8(stack)
    y, states = served(x)
    with torch.inference_mode():
        assert torch.equal(stack(x), want)
        y2, states2 = served(x)
        assert torch.equal(y2, y) and all(torch.equal(a.h, b.h) for a, b in zip(states, states2))
        served(x[:, :1], states2)
    for model in (stack, lambda t: served(t)[0]):
        assert model(x[:0]).shape == (0, 7, 64) and model(x[:, :0]).shape == (2, 0, 64)
    _, none = served(x[:0])
    assert all(s.h.shape == (0, 128) for s in none)


@gpu
def test_calls_from_several_host_threads():
    """Streams and threads of their own, more operands than the maps that a thread keeps."""
    import concurrent.futures
    torch.manual_seed(3)
    stack = SSMStackFp8(blocks(2, 96, 1.5))
    inputs = [torch.randn(2, 1 + 3 * i, 96, device="cuda") for i in range(24)]
    want = [stack(x)[0] for x in inputs]
    torch.cuda.synchronize()

    def work(order):
        with torch.cuda.stream(torch.cuda.Stream()):
            got = [(i, stack(inputs[i])[0]) for i in order]
            torch.cuda.current_stream().synchronize()
        return all(torch.equal(y, want[i]) for i, y in got)

    with concurrent.futures.ThreadPoolExecutor(4) as pool:
        assert all(pool.map(work, [range(24), range(23, -1, -1), range(0, 24, 2), range(1, 24, 2)]))
    _lib.check_device_status(synchronize=True)
