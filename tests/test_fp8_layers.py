"""The blocks that call the residual norm and the 8-bit product: ``SSMStack`` (training) against the same blocks one after
the other, ``SSMFp8`` / ``SSMStackFp8`` (serving) against a plain 64-bit run of the same quantised arithmetic, prompts
against single tokens, captured against eager runs."""
import copy

import pytest
import torch

from quick_ssm_b200 import _lib, fp8
from quick_ssm_b200.layers import SSM, SSMFp8, SSMFused, SSMStack, SSMStackFp8
from quick_ssm_b200.norm import add_rms_norm
from quick_ssm_b200.streaming import ScanState, gated_scan_chunk, scan_chunk

from test_fp8 import plain_norm, plain_quantize, wide

gpu = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def blocks(n, hidden, mult, dtype=F32, compute=BF16, device="cuda", seed=0):
    torch.manual_seed(seed)
    made = [SSM(hidden, mult, dtype=dtype, compute_dtype=compute) for _ in range(n)]
    with torch.no_grad():
        for b in made:
            b.pre_norm.weight.add_(0.3 * torch.randn(hidden))
            b.A_proj.bias.add_(1.5)  # decays near one, as trained blocks have them
    return [b.to(device) for b in made]


def rel(got, want):
    return float((got.double().cpu() - want.double().cpu()).norm() / want.double().norm())


# ------------------------------------------------------------------------------------------------
# CPU
# ------------------------------------------------------------------------------------------------
def test_stack_on_cpu_is_the_sequence_of_its_blocks():
    made = blocks(3, 16, 2.0, compute=F32, device="cpu")
    stack = SSMStack(3, 16, 2.0, compute_dtype=F32)
    stack.load_state_dict({f"layers.{k}": v for k, v in torch.nn.Sequential(*made).state_dict().items()})
    x = want = torch.randn(2, 7, 16)
    for b in made:
        want = b(want, backend="torch")
    assert torch.equal(stack(x, backend="torch"), want)


def test_serving_refusals():
    with pytest.raises(RuntimeError, match="CUDA"):
        SSMFp8(SSM(16))
    with pytest.raises(ValueError, match="pre-norm"):
        SSMFp8(SSM(16, use_norm=False))
    with pytest.raises(ValueError, match="residual"):
        SSMFp8(SSM(16, use_residual=False))
    with pytest.raises(RuntimeError, match="CUDA"):
        gated_scan_chunk(*(torch.zeros(1, 2, 8) for _ in range(5)))
    with pytest.raises(ValueError, match="shape"):
        gated_scan_chunk(*(torch.zeros(1, 2, 8 + (i == 3)) for i in range(5)))


# ------------------------------------------------------------------------------------------------
# training
# ------------------------------------------------------------------------------------------------
@gpu
def test_stack_trains_like_its_blocks_one_after_the_other():
    """fp32 throughout, so what differs is the order of fp32 sums: 1e-5 of the largest value per block, four blocks,
    forward and backward (8 passes)."""
    made = blocks(4, 96, 2.0, compute=F32)
    seq = [SSMFused(96, 2.0, compute_dtype=F32).cuda() for _ in made]
    stack = SSMStack(4, 96, 2.0, compute_dtype=F32).cuda()
    for i, b in enumerate(made):
        seq[i].load_state_dict(b.state_dict())
        stack.layers[i].load_state_dict(b.state_dict())
    x, dy = torch.randn(2, 50, 96, device="cuda"), torch.randn(2, 50, 96, device="cuda")
    xs, xt = x.clone().requires_grad_(), x.clone().requires_grad_()
    want = xs
    for b in seq:
        want = b(want)
    want.backward(dy)
    got = stack(xt)
    got.backward(dy)
    pairs = [(got, want), (xt.grad, xs.grad)]
    pairs += [(p.grad, q.grad) for a, b in zip(stack.layers, seq) for p, q in zip(a.parameters(), b.parameters())]
    for g, w in pairs:
        assert (g - w).abs().max() <= 8e-5 * w.abs().max()
    _lib.check_device_status(synchronize=True)


@gpu
@pytest.mark.parametrize("x_dtype", [F32, BF16, torch.float16], ids=str)
def test_stack_under_autocast_takes_the_types_that_its_blocks_take(x_dtype):
    """bf16 branches on a residual stream of another type: promoted as the sequence's sums are."""
    seq = torch.nn.Sequential(*(SSMFused(64, compute_dtype=BF16) for _ in range(3))).cuda()
    stack = SSMStack(3, 64, compute_dtype=BF16).cuda()
    stack.load_state_dict({f"layers.{k}": v for k, v in seq.state_dict().items()})
    x = torch.randn(2, 9, 64, device="cuda").to(x_dtype)
    with torch.autocast("cuda", dtype=BF16):
        want, got = seq(x), stack(x)
    assert got.dtype == want.dtype and got.shape == want.shape and torch.isfinite(got).all()
    got.float().square().mean().backward()
    assert all(torch.isfinite(p.grad).all() for p in stack.parameters())


@gpu
def test_residual_norm_captured_with_its_backward():
    """Forward and backward in one graph, replayed on new inputs, equal the eager passes bit for bit; two such graphs
    replayed in turn do not disturb each other."""
    graphs = []
    for rows, H, dt in ((300, 512, BF16), (1000, 130, F32)):
        x, r = (torch.randn(rows, H, device="cuda").to(dt).requires_grad_() for _ in range(2))
        w = torch.rand(H, device="cuda").add_(0.5).requires_grad_()
        dy, dh = torch.randn_like(x), torch.randn_like(r)

        def step(x=x, r=r, w=w, dy=dy, dh=dh):
            y, h = add_rms_norm(x, r, w)
            return (y.detach(), h.detach(), *torch.autograd.grad((y, h), (x, r, w), (dy, dh)))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out, step, (x, r, w, dy, dh)))
    for turn in range(3):
        for _, _, _, ins in graphs:
            with torch.no_grad():
                for t in ins:
                    t.copy_(torch.randn_like(t))
        for graph, *_ in graphs:
            graph.replay()
        for _, out, step, _ in graphs:
            for got, want in zip(out, step()):
                assert torch.equal(got, want)


# ------------------------------------------------------------------------------------------------
# serving
# ------------------------------------------------------------------------------------------------
def plain_block(block, x, res, state):
    """The serving block's arithmetic in 64 bits: its quantisation points, none of its 16-bit roundings.
    x, res: [B, L, hidden] on the CPU; returns out, h, state [B, n]."""
    B, L, H = x.shape
    n = block.state_size_dim
    y, h, _ = plain_norm(x.reshape(-1, H), None if res is None else res.reshape(-1, H), block.norm_weight.cpu(), block.eps)
    w = {k: wide(getattr(block, f"{k}_values").cpu().view(torch.float8_e4m3fn), getattr(block, f"{k}_scales").cpu(), 128) for k in ("in", "out")}
    p = wide(*plain_quantize(y.float(), 1), 1) @ w["in"].t() + block.in_bias.double().cpu()
    pa, px, pc1, pc2, pd = p.view(B, L, 5 * n).split(n, -1)
    a, b, c = torch.sigmoid(pa), torch.sigmoid(pd), torch.nn.functional.silu(pc1) * pc2
    s, outs = state, []
    for t in range(L):
        s = a[:, t] * s + b[:, t] * px[:, t]
        outs.append(c[:, t] * s)
    out = wide(*plain_quantize(torch.stack(outs, 1).reshape(-1, n).float(), 1), 1) @ w["out"].t() + block.out_bias.double().cpu()
    return out.view(B, L, H), h.view(B, L, H), s


@gpu
@pytest.mark.parametrize("hidden,mult,L,res", [(64, 2.0, 40, F32), (128, 4.0, 1, BF16), (96, 1.5, 17, F32), (40, 1.1, 9, None)],
                         ids=str)
def test_serving_block_follows_the_plain_arithmetic(hidden, mult, L, res):
    """A bf16 rounding (2^-8 at most, 2^-9.8 in the mean) of the projections moves a value across a border of the next
    e4m3 rounding, 2^-4 of it, about once in 2^-9.8 / 2^-4 = 1/56 values: an error of 2^-4 / sqrt(56) = 0.8 % in norm
    behind each of the two quantisations of rounded values, 0.1 % for each of five roundings on the way (projections,
    gates, the product of two, y, out).  3 % covers them added up with a margin of two."""
    block = SSMFp8(blocks(1, hidden, mult)[0])
    torch.manual_seed(5)
    x = torch.randn(3, L, hidden).to(BF16)
    r = None if res is None else torch.randn(3, L, hidden).mul(2).to(res)
    s0 = torch.randn(3, block.state_size_dim)
    out, h, state = block(x.cuda(), None if r is None else r.cuda(), ScanState(s0.cuda()))
    want, want_h, want_s = plain_block(block, x, r, s0.double())
    assert out.dtype == BF16 and h.dtype == (res or BF16) and torch.equal(h.double().cpu(), want_h)
    assert rel(out, want) < 0.03 and rel(state.h, want_s) < 0.03
    _lib.check_device_status(synchronize=True)


@gpu
def test_serving_stack_is_near_the_stack_it_was_made_from():
    """e4m3 rounds a value by 2^-4 at most, 2^-5.8 in the mean of squares (1.8 %); each product has two such operands
    (2.5 % in norm), a block two products in a row with gates of slope at most 1.1 between them (under 10 %), and the
    residual stream, which is not quantised, carries most of the output: 10 % of the branches' sum."""
    made = blocks(3, 256, 2.0, compute=BF16)
    stack = SSMStackFp8(made)
    x = torch.randn(2, 64, 256, device="cuda")
    want = x
    with torch.no_grad():
        for b in made:
            want = b(want, scan_out_dtype=F32)
        got, states = stack(x)
    assert got.dtype == F32 and len(states) == 3
    assert rel(got - x, want - x) < 0.10


@gpu
@pytest.mark.parametrize("xd", [F32, BF16], ids=["fp32", "bf16"])
def test_prompt_and_single_tokens_agree(xd):
    """A prompt at once, in two pieces, and token by token.  Rows are quantised alone and products summed in fp32, so the
    passes differ by fp32 sums that round differently to bf16, now and then: a bf16 step (2^-8) and its consequences
    for the next quantisation, as in the block's test but rarer."""
    stack = SSMStackFp8(blocks(2, 128, 2.0))
    x = torch.randn(5, 20, 128, device="cuda").to(xd)
    whole, end = stack(x)
    first, mid = stack(x[:, :13])
    second, end2 = stack(x[:, 13:], mid)
    tokens, s = [], None
    for t in range(20):
        y, s = stack(x[:, t:t + 1], s)
        tokens.append(y)
    for got in (torch.cat([first, second], 1), torch.cat(tokens, 1)):
        assert rel(got, whole) < 0.02
    for a, b, c in zip(end, end2, s):
        assert rel(b.h, a.h) < 0.02 and rel(c.h, a.h) < 0.02
    empty, same = stack(x[:, :0], end)
    assert empty.shape == (5, 0, 128) and all(torch.equal(a.h, b.h) for a, b in zip(same, end))
    with pytest.raises(ValueError, match="states"):
        stack(x, end[:1])
    with pytest.raises(ValueError):
        stack(x[0])


@gpu
def test_single_token_step_captured_and_replayed():
    """A decoding step with its states updated in place, captured once and replayed, equals eager steps bit for bit; an
    eager prompt through the same blocks in between does not disturb it."""
    stack = SSMStackFp8(blocks(2, 128, 4.0))
    x = torch.randn(4, 1, 128, device="cuda").to(BF16)
    states = [ScanState.zeros(4, 512) for _ in range(2)]

    def step():
        y, after = stack(x, states)
        for s, a in zip(states, after):
            s.h.copy_(a.h)
        return y

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step()
    for s in states:
        s.h.zero_()
    eager = None
    for t in range(4):
        x.copy_(torch.randn(4, 1, 128, device="cuda"))
        graph.replay()
        want, eager = stack(x, eager)
        stack(torch.randn(2, 33, 128, device="cuda"))
        assert torch.equal(y, want)
        assert all(torch.equal(a.h, b.h) for a, b in zip(states, eager))
    _lib.check_device_status(synchronize=True)


@gpu
def test_serving_blocks_copy_and_load():
    made = blocks(2, 72, 1.5)
    a, b = SSMFp8(made[0]), SSMFp8(made[1])
    x = torch.randn(2, 6, 72, device="cuda")
    want = a(x)[0]
    assert not torch.equal(b(x)[0], want)
    b.load_state_dict(a.state_dict())
    assert torch.equal(b(x)[0], want) and torch.equal(copy.deepcopy(a)(x)[0], want)
    assert torch.equal(SSMFp8(made[0]).cpu().cuda()(x)[0], want)


@gpu
def test_gated_chunks_on_slices_match_separate_gates():
    """Column slices of one projection, with a carried state, fused and composed (sizes the copy engine cannot address)."""
    torch.manual_seed(3)
    for n in (64, 36):
        p = torch.randn(3, 30, 5 * n, device="cuda").to(BF16)
        parts = p.split(n, -1)
        y, s = gated_scan_chunk(*parts)
        a, x, c, b = (torch.sigmoid(parts[0]), parts[1], (torch.nn.functional.silu(parts[2]) * parts[3]), torch.sigmoid(parts[4]))
        want, ws = scan_chunk(x, a, b, c, out_dtype=BF16)
        y1, s1 = gated_scan_chunk(*(t[:, :11] for t in parts))
        y2, s2 = gated_scan_chunk(*(t[:, 11:] for t in parts), s1)
        # gates rounded to bf16 from approximations good to bf16: a step of 2^-8 here and there
        for g, w in ((y, want), (torch.cat([y1, y2], 1), want), (s.h, ws.h), (s2.h, ws.h)):
            assert rel(g, w) < 2 ** -7
        strided = ScanState(s1.h.t().contiguous().t())  # a state in another layout
        y3, s3 = gated_scan_chunk(*(t[:, 11:] for t in parts), strided)
        assert torch.equal(y3, y2) and torch.equal(s3.h, s2.h)


@gpu
@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_tensors_of_another_device_than_the_current_one():
    x = torch.randn(70, 256, device="cuda:1")
    w = fp8.quantize_weight(torch.randn(300, 256, device="cuda:1"))
    with torch.cuda.device(0):
        y = fp8.matmul_fp8(fp8.quantize_rows(x), w)
    with torch.cuda.device(1):
        want = fp8.matmul_fp8(fp8.quantize_rows(x), w)
    assert y.device == x.device and torch.equal(y, want)
