"""Cases of the 8-bit serving path and of the residual RMS norm around the gated scan.

An SSM block normalises its residual stream, multiplies it with five projections, scans, and
multiplies the result with the output projection.  Four operators carry that in 8 bits:

  norm_train   ``norm.add_rms_norm``: h = x + residual, y = h * weight / sqrt(mean(h^2) + eps),
               forward and backward (the training form);
  norm_fp8     ``norm.add_rms_norm_fp8``: the same sum and norm, y left in e4m3 with one scale for
               each 128 values of a row (the serving form; prompts and single tokens);
  quant        ``fp8.quantize_rows`` / ``fp8.quantize_weight``: e4m3 values with a scale for each
               128 values of a row, or for each 128 x 128 block of a weight;
  matmul       ``fp8.matmul_fp8``: y[m, n] = sum_k x[m, k] w[n, k] + bias[n] on such operands, the
               scales applied per block of 128 along k.

Quantisation: scale = max(amax, 2^-100) / 448, value = e4m3(v / scale), round to nearest even.
The norm is that of the stored (rounded) sum h.
"""
import torch

own = False

E4M3_MAX = 448.0
AMAX_FLOOR = 2.0 ** -100
EPS = 1e-5
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------
def listed():
    return [
        # decoding one sequence: the norm before the projections, latency only
        dict(name="norm_fp8 one token", op="norm_fp8", rows=1, H=1024, x="bf16", res="bf16"),
        # a prompt batch (16 x 4096 tokens, hidden 1024) over a 32-bit residual stream
        dict(name="norm_fp8 prompt", op="norm_fp8", rows=65536, H=1024, x="bf16", res="fp32"),
        # training the 12-layer configuration: 16 x 4096 tokens, hidden 1024, fp32 parameters
        dict(name="norm_train fp32", op="norm_train", rows=65536, H=1024, x="fp32", res="fp32"),
        # training with 16-bit activations, a hidden size and a row count that fit no vector or tile
        dict(name="norm_train odd bf16", op="norm_train", rows=4099, H=2050, x="bf16", res="bf16"),
        # the scan's output of 16 sequences that decode together, before the output projection
        dict(name="quant decode batch", op="quant", what="rows", rows=16, K=4096, x="bf16"),
        # the scan's output of a prompt batch (state size 4096)
        dict(name="quant prompt", op="quant", what="rows", rows=65536, K=4096, x="bf16"),
        # loading a block: its five projections as one weight
        dict(name="quant weight", op="quant", what="weight", rows=20480, K=1024, x="fp32"),
        # decoding one sequence: five projections of one token, bound by reading the weight
        dict(name="matmul one token", op="matmul", M=1, K=1024, N=20480, out="bf16", bias=True),
        # decoding 64 sequences together: the output projection, few rows and a long sum
        dict(name="matmul decode batch", op="matmul", M=64, K=4096, N=1024, out="bf16", bias=True),
        # a prompt of 4 x 4096 tokens: five projections
        dict(name="matmul prompt in", op="matmul", M=16384, K=1024, N=20480, out="bf16", bias=True),
        # the same prompt's output projection
        dict(name="matmul prompt out", op="matmul", M=16384, K=4096, N=1024, out="bf16", bias=True),
        # a ragged prompt through a layer whose sizes fit no tile, 32-bit output
        dict(name="matmul ragged fp32", op="matmul", M=1537, K=1100, N=2500, out="fp32", bias=False),
    ]


def _spread(rng, lo, hi):
    """A whole number whose logarithm is uniform between those of lo and hi."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["norm_fp8", "norm_train", "quant", "matmul", "matmul"])
    x = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op in ("norm_fp8", "norm_train"):
        H = _spread(rng, 16, 16384)
        rows = _spread(rng, 1, max(1, min(65536, 2 ** 26 // H)))
        res = rng.choice([x, "fp32"])
        if op == "norm_fp8" and rng.random() < 0.2:
            res = "none"  # the first block of a stack: nothing to add yet
        return dict(op=op, rows=rows, H=H, x=x, res=res)
    if op == "quant":
        K = _spread(rng, 16, 16384)
        rows = _spread(rng, 1, max(1, min(65536, 2 ** 27 // K)))
        return dict(op=op, what=rng.choice(["rows", "rows", "weight"]), rows=rows, K=K, x=x)
    K, N = _spread(rng, 16, 16384), _spread(rng, 16, 20480)
    M = _spread(rng, 1, max(1, min(16384, 16384 * 1024 * 20480 // (K * N))))
    return dict(op=op, M=M, K=K, N=N, out=rng.choice(["bf16", "bf16", "fp16", "fp32"]), bias=rng.random() < 0.5)


def work(case):
    size = {"fp32": 4, "bf16": 2, "fp16": 2, "none": 0}
    if case["op"] == "norm_train":  # forward reads x, residual and writes y, h; backward reads dy, dh, h, writes dx, dres
        n = case["rows"] * case["H"]
        sx, sr = size[case["x"]], size[case["res"]]
        # one gradient where both types are the same, two otherwise
        grads = sx if case["x"] == case["res"] else sx + sr
        return {"bytes": n * (2 * sx + 2 * sr) + n * (sx + 2 * sr + grads) + 3 * 4 * case["H"], "flops": 16 * n}
    if case["op"] == "norm_fp8":
        n = case["rows"] * case["H"]
        blocks = case["rows"] * -(-case["H"] // 128)
        return {"bytes": n * (size[case["x"]] + 2 * size[case["res"]] + 1) + 4 * blocks + 4 * case["H"], "flops": 8 * n}
    if case["op"] == "quant":
        n = case["rows"] * case["K"]
        blocks = -(-case["K"] // 128) * (case["rows"] if case["what"] == "rows" else -(-case["rows"] // 128))
        return {"bytes": n * (size[case["x"]] + 1) + 4 * blocks, "flops": 3 * n}
    M, K, N = case["M"], case["K"], case["N"]
    kb = -(-K // 128)
    nbytes = M * K + N * K + 4 * kb * (M + -(-N // 128)) + M * N * size[case["out"]] + (4 * N if case["bias"] else 0)
    return {"bytes": nbytes, "flops": 2 * M * N * K}


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _activations(rows, cols, gen):
    """Values as a residual branch holds them: normal, with a spread between channels of about e."""
    spread = torch.randn(cols, generator=gen, device="cuda").exp()
    return torch.randn(rows, cols, generator=gen, device="cuda") * spread


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    if case["op"] in ("norm_train", "norm_fp8"):
        rows, H, dt = case["rows"], case["H"], DTYPES[case["x"]]
        s = {"op": case["op"], "x": _activations(rows, H, gen).to(dt), "w": 1.0 + 0.3 * randn(H)}
        s["res"] = None if case["res"] == "none" else (4.0 * randn(rows, H)).to(DTYPES[case["res"]])
        if case["op"] == "norm_train":
            s["dy"], s["dh"] = randn(rows, H).to(dt), randn(rows, H).to(DTYPES[case["res"]])
            for k in ("x", "res", "w"):
                s[k].requires_grad_(True)
        return s
    if case["op"] == "quant":
        data = _activations(case["rows"], case["K"], gen).to(DTYPES[case["x"]])
        return {"op": "quant", "what": case["what"], "data": data}
    M, K, N = case["M"], case["K"], case["N"]
    xq, xs = _quantise(_activations(M, K, gen), 1)
    wq, ws = _quantise(randn(N, K) * K ** -0.5, 128)
    # as the quantiser leaves them: rows start on 16-byte boundaries, the rows' scales lie block by block
    pitch = -(-K // 16) * 16
    xp = torch.zeros(M, pitch, dtype=torch.uint8, device="cuda")
    wp = torch.zeros(N, pitch, dtype=torch.uint8, device="cuda")
    xp[:, :K] = xq.view(torch.uint8)
    wp[:, :K] = wq.view(torch.uint8)
    f8 = torch.float8_e4m3fn
    return {"op": "matmul", "xq": xp.view(f8)[:, :K], "xs": xs.t().contiguous().t(), "wq": wp.view(f8)[:, :K], "ws": ws,
            "bias": randn(N) if case["bias"] else None, "out": DTYPES[case["out"]]}


# ------------------------------------------------------------------------------------------------
# the operators: the framework's, or their plain form
# ------------------------------------------------------------------------------------------------
def _blocked(v, block_rows):
    """[rows, K] padded with zeros to whole blocks, as [row blocks, block_rows, column blocks, 128]."""
    rows, K = v.shape
    pr, pk = -rows % block_rows, -K % 128
    if pr or pk:
        v = torch.nn.functional.pad(v, (0, pk, 0, pr))
    return v.view(v.shape[0] // block_rows, block_rows, v.shape[1] // 128, 128)


def _quantise(v, block_rows):
    """fp32 [rows, K] -> (e4m3 [rows, K], fp32 scales [row blocks, column blocks])."""
    rows, K = v.shape
    b = _blocked(v, block_rows)
    scales = b.abs().amax(dim=(1, 3)).clamp_min(AMAX_FLOOR) / E4M3_MAX
    q = (b / scales[:, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    q = q.view(b.shape[0] * block_rows, b.shape[2] * 128)
    return (q if q.shape == (rows, K) else q.view(torch.uint8)[:rows, :K].contiguous().view(torch.float8_e4m3fn)), scales


def _dequantise(q, scales, block_rows):
    rows, K = q.shape
    b = _blocked(q.float(), block_rows) * scales[:, None, :, None]
    return b.reshape(b.shape[0] * block_rows, b.shape[2] * 128)[:rows, :K]


def _plain_norm(x, res, w):
    """(y in 32 bits, the stored sum, 1/rms)"""
    h = x if res is None else (x.float() + res.float()).to(res.dtype)
    hf = h.float()
    r = torch.rsqrt(hf.square().mean(-1, keepdim=True) + EPS)
    return hf * r * w, h, r


def _norm_train(s):
    x, res, w, dy, dh = s["x"], s["res"], s["w"], s["dy"], s["dh"]
    if own:
        from quick_ssm_b200.norm import add_rms_norm
        y, h = add_rms_norm(x, res, w, EPS)
        dx, dres, dw = torch.autograd.grad((y, h), (x, res, w), (dy, dh))
        return {"y": y.detach(), "h": h.detach(), "dx": dx, "dres": dres, "dw": dw}
    with torch.no_grad():
        y, h, r = _plain_norm(x, res, w)
        hf, g = h.float(), dy.float() * w
        dw = (dy.float() * hf * r).sum(0)
        d = dh.float() + r * g - hf * (r * r * r * (hf * g).mean(-1, keepdim=True))
        return {"y": y.to(x.dtype), "h": h, "dx": d.to(x.dtype), "dres": d.to(res.dtype), "dw": dw}


def _norm_fp8(s):
    x, res, w = s["x"], s["res"], s["w"]
    if own:
        from quick_ssm_b200.norm import add_rms_norm_fp8
        q, h = add_rms_norm_fp8(x, res, w, EPS)
        return {"q": q.values, "scales": q.scales, "h": h}
    y, h, _ = _plain_norm(x, res, w)
    q, scales = _quantise(y, 1)
    return {"q": q, "scales": scales, "h": h}


def _quant(s):
    if own:
        from quick_ssm_b200 import fp8
        q = (fp8.quantize_rows if s["what"] == "rows" else fp8.quantize_weight)(s["data"])
        return {"q": q.values, "scales": q.scales}
    q, scales = _quantise(s["data"].float(), 1 if s["what"] == "rows" else 128)
    return {"q": q, "scales": scales}


def _matmul(s):
    if own:
        from quick_ssm_b200 import fp8
        return fp8.matmul_fp8(fp8.Fp8Rows(s["xq"], s["xs"]), fp8.Fp8Weight(s["wq"], s["ws"]), s["bias"], out_dtype=s["out"])
    y = _dequantise(s["xq"], s["xs"], 1) @ _dequantise(s["wq"], s["ws"], 128).t()
    return (y if s["bias"] is None else y + s["bias"]).to(s["out"])


def run(state):
    return {"norm_train": _norm_train, "norm_fp8": _norm_fp8, "quant": _quant, "matmul": _matmul}[state["op"]](state)


# ------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ------------------------------------------------------------------------------------------------
def _e4m3_64(v):
    """float64 -> the nearest e4m3 value (ties to even), as float64: 3 fraction bits, exponents from -6."""
    mant, expo = torch.frexp(v)  # v = mant * 2^expo, 0.5 <= |mant| < 1
    step = torch.ldexp(torch.ones_like(v), expo.clamp_min(-5) - 4)
    return (torch.round(v / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def _quantise_64(v, block_rows):
    rows, K = v.shape
    kb, rb = -(-K // 128), -(-rows // block_rows)
    full = v.new_zeros(rb * block_rows, kb * 128)
    full[:rows, :K] = v
    amax = full.abs().reshape(rb, block_rows, kb, 128).amax(3).amax(1)
    scales = torch.maximum(amax, torch.full_like(amax, AMAX_FLOOR)) / E4M3_MAX
    per = scales.repeat_interleave(block_rows, 0)[:rows].repeat_interleave(128, 1)[:, :K]
    return {"q": _e4m3_64(v / per), "scales": scales}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "quant":
            return _quantise_64(s["data"].double(), 1 if case["what"] == "rows" else 128)
        if case["op"] == "matmul":
            K, N = case["K"], case["N"]
            x = s["xq"].to(torch.float32).double() * s["xs"].double().repeat_interleave(128, 1)[:, :K]
            w = s["ws"].double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
            y = torch.matmul(x, (s["wq"].to(torch.float32).double() * w).t())
            return y if s["bias"] is None else y.add_(s["bias"].double())
        x, w = s["x"].double(), s["w"].double()
        total = x if s["res"] is None else x + s["res"].double()
        # the norm's input is the sum as it is stored; what is returned for h is the sum itself
        h = total if s["res"] is None else total.to(s["res"].dtype).double()
        inv = 1.0 / torch.sqrt((h * h).sum(-1, keepdim=True) / h.shape[-1] + EPS)
        y = h * inv * w
        if case["op"] == "norm_fp8":
            return {**_quantise_64(y, 1), "h": total}
        dy, dh = s["dy"].double(), s["dh"].double()
        xhat = h * inv
        gw = dy * w
        d = dh + inv * (gw - xhat * (gw * xhat).sum(-1, keepdim=True) / h.shape[-1])
        return {"y": y, "h": total, "dx": d, "dres": d, "dw": (dy * xhat).sum(0)}
