"""The operators of a quantized feed-forward layer beside its plain GEMMs, as measured cases.

  add_norm  residual addition, RMSNorm and FP8 quantization in one pass; one scale per 128 columns ("block") or per row ("token")
  linear    FP8 GEMM with bias, activation and residual in its epilogue: activation(x @ w^T + bias) + residual, with per-token /
            per-channel scales ("token", optionally batched) or 1x128 / 128x128 block scales ("block")
  gated     both projections of a gated feed-forward layer in one block-scale GEMM, activation(gate) * up in its epilogue, the
            result in bf16 or as FP8 codes with one scale per 128 columns ("fp8"), the next GEMM's operand

Sizes are those of the repository's benchmark configurations and tests: one decoded token to a 16384-row prefill, row counts that
are not multiples of any tile, widths that are only multiples of 8 where the operator takes them.
"""
import os
import sys

import torch

own = False

DEV = "cuda"
EPS = 1e-6
E4M3 = torch.float8_e4m3fn
ACTIVATIONS = ("none", "relu", "gelu", "gelu_tanh", "silu")


def listed():
    return [
        # Between two layers while one sequence is decoded: launch latency is all of it.
        {"name": "norm_one_token", "op": "add_norm", "M": 1, "D": 4096, "scales": "block"},
        # The same for a batch of decoded sequences in a per-token-scaled model.
        {"name": "norm_decode", "op": "add_norm", "M": 32, "D": 8192, "scales": "token"},
        # A mid-sized ragged batch; the width is a multiple of 8 and not of 16.
        {"name": "norm_ragged", "op": "add_norm", "M": 1000, "D": 4104, "scales": "token"},
        # The longest prefill that the benchmark runs.
        {"name": "norm_prefill", "op": "add_norm", "M": 16384, "D": 8192, "scales": "block"},
        # Down-projection of a decode step, added to the residual stream: the weights have to cross HBM once.
        {"name": "down_decode", "op": "linear", "scales": "block", "batch": 1, "M": 16, "N": 4096, "K": 14336, "bias": False,
         "activation": "none", "residual": True},
        # Down-projection of a prefill with block scales.
        {"name": "down_prefill", "op": "linear", "scales": "block", "batch": 1, "M": 4096, "N": 4096, "K": 14336, "bias": False,
         "activation": "none", "residual": True},
        # First projection of a feed-forward layer without gate, a ragged prefill.
        {"name": "fc_gelu", "op": "linear", "scales": "token", "batch": 1, "M": 2000, "N": 14336, "K": 4096, "bias": True,
         "activation": "gelu", "residual": False},
        # Batched projections of a few ragged rows with everything that the epilogue does; N is a multiple of 8 only.
        {"name": "batched_ragged", "op": "linear", "scales": "token", "batch": 4, "M": 77, "N": 1032, "K": 1024, "bias": True,
         "activation": "gelu_tanh", "residual": True},
        # Gate and up projection of one decoded token.
        {"name": "gated_one_token", "op": "gated", "M": 1, "F": 14336, "K": 4096, "activation": "silu", "output": "fp8"},
        # A decode step of a batch that fills no tile, in the largest layer of the benchmark.
        {"name": "gated_decode", "op": "gated", "M": 24, "F": 28672, "K": 8192, "activation": "silu", "output": "bf16"},
        # A short ragged prompt in a small layer.
        {"name": "gated_ragged", "op": "gated", "M": 300, "F": 4096, "K": 2048, "activation": "gelu_tanh", "output": "fp8"},
        # A prefill.
        {"name": "gated_prefill", "op": "gated", "M": 4096, "F": 14336, "K": 4096, "activation": "silu", "output": "fp8"},
    ]


def draw(rng):
    def size(low, high, multiple):
        """Log-uniform over [low, high], a multiple of `multiple`."""
        v = low * (high / low) ** rng.random()
        return max(multiple, int(round(v / multiple)) * multiple)

    op = rng.choice(["add_norm", "linear", "linear", "gated", "gated"])
    if op == "add_norm":
        scales = rng.choice(["block", "token"])
        D = size(512, 16384, 128 if scales == "block" else 8)
        return {"op": op, "M": size(1, min(16384, 16384 * 8192 // D), 1), "D": D, "scales": scales}
    cost = 4096 * 28672 * 4096                     # no more than the largest listed product
    if op == "linear":
        scales = rng.choice(["block", "token"])
        batch = rng.choice([1, 1, 2, 4]) if scales == "token" else 1
        N = size(1024, 14336, 128 if scales == "block" or rng.random() < 0.5 else 8)
        K = size(1024, 14336, 128)
        return {"op": op, "scales": scales, "batch": batch, "M": size(1, min(8192, cost // (batch * N * K)), 1), "N": N, "K": K,
                "bias": rng.random() < 0.5, "activation": rng.choice(ACTIVATIONS), "residual": rng.random() < 0.5}
    F, K = size(1024, 28672, 128), size(1024, 8192, 128)
    return {"op": op, "M": size(1, min(8192, cost // (2 * F * K)), 1), "F": F, "K": K, "activation": rng.choice(ACTIVATIONS[1:]),
            "output": rng.choice(["fp8", "bf16"])}


# ---- inputs ---------------------------------------------------------------------------------------

def _activations(g, rows, K):
    """N(0, 1) with 1 % of the channels 20 times as large (outlier channels)."""
    x = torch.randn(rows, K, generator=g, device=DEV)
    x[:, torch.randperm(K, generator=g, device=DEV)[: max(1, K // 100)]] *= 20.0
    return x.bfloat16()


def _randn(g, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).bfloat16()


def _rows_fp8(x, group):
    """Codes and scales with one scale per `group` columns of a row."""
    v = x.float().view(x.shape[0], -1, group)
    s = (v.abs().amax(2, keepdim=True) / 448.0).clamp_min(1e-10)
    return (v / s).clamp(-448.0, 448.0).to(E4M3).view(x.shape), s.view(x.shape[0], -1)


def _tiles_fp8(w):
    """Codes and scales [K/128, N/128] of a weight with one scale per 128 x 128 tile."""
    N, K = w.shape
    v = w.float().view(N // 128, 128, K // 128, 128)
    s = (v.abs().amax((1, 3), keepdim=True) / 448.0).clamp_min(1e-10)
    return (v / s).clamp(-448.0, 448.0).to(E4M3).view(N, K), s.view(N // 128, K // 128).t().contiguous()


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    c = dict(case)
    s = {"case": c}
    M = c["M"]
    if c["op"] == "add_norm":
        D = c["D"]
        s["x"], s["residual"] = _randn(g, M, D), _activations(g, M, D)
        s["weight"] = (1.0 + 0.1 * torch.randn(D, generator=g, device=DEV)).bfloat16()
        s["sum"] = torch.empty(M, D, dtype=torch.bfloat16, device=DEV)
        s["codes"] = torch.empty(M, D, dtype=E4M3, device=DEV)
        s["scales"] = torch.empty(M, D // 128 if c["scales"] == "block" else 1, device=DEV)
        return s
    K = c["K"]
    if c["op"] == "gated":
        F = c["F"]
        s["a"], s["a_scale"] = _rows_fp8(_activations(g, M, K), 128)
        s["b"], s["b_scale"] = _tiles_fp8(_randn(g, 2 * F, K, scale=0.02))         # gate rows, then up rows
        s["c"] = torch.empty(M, F, dtype=E4M3 if c["output"] == "fp8" else torch.bfloat16, device=DEV)
        s["c_scale"] = torch.empty(M, F // 128, device=DEV) if c["output"] == "fp8" else None
        return s
    B, N = c["batch"], c["N"]
    lead = (B,) if B > 1 else ()
    if c["scales"] == "block":
        s["a"], s["a_scale"] = _rows_fp8(_activations(g, M, K), 128)
        s["b"], s["b_scale"] = _tiles_fp8(_randn(g, N, K, scale=0.02))
    else:
        a, sa = _rows_fp8(_activations(g, B * M, K), K)
        b, sb = _rows_fp8(_randn(g, B * N, K, scale=0.02), K)
        s["a"], s["b"] = a.view(*lead, M, K), b.view(*lead, N, K)
        s["a_scale"], s["b_scale"] = sa.view(*lead, M), sb.view(*lead, N)
    s["bias"] = _randn(g, *lead, N) if c["bias"] else None
    s["residual"] = _randn(g, *lead, M, N) if c["residual"] else None
    s["c"] = torch.empty(*lead, M, N, dtype=torch.bfloat16, device=DEV)
    return s


# ---- one pass -------------------------------------------------------------------------------------

def run(state):
    c = state["case"]
    if own:
        return _run_own(c, state)
    if c["op"] == "add_norm":
        return _plain_add_norm(c, state)
    return _plain_gated(c, state) if c["op"] == "gated" else _plain_linear(c, state)


_hk = None


def _framework():
    global _hk
    if _hk is None:
        package = os.path.abspath("amd-kernels_b200")
        if package not in sys.path:
            sys.path.insert(0, package)
        import hipkittens
        _hk = hipkittens
    return _hk


def _run_own(c, s):
    hk = _framework()
    if c["op"] == "add_norm":
        hk.fused_add_rmsnorm_fp8_quant_fwd(s["x"], s["residual"], s["weight"], s["codes"], s["scales"], s["sum"], EPS)
        return s["sum"], s["codes"], s["scales"]
    if c["op"] == "gated":
        hk.gemm.a8w8_blockscale.dispatch_gated(s["a"], s["b"], s["c"], s["a_scale"], s["b_scale"], s["c_scale"], c["activation"])
        return (s["c"], s["c_scale"]) if c["output"] == "fp8" else s["c"]
    gemm = hk.gemm.a8w8_blockscale if c["scales"] == "block" else hk.gemm.a8w8_per_token
    gemm.dispatch_epilogue(s["a"], s["b"], s["c"], s["a_scale"], s["b_scale"], s["bias"], c["activation"], s["residual"])
    return s["c"]


def _to_fp8(y, group):
    v = y.view(y.shape[0], -1, group)
    s = (v.abs().amax(2, keepdim=True) / 448.0).clamp_min(1e-10)
    return (v / s).clamp(-448.0, 448.0).to(E4M3).view(y.shape), s.view(y.shape[0], -1)


def _act(v, name):
    if name == "relu":
        return v.clamp_min(0.0)
    if name == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * 0.5 ** 0.5))
    if name == "gelu_tanh":
        return 0.5 * v * (1.0 + torch.tanh((2.0 / torch.pi) ** 0.5 * (v + 0.044715 * v * v * v)))
    if name == "silu":
        return v / (1.0 + torch.exp(-v))
    return v


def _plain_add_norm(c, s):
    # the sum is rounded once, to the type of the residual stream, and the norm is that of the stream
    total = (s["x"].float() + s["residual"].float()).bfloat16()
    h = total.float()
    y = h * torch.rsqrt((h * h).mean(1, keepdim=True) + EPS) * s["weight"].float()
    codes, scales = _to_fp8(y, 128 if c["scales"] == "block" else c["D"])
    return total, codes, scales


def _block_product(s):
    """x @ w^T of block-scaled operands."""
    a = s["a"].float().view(s["a"].shape[0], -1, 128) * s["a_scale"][:, :, None]
    N, K = s["b"].shape
    b = s["b"].float().view(N // 128, 128, K // 128, 128) * s["b_scale"].t()[:, None, :, None]
    return a.view(s["a"].shape) @ b.view(N, K).t()


def _plain_gated(c, s):
    p = _block_product(s)
    y = _act(p[:, :c["F"]], c["activation"]) * p[:, c["F"]:]
    return _to_fp8(y, 128) if c["output"] == "fp8" else y.bfloat16()


def _plain_linear(c, s):
    if c["scales"] == "block":
        v = _block_product(s)
    else:
        v = (s["a"].float() @ s["b"].float().transpose(-1, -2)) * s["a_scale"][..., :, None] * s["b_scale"][..., None, :]
    if s["bias"] is not None:
        v = v + s["bias"].float().unsqueeze(-2)
    v = _act(v, c["activation"])
    if s["residual"] is not None:
        v = v + s["residual"].float()
    return v.bfloat16()


# ---- what a pass cannot do without -----------------------------------------------------------------

def work(case):
    c, M = case, case["M"]
    if c["op"] == "add_norm":
        D = c["D"]
        n = M * D
        # x and residual in, sum and codes out, the scales; per element: the sum, its square and sum, norm, gain, maximum, division
        return {"bytes": n * (2 + 2 + 2 + 1) + 2 * D + 4 * M * (D // 128 if c["scales"] == "block" else 1), "flops": 8 * n}
    K = c["K"]
    if c["op"] == "gated":
        F = c["F"]
        out = M * F + 4 * M * (F // 128) if c["output"] == "fp8" else 2 * M * F
        return {"bytes": (M + 2 * F) * K + 4 * M * (K // 128) + 4 * (K // 128) * (2 * F // 128) + out, "flops": 2 * M * 2 * F * K}
    B, N = c["batch"], c["N"]
    scales = 4 * (M * (K // 128) + (K // 128) * (N // 128)) if c["scales"] == "block" else 4 * B * (M + N)
    extra = (2 * B * N if c["bias"] else 0) + (2 * B * M * N if c["residual"] else 0)
    return {"bytes": B * (M + N) * K + scales + extra + 2 * B * M * N, "flops": 2 * B * M * N * K}


# ---- the definition in 64 bits ------------------------------------------------------------------------

def _exact_act(v, name):
    if name == "relu":
        return torch.where(v > 0, v, torch.zeros_like(v))
    if name == "gelu":
        return v * 0.5 * torch.special.erfc(-v / 2.0 ** 0.5)                 # x times the normal distribution function
    if name == "gelu_tanh":
        return v * torch.sigmoid(2.0 * (2.0 / torch.pi) ** 0.5 * (v + 0.044715 * v.pow(3)))
    if name == "silu":
        return v * torch.sigmoid(v)
    return v


def _exact_scaled(y, group):
    """The quotients before they are rounded to 8 bits, and the scales."""
    top = y.abs().unflatten(1, (-1, group)).amax(2)
    scale = torch.maximum(top / 448.0, torch.full_like(top, 1e-10))
    return y / scale.repeat_interleave(group, 1), scale


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] == "add_norm":
        total = (s["x"].double() + s["residual"].double()).to(torch.bfloat16).double()
        y = total / (total.pow(2).mean(1, keepdim=True) + EPS).sqrt() * s["weight"].double()
        return (total, *_exact_scaled(y, 128 if c["scales"] == "block" else c["D"]))
    a, b = s["a"].double(), s["b"].double()
    if c["op"] == "gated" or c["scales"] == "block":
        a *= s["a_scale"].double().repeat_interleave(128, 1)
        b *= s["b_scale"].double().t().repeat_interleave(128, 0).repeat_interleave(128, 1)
    else:
        a *= s["a_scale"].double().unsqueeze(-1)
        b *= s["b_scale"].double().unsqueeze(-1)
    if c["op"] == "gated":
        gate, up = (a @ half.t() for half in b.chunk(2))
        y = _exact_act(gate, c["activation"]) * up
        return _exact_scaled(y, 128) if c["output"] == "fp8" else y
    v = torch.einsum("...mk,...nk->...mn", a, b)
    if c["bias"]:
        v += s["bias"].double().unsqueeze(-2)
    v = _exact_act(v, c["activation"])
    return v + s["residual"].double() if c["residual"] else v
