"""TEST INFRASTRUCTURE — the correctness oracle.  Not part of the product.

Only tests/, __graft_entry__.smoke() and the CPU-baseline legs of bench.py may
import this package; nothing under peakgemm_b200/ does.

GEMM oracle: the reference project checks its half-precision kernel against
``sgemm::sgemm_naive_kernel`` (src/impl/sgemm_impl.h:9-26; used by
test/cpp/test_gemm_half.cpp:62-63): ``acc_fp32 += float(a[mi*k+ki]) * float(b[ni*k+ki])``
over increasing ki, then a cast to the 16-bit type.  ``gemm_exact`` is that loop
in C (oracle/gemm_oracle.c, bit-identical to the reference kernel because the
products are exact in fp32); ``gemm_fp32`` is the same contraction through
torch's CPU fp32 matmul (summation order differs; what test/test_gemm.py:37-38
does with F.linear) and is the fast form used for large shapes and as the timed
CPU baseline.

PARITY PINNING.  The reference ships no golden vectors for this path (its tests
use unseeded random inputs and print, test/cpp/test_gemm_half.cpp:37-46,
test/test_gemm.py:55-60).  The GEMM oracle is pinned against outputs of the
reference's own kernels run on a B200 (tests/golden/, made by
tests/golden/make_golden.py from oracle/_ref/libref_peakgemm.so).

RMSNorm oracle: PARITY UNPINNED — the reference has no RMSNorm operator, kernel or
test.  The oracle is the textbook definition in fp32 (what
torch.nn.functional.rms_norm computes) with the closed-form gradients.
"""
from __future__ import annotations

import ctypes
import importlib.util
import math
import os

import numpy as np
import torch

_HERE = os.path.dirname(os.path.abspath(__file__))


def _builder():
    spec = importlib.util.spec_from_file_location("_oracle_build", os.path.join(_HERE, "build_oracle.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


_cpu_lib = None


def cpu_lib() -> ctypes.CDLL:
    global _cpu_lib
    if _cpu_lib is None:
        path = _builder().build_cpu()
        lib = ctypes.CDLL(path)
        i64, p = ctypes.c_int64, ctypes.c_void_p
        for name in ("oracle_gemm", "oracle_gemm_acc"):
            fn = getattr(lib, name)
            fn.restype = ctypes.c_int
            fn.argtypes = [p, p, p, i64, i64, i64, ctypes.c_int]
        _cpu_lib = lib
    return _cpu_lib


def _bits(t: torch.Tensor) -> np.ndarray:
    assert t.dtype in (torch.bfloat16, torch.float16) and t.device.type == "cpu"
    return t.contiguous().view(torch.int16).numpy().view(np.uint16)


def gemm_exact(a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    """C = A @ B^T exactly as sgemm_naive_kernel computes it (k-ordered fp32 sum, cast to a.dtype)."""
    m, k = a.shape
    n = b.shape[0]
    assert b.shape[1] == k and a.dtype == b.dtype
    ab, bb = _bits(a), _bits(b)
    c = np.empty((m, n), dtype=np.uint16)
    r = cpu_lib().oracle_gemm(c.ctypes.data, ab.ctypes.data, bb.ctypes.data, m, n, k, int(a.dtype == torch.bfloat16))
    assert r == 0
    return torch.from_numpy(c.view(np.int16)).view(a.dtype)


def gemm_exact_acc(a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    """The unrounded fp32 accumulators of gemm_exact."""
    m, k = a.shape
    n = b.shape[0]
    ab, bb = _bits(a), _bits(b)
    acc = np.empty((m, n), dtype=np.float32)
    r = cpu_lib().oracle_gemm_acc(acc.ctypes.data, ab.ctypes.data, bb.ctypes.data, m, n, k,
                                  int(a.dtype == torch.bfloat16))
    assert r == 0
    return torch.from_numpy(acc)


def gemm_fp32(a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    """fp32 C = A.float() @ B.float()^T on the CPU (torch); unrounded."""
    return torch.nn.functional.linear(a.float(), b.float())


def gemm_tolerance(k: int, c_ref: torch.Tensor, out_dtype: torch.dtype = torch.bfloat16) -> float:
    """Acceptance bound on max|C - C_ref| for a 16-bit output.

    2e-2 * sqrt(k/4096) * max|C_ref|  (the accumulation term), plus one unit of output rounding at
    max|C_ref|: 2^-8 relative for bf16, 2^-11 for fp16.  Without the second term the bound drops
    below the rounding of the output type itself for k < ~160 (bf16), which no kernel could meet.
    """
    cmax = float(c_ref.abs().max())
    eps_out = 2.0 ** -8 if out_dtype == torch.bfloat16 else 2.0 ** -11
    return 2e-2 * math.sqrt(max(k, 1) / 4096.0) * cmax + eps_out * cmax


def reference_abs_tolerance(k: int) -> float:
    """The reference test's own bound: |out - ref| <= 0.5 * k / 4096 (test_gemm_half.cpp:158,167)."""
    return 0.5 * k / 4096.0


# ------------------------------------------------------------------ RMSNorm ----

def rmsnorm_fwd(x: torch.Tensor, gamma: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    """fp32 y (unrounded) = x * rsqrt(mean(x^2) + eps) * gamma over the last dimension."""
    xf = x.float()
    rstd = torch.rsqrt(xf.pow(2).mean(dim=-1, keepdim=True) + eps)
    return (xf * rstd) * gamma.float()


def rmsnorm_bwd(dy: torch.Tensor, x: torch.Tensor, gamma: torch.Tensor, eps: float = 1e-6):
    """fp32 (dx, dgamma), closed form:  dx = rstd * (g - xhat * mean(g * xhat)),  dgamma = sum_rows dy * xhat."""
    xf, dyf, g32 = x.float(), dy.float(), gamma.float()
    rstd = torch.rsqrt(xf.pow(2).mean(dim=-1, keepdim=True) + eps)
    xhat = xf * rstd
    g = dyf * g32
    dx = rstd * (g - xhat * (g * xhat).mean(dim=-1, keepdim=True))
    dgamma = (dyf * xhat).reshape(-1, x.shape[-1]).double().sum(dim=0).float()
    return dx, dgamma


def rmsnorm_bwd_dx_slack(dy: torch.Tensor, x: torch.Tensor, gamma: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    """Per-element absolute slack for dx on top of one 16-bit ulp: the fp32 error of the formula itself.

    dx = rstd * (g - xhat * c), c = mean_j(g * xhat), subtracts two fp32 numbers that can nearly cancel,
    and c is itself a sum of h terms of mixed sign.  Two correct fp32 evaluations that differ only in the
    order of the row reductions can therefore differ by about
        2^-24 * rstd * ( 8 |g| + 8 |xhat c| + |xhat| * sqrt(h) * mean_j |g xhat| )
    (a few roundings on each operand, plus the summation error of c, ~ sqrt(h) * 2^-24 * mean|terms|),
    which exceeds one 16-bit ulp only where dx cancelled to almost nothing.  This returns that bound.
    """
    xf, dyf, g32 = x.float(), dy.float(), gamma.float()
    h = x.shape[-1]
    rstd = torch.rsqrt(xf.pow(2).mean(dim=-1, keepdim=True) + eps)
    xhat = xf * rstd
    g = dyf * g32
    gx = g * xhat
    c = gx.mean(dim=-1, keepdim=True)
    c_err = math.sqrt(h) * gx.abs().mean(dim=-1, keepdim=True)
    return 2.0 ** -24 * rstd * (8.0 * g.abs() + 8.0 * (xhat * c).abs() + xhat.abs() * c_err)


def within_ulp_or_slack(out: torch.Tensor, ref_fp32: torch.Tensor, slack: torch.Tensor | None = None,
                        ulps: int = 1) -> torch.Tensor:
    """Elementwise: out within `ulps` 16-bit ulps of round(ref), or |out - ref| <= slack."""
    ok = ulp_distance_16(out, ref_fp32) <= ulps
    if slack is not None:
        ok |= (out.float() - ref_fp32).abs() <= slack + (ref_fp32.to(out.dtype).float() - ref_fp32).abs()
    return ok


def ulp_distance_16(out: torch.Tensor, ref_fp32: torch.Tensor) -> torch.Tensor:
    """|out - round(ref)| in units of out's 16-bit ulp at round(ref), elementwise (int64).

    Both are mapped to a monotone integer line (sign-magnitude -> two's complement),
    so the difference counts representable values between them."""
    ref = ref_fp32.to(out.dtype)

    def line(t):
        i = t.contiguous().view(torch.int16).to(torch.int64)
        return torch.where(i < 0, -(i & 0x7FFF), i)

    return (line(out) - line(ref)).abs()


# ---------------------------------------------------- fused epilogue / chains ----
# PARITY UNPINNED: the reference has no fused epilogue and no RMSNorm; these restate the definitions.

def rmsnorm_rstd(x: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    """rstd[r] = rsqrt(mean(x[r,:]^2) + eps), evaluated in float64, returned as float64."""
    xd = x.double()
    return torch.rsqrt(xd.pow(2).mean(dim=-1) + eps)


def gemm_fused(a: torch.Tensor, b: torch.Tensor, row_scale=None, bias=None, residual=None) -> torch.Tensor:
    """Unrounded fp32 row_scale[:,None] * (A @ B^T) + bias[None,:] + residual (absent terms skipped)."""
    out = gemm_fp32(a, b).double()
    if row_scale is not None:
        out = out * row_scale.double()[:, None]
    if bias is not None:
        out = out + bias.double()[None, :]
    if residual is not None:
        out = out + residual.double()
    return out.float()


def gemm_fused_slack(a: torch.Tensor, b: torch.Tensor, row_scale=None) -> torch.Tensor:
    """Per-element slack for a fp32 accumulation in another order: 2^-17 * |row_scale| * (|A| @ |B|^T).

    The forward error of a length-k fp32 dot product is bounded by k * 2^-24 * sum|a_i b_i| and is
    typically sqrt(k) * 2^-24 of it; 2^-17 covers k up to 16384 at the typical rate."""
    s = torch.nn.functional.linear(a.float().abs(), b.float().abs()) * 2.0 ** -17
    if row_scale is not None:
        s = s * row_scale.float().abs()[:, None]
    return s


def rmsnorm_linear(x: torch.Tensor, gamma: torch.Tensor, w: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    """Unrounded fp32 rms_norm(x; gamma) @ w^T by the definition (no folding, no intermediate rounding)."""
    y = x.double() * rmsnorm_rstd(x, eps)[:, None] * gamma.double()[None, :]
    return (y @ w.double().t()).float()


# ------------------------------------------------------------ input generators ----
# Seeded on the CPU so the oracle and the GPU see identical bits.

def gemm_inputs_uniform(m: int, n: int, k: int, dtype: torch.dtype, seed: int):
    """A[m,k], B[n,k] ~ U[-1,1] (the distribution of test/test_gemm.py:24-29), drawn A then B."""
    g = torch.Generator().manual_seed(seed)
    a = (torch.rand(m, k, generator=g) * 2 - 1).to(dtype)
    b = (torch.rand(n, k, generator=g) * 2 - 1).to(dtype)
    return a, b


def gemm_inputs_llm(m: int, n: int, k: int, dtype: torch.dtype, seed: int):
    """Activations A ~ N(0,1), weights B ~ N(0, 0.02)."""
    g = torch.Generator().manual_seed(seed)
    a = torch.randn(m, k, generator=g).to(dtype)
    b = (0.02 * torch.randn(n, k, generator=g)).to(dtype)
    return a, b


def rmsnorm_inputs(rows: int, h: int, dtype: torch.dtype, seed: int):
    """x, dy ~ N(0,1) in `dtype`; gamma ~ N(1, 0.1) fp32; drawn x, dy, gamma."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, h, generator=g).to(dtype)
    dy = torch.randn(rows, h, generator=g).to(dtype)
    gamma = 1 + 0.1 * torch.randn(h, generator=g)
    return x, dy, gamma


# ------------------------------------------------ norms around a gated residual ----
# PARITY UNPINNED: the reference has neither operator; these restate the definitions in float64, on the inputs' device,
# together with per-element bounds on what an fp32 evaluation may be off by.
#
# Bounds.  The sums over a row are sums of h products in some tree order: each of a row's at most 64 serial additions in
# 32 bits (a thread's further ones, which grow with h, are in 64), 5 shuffle levels and 32 warp sums rounds by 2^-24, so a sum of positive terms is within 2^-17 of itself, rstd (its
# inverse square root) within 2^-18 + 2^-22, and a sum of mixed terms within 2^-17 of the sum of their absolute values.
# REL = 2^-17 covers a product of such a factor with the few roundings of the elementwise arithmetic.

REL = 2.0 ** -17


def _residual_terms(u, residual, gamma_post, gate, res_scale, eps):
    u = u.double()
    rows, h = u.shape
    one = torch.ones(1, 1, dtype=torch.float64, device=u.device)
    rstd = torch.rsqrt(u.pow(2).mean(-1, keepdim=True) + eps) if gamma_post is not None else one
    gp = gamma_post.double()[None, :] if gamma_post is not None else one
    g = one if gate is None else gate.double().repeat_interleave(rows // gate.shape[0], dim=0)
    al = one if res_scale is None else res_scale.double()[None, :]
    return u, rstd, gp, g, al


def rmsnorm_residual_fwd(u, residual, gamma_post=None, gate=None, res_scale=None, gamma_pre=None, eps: float = 1e-6):
    """(s, y, bound of s, bound of y) unrounded, float64; y and its bound None without gamma_pre."""
    u, rstd, gp, g, al = _residual_terms(u, residual, gamma_post, gate, res_scale, eps)
    a, b = al * residual.double(), g * (u * rstd * gp)
    s = a + b
    es = REL * (a.abs() + b.abs())
    if gamma_pre is None:
        return s, None, es, None
    rs = torch.rsqrt(s.pow(2).mean(-1, keepdim=True) + eps)
    y = s * rs * gamma_pre.double()
    # rstd(s) moves by rstd^2 * mean(|s| * error of s) relatively
    ey = es * rs * gamma_pre.double().abs() + y.abs() * (REL + rs * rs * (s.abs() * es).mean(-1, keepdim=True))
    return s, y, es, ey


def rmsnorm_residual_bwd(dy, ds, s, u, residual=None, gamma_post=None, gate=None, res_scale=None, gamma_pre=None,
                         eps: float = 1e-6, serial_rows: int = 512):
    """{name: (gradient, bound)} unrounded, float64.  serial_rows: rows that are added one after the other at most."""
    shape = (s if s is not None else u if u is not None else ds).shape
    dev = (ds if ds is not None else dy).device
    rows, h = shape
    ref = u if u is not None else torch.zeros(shape, device=dev)
    ud, rstd, gp, g, al = _residual_terms(ref, residual, gamma_post, gate, res_scale, eps)
    D = ds.double() if ds is not None else torch.zeros(shape, dtype=torch.float64, device=dev)
    eD = torch.zeros_like(D)
    out = {}
    step = (min(rows, serial_rows) + 64) * 2.0 ** -24
    if gamma_pre is not None:
        sd = s.double()
        rs = torch.rsqrt(sd.pow(2).mean(-1, keepdim=True) + eps)
        sh, w = sd * rs, dy.double() * gamma_pre.double()
        c = (w * sh).mean(-1, keepdim=True)
        D = D + rs * (w - sh * c)
        eD = REL * ((ds.double().abs() if ds is not None else 0) + rs * (w.abs() + sh.abs() * (c.abs() + (w * sh).abs().mean(-1, keepdim=True))))
        t = dy.double() * sh
        out["dgamma_pre"] = (t.sum(0), ((REL + step) * t.abs()).sum(0))
    out["dresidual"] = (al * D, al.abs() * (eD + REL * D.abs()))
    if res_scale is not None and residual is not None:
        t, e = D * residual.double(), (eD + (REL + step) * D.abs()) * residual.double().abs()
        one = res_scale.numel() == 1
        out["dres_scale"] = (t.sum().view(1), e.sum().view(1)) if one else (t.sum(0), e.sum(0))
    uh = ud * rstd
    if gate is not None and u is not None:
        p = uh * gp
        G = gate.shape[0]
        out["dgate"] = ((D * p).view(G, -1, h).sum(1), ((eD + (REL + step) * D.abs()) * p.abs()).view(G, -1, h).sum(1))
    e = g * D
    ee = g.abs() * (eD + REL * D.abs())
    if gamma_post is None:
        out["du"] = (e.expand(shape), ee.expand(shape))
    else:
        t = e * uh
        out["dgamma_post"] = (t.sum(0), ((ee + (REL + step) * e.abs()) * uh.abs()).sum(0))
        v = e * gp
        ev = ee * gp.abs() + REL * v.abs()
        c = (v * uh).mean(-1, keepdim=True)
        ec = ((ev + REL * v.abs()) * uh.abs()).mean(-1, keepdim=True)
        out["du"] = (rstd * (v - uh * c), rstd * (ev + uh.abs() * (ec + REL * c.abs())) + REL * (rstd * (v - uh * c)).abs())
    return out


def rmsnorm_residual_inputs(rows: int, h: int, dtype: torch.dtype, seed: int, *, post=True, gates=0, res_scale=0, pre=True):
    """Seeded inputs of the operator: u, residual, ds, dy ~ N(0,1), gains ~ N(1, 0.1), gate ~ N(0, 0.5)."""
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g)    # noqa: E731
    x = {"u": n(rows, h).to(dtype), "residual": n(rows, h).to(dtype), "ds": n(rows, h).to(dtype),
         "dy": n(rows, h).to(dtype) if pre else None}
    x["gamma_post"] = 1 + 0.1 * n(h) if post else None
    x["gamma_pre"] = 1 + 0.1 * n(h) if pre else None
    x["gate"] = (0.5 * n(gates, h)).to(dtype) if gates else None
    x["res_scale"] = 1 + 0.1 * n(res_scale) if res_scale else None
    return x


# --------------------------------------------------- adapters beside a projection ----
# PARITY UNPINNED: the reference has no adapters; the definition in float64, on the inputs' device.

def gemm_lora(a, b, lora_a, lora_b, ids, scale=None, row_scale=None, bias=None, residual=None, v_terms: int = 1):
    """(d, bound) unrounded, float64.

    bound: fp32 sums of products in another order are within 2^-17 of the sum of absolute values (gemm_fused_slack);
    v = scale * a A^T may go into the second product as the sum of v_terms values of the 16-bit type, each the rounding of
    what the ones before leave: half a step, eps / 2, of itself with one term, (eps / 2)^2 with two (and half the smallest
    step, where what is rounded is below the normal range)."""
    L, r, k = lora_a.shape
    ids = ids.long()
    u16 = (torch.finfo(a.dtype).eps / 2) ** v_terms
    tiny = torch.finfo(a.dtype).smallest_normal * torch.finfo(a.dtype).eps / 2
    x, w = a.double(), b.double()
    d, e = x @ w.t(), 2.0 ** -17 * (x.abs() @ w.abs().t())
    for i in range(L):
        t = (ids == i).nonzero()[:, 0]
        if t.numel() == 0:
            continue
        s = 1.0 if scale is None else float(scale[i])
        A, B = lora_a[i].double(), lora_b[i].double()
        v = s * (x[t] @ A.t())
        ev = u16 * v.abs() + tiny + 2.0 ** -17 * abs(s) * (x[t].abs() @ A.abs().t())
        d[t] += v @ B.t()
        e[t] += (ev + 2.0 ** -17 * v.abs()) @ B.abs().t()
    if row_scale is not None:
        d, e = d * row_scale.double()[:, None], e * row_scale.double().abs()[:, None]
    for term in (bias, residual):
        if term is not None:
            d = d + term.double()
            e = e + 2.0 ** -23 * term.double().abs()
    return d, e + 2.0 ** -22 * d.abs()


def gemm_lora_inputs(m: int, n: int, k: int, adapters: int, rank: int, dtype: torch.dtype, seed: int, ids: str = "mixed"):
    """Seeded inputs: x ~ N(0,1), W ~ N(0, 0.02), A ~ N(0, 1/k), B ~ N(0, 0.02), scales in [0.5, 2); about an eighth of
    the rows without an adapter.  ids: "mixed" token by token, "runs" of one adapter each, "one", "none"."""
    g = torch.Generator().manual_seed(seed)
    n_ = lambda *s: torch.randn(*s, generator=g)    # noqa: E731
    x = {"a": n_(m, k).to(dtype), "b": (0.02 * n_(n, k)).to(dtype), "lora_a": (k ** -0.5 * n_(adapters, rank, k)).to(dtype),
         "lora_b": (0.02 * n_(adapters, n, rank)).to(dtype), "scale": 0.5 + 1.5 * torch.rand(adapters, generator=g)}
    i = torch.randint(0, adapters, (m,), generator=g)
    i[torch.rand(m, generator=g) < 0.125] = -1
    if ids == "runs":
        i = i.sort().values
    elif ids == "one":
        i[:] = adapters - 1
    elif ids == "none":
        i[:] = -1
    x["ids"] = i.int()
    return x


def gemm_lora_terms(m: int, n: int, dtype: torch.dtype, seed: int):
    g = torch.Generator().manual_seed(seed)
    return {"row_scale": 0.5 + torch.rand(m, generator=g), "bias": torch.randn(n, generator=g).to(dtype),
            "residual": torch.randn(m, n, generator=g).to(dtype)}
