"""GPU: rms_norm_residual_fwd / _bwd against their definitions in float64.

Bounds (derived in oracle/__init__.py, before any run): a 16-bit output is the rounding of a number within the fp32
evaluation's bound of the exact one (half a step of the type on top, helpers.elementwise_ok); fp32 sums are within
their bound of the exact sums.  The reference project has no such operator (parity unpinned).
"""
import pytest
import torch

import oracle
from tests import helpers

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
PARAMS = ("gamma_post", "gate", "res_scale", "gamma_pre")


def make(rows, h, dtype, seed, **terms):
    x = oracle.rmsnorm_residual_inputs(rows, h, dtype, seed, **terms)
    return {k: v.cuda() if v is not None else None for k, v in x.items()}


def params(x):
    return {k: x[k] for k in PARAMS}


def check16(out, ref, bound, what):
    """Finite where the exact value rounds to a finite one; past the type's range (an fp16 row of zeros with rstd = 316
    has gradients of 316^2 = 10^5 > 65504) the infinity of its sign."""
    over = ~torch.isfinite(ref.to(out.dtype).float())
    assert torch.equal(torch.isfinite(out.float()), ~over), f"{what}: finite where it should not be, or the other way round"
    # the bound widened by the float64 reference's own rounding to fp32
    ok = helpers.elementwise_ok(out, ref.float(), (bound + 2.0 ** -24 * ref.abs()).float())
    ok = torch.where(over, out == ref.to(out.dtype), ok)
    assert ok.all(), f"{what}: {int((~ok).sum())} elements off, worst {(out.double() - ref).abs()[~ok].max().item():.3g}"


def check32(out, ref, bound, what):
    err = (out.double() - ref).abs()
    assert (err <= bound + 2.0 ** -24 * ref.abs()).all(), f"{what}: {err.max().item():.3g}, bound {bound.max().item():.3g}"


def forward(x, s=None, y=None, eps=1e-6):
    import PeakGemm

    s = helpers.garbage_like(x["u"].shape, x["u"].dtype, "cuda") if s is None else s
    if y is None and x["gamma_pre"] is not None:
        y = helpers.garbage_like(x["u"].shape, x["u"].dtype, "cuda")
    PeakGemm.rms_norm_residual_fwd(s, y, x["u"], x["residual"], eps=eps, **params(x))
    return s, y


def backward(x, s, du=None, dresidual=None, eps=1e-6):
    import PeakGemm

    shape, dtype = x["u"].shape, x["u"].dtype
    out = {"du": helpers.garbage_like(shape, dtype, "cuda") if du is None else du,
           "dresidual": helpers.garbage_like(shape, dtype, "cuda") if dresidual is None else dresidual}
    grads = {"d" + k: None if x[k] is None else torch.full_like(x[k], float("nan")) for k in PARAMS}
    PeakGemm.rms_norm_residual_bwd(out["du"], out["dresidual"], x["dy"], x["ds"], s, x["u"], residual=x["residual"],
                                   eps=eps, **params(x), **grads)
    out.update({k: v for k, v in grads.items() if v is not None})
    return out


def check_forward(x, s, y, eps=1e-6):
    rs, ry, es, ey = oracle.rmsnorm_residual_fwd(x["u"], x["residual"], **params(x), eps=eps)
    check16(s, rs, es, "s")
    if y is not None:
        check16(y, ry, ey, "y")


def check_backward(x, s, out, eps=1e-6):
    ref = oracle.rmsnorm_residual_bwd(x["dy"], x["ds"], s, x["u"], x["residual"], **params(x), eps=eps)
    assert set(out) <= set(ref)
    for k, v in out.items():
        (check16 if v.dtype != torch.float32 else check32)(v, *ref[k], k)


# every width class (one warp per row, several vectors per thread, rows over 16384 elements), odd row counts
SHAPES = [(1, 8), (5, 8), (7, 64), (33, 256), (100, 1000), (257, 4096), (64, 8192), (19, 5120), (301, 2048), (5, 16384),
          (4, 16392), (3, 24576), (2, 65544), (301, 4104), (150, 8200), (77, 12288), (40, 32768), (9, 32776)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows,h", SHAPES)
def test_all_terms(cuda, rows, h, dtype):
    for gates, res in ((0, 1), (1, h), (rows, 0)):
        x = make(rows, h, dtype, 61, gates=gates, res_scale=res)
        s, y = forward(x)
        check_forward(x, s, y)
        check_backward(x, s, backward(x, s))


@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("pre", [True, False])
@pytest.mark.parametrize("gates", [0, 1, 6, 66])
@pytest.mark.parametrize("res", [0, 1, 520])
def test_every_combination_of_terms(cuda, post, pre, gates, res):
    x = make(66, 520, BF16, 62, post=post, pre=pre, gates=gates, res_scale=res)
    s, y = forward(x)
    check_forward(x, s, y)
    check_backward(x, s, backward(x, s))


@pytest.mark.parametrize("rows,gates", [(2, 2), (600, 2), (600, 3), (600, 100), (600, 200), (600, 300), (599, 599),
                                        (2400, 8), (5000, 1250), (5000, 2500), (1021, 1)])
def test_gates_over_any_number_of_rows(cuda, rows, gates):
    """A gate whose rows are cut between workers, gates of a few rows, one row each."""
    x = make(rows, 264, F16, 63, gates=gates, res_scale=264)
    s, y = forward(x)
    check_forward(x, s, y)
    check_backward(x, s, backward(x, s))


@pytest.mark.parametrize("rows,h,gates,res,pre", [(1800, 8192, 5, 8192, True), (1800, 8000, 450, 8000, False),
                                                  (300, 16384, 6, 1, True), (40, 32760, 8, 32760, True),
                                                  (700, 8200, 7, 8200, True), (500, 12296, 500, 1, False),
                                                  (333, 32768, 3, 32768, True)])
def test_wide_rows_share_gates(cuda, rows, h, gates, res, pre):
    """Gates that do not fit the ring beside the rows; rows of several blocks, more of them than fit the device at once."""
    x = make(rows, h, BF16, 69, pre=pre, gates=gates, res_scale=res)
    s, y = forward(x)
    check_forward(x, s, y)
    check_backward(x, s, backward(x, s))


@pytest.mark.parametrize("h", [65544, 1 << 20, 1 << 22])
def test_sums_over_any_width_keep_their_bits(cuda, h):
    """A row of one value, 1.9765625, whose square every fp32 addition rounds the same way from 1024 on: thousands of them
    one after the other are 2^-14 off, eight times what the bounds allow a sum over a row."""
    x = make(2, h, BF16, 70, gates=0, res_scale=0)
    x["u"].fill_(1.9765625)
    s, y = forward(x)
    check_forward(x, s, y)
    check_backward(x, s, backward(x, s))
    s.fill_(1.9765625)
    check_backward(x, s, backward(x, s))


def test_benchmark_size(cuda):
    x = make(8192, 4096, BF16, 64, gates=8, res_scale=1)
    s, y = forward(x)
    check_forward(x, s, y)
    check_backward(x, s, backward(x, s))


@pytest.mark.parametrize("rows,h", [(257, 512), (40, 4096), (3, 24576)])
def test_outputs_may_replace_inputs(cuda, rows, h):
    x = make(rows, h, BF16, 65, gates=1, res_scale=h)
    s, y = forward(x)
    out = backward(x, s)
    z = {k: v.clone() if v is not None else None for k, v in x.items()}
    s2, y2 = forward(z, s=z["residual"], y=z["u"])
    assert torch.equal(s, s2) and torch.equal(y, y2)
    for name in ("u", "dy"):
        z = {k: v.clone() if v is not None else None for k, v in x.items()}
        out2 = backward(z, s, du=z[name], dresidual=z["ds"])
        for k in out:
            assert torch.equal(out[k], out2[k]), (name, k)


@pytest.mark.parametrize("rows,h", [(37, 512), (700, 4096), (3, 24576)])
def test_same_bits_on_every_call(cuda, rows, h):
    x = make(rows, h, BF16, 66, gates=1, res_scale=1)
    s, _ = forward(x)
    first = backward(x, s)
    for _ in range(3):
        again = backward(x, s)
        for k in first:
            assert torch.equal(first[k], again[k]), k


def test_a_row_only_touches_itself(cuda):
    """A row of NaN, of infinities, of zeros, of the smallest and of large values leaves the other rows' bits alone."""
    x = make(24, 1024, BF16, 67, gates=24)
    s, y = forward(x)
    out = backward(x, s)
    z = {k: v.clone() if v is not None else None for k, v in x.items()}
    for row, v in ((3, float("nan")), (7, float("inf")), (11, 0.0), (13, 1e-30), (17, 1e18)):
        z["u"][row], z["residual"][row] = v, v
    s2, y2 = forward(z)
    out2 = backward(z, s2)
    keep = [r for r in range(24) if r not in (3, 7, 11, 13, 17)]
    for a, b in ((s, s2), (y, y2), (out["du"], out2["du"]), (out["dresidual"], out2["dresidual"]), (out["dgate"], out2["dgate"])):
        assert torch.equal(a[keep], b[keep])
    assert torch.isnan(s2[3].float()).all() and torch.isnan(y2[3].float()).all()
    assert (s2[11] == 0).all() and (y2[11] == 0).all()
    assert torch.isfinite(out2["du"][[11, 13]].float()).all()


@pytest.mark.parametrize("eps", [1e-5, 1e-12, 1.0])
def test_zero_rows_and_eps(cuda, eps):
    x = make(9, 256, F16, 68, gates=3, res_scale=1)
    x["u"][4] = 0
    x["residual"][4] = 0
    x["residual"][5] = 0
    s, y = forward(x, eps=eps)
    check_forward(x, s, y, eps)
    if eps > 1e-8:                  # below that fp16 gradients of an all-zero row exceed 65504
        check_backward(x, s, backward(x, s, eps=eps), eps)


def test_no_rows(cuda):
    import PeakGemm

    e = torch.empty(0, 64, dtype=BF16, device="cuda")
    g = torch.ones(64, device="cuda")
    PeakGemm.rms_norm_residual_fwd(e, e, e, e, gamma_post=g, gamma_pre=g)
    a, b, c = (torch.full((n,), 7.0, device="cuda") for n in (64, 64, 1))
    PeakGemm.rms_norm_residual_bwd(e, e, e, e, e, e, residual=e, gamma_post=g, gamma_pre=g,
                                   res_scale=torch.ones(1, device="cuda"), dgamma_post=a, dgamma_pre=b, dres_scale=c)
    torch.cuda.synchronize()
    assert (a == 0).all() and (b == 0).all() and (c == 0).all()


def test_operators_refuse(cuda):
    import PeakGemm

    x = make(6, 64, BF16, 75, gates=3, res_scale=64)
    u, p = x["u"], params(x)
    new = lambda: torch.empty_like(u)      # noqa: E731
    f = dict(s=new(), y=new(), u=u, residual=x["residual"])
    PeakGemm.rms_norm_residual_fwd(**f, **p)
    for key, t in (("s", u[:5]), ("s", u.half()), ("residual", u.view(2, 3, 64)), ("residual", u.cpu()), ("y", u[:, :32]),
                   ("gamma_post", p["gamma_post"][:32]), ("gamma_post", p["gamma_post"].to(BF16)), ("gate", u[:4]),
                   ("gate", x["gate"].half()), ("gate", x["gate"][:, :32]), ("res_scale", p["gamma_post"][:8]),
                   ("res_scale", x["res_scale"].view(1, 64)), ("gamma_pre", p["gamma_pre"].cpu())):
        with pytest.raises((RuntimeError, NotImplementedError)):
            PeakGemm.rms_norm_residual_fwd(**{**f, **p, key: t})
    with pytest.raises(AssertionError):
        PeakGemm.rms_norm_residual_fwd(**{**f, **p, "y": None})
    g = dict(du=new(), dresidual=new(), dy=x["dy"], ds=x["ds"], s=f["s"], u=u, residual=x["residual"], dgate=x["gate"].clone())
    PeakGemm.rms_norm_residual_bwd(**g, **p)
    for key, t in (("du", u.float()), ("dresidual", u[:5]), ("dy", None), ("s", None), ("u", None), ("dgate", u[:1]),
                   ("gate", None), ("dgamma_post", p["gamma_post"][:8]), ("dres_scale", p["gamma_post"][:1]),
                   ("dgamma_pre", p["gamma_pre"].to(BF16)), ("ds", u.t())):
        with pytest.raises((RuntimeError, NotImplementedError, AssertionError)):
            PeakGemm.rms_norm_residual_bwd(**{**g, **p, key: t})
    with pytest.raises(RuntimeError):
        PeakGemm.rms_norm_residual_bwd(new(), new(), None, None, f["s"], u)                  # nothing comes in
    with pytest.raises(RuntimeError):
        PeakGemm.rms_norm_residual_bwd(new(), new(), None, x["ds"], f["s"], u, dgate=u)      # the gradient of nothing
    torch.cuda.synchronize()


def test_only_the_wanted_gradients(cuda):
    """ds or dy missing, sums not asked for, inputs that are then not needed."""
    import PeakGemm

    x = make(70, 768, BF16, 69, gates=2, res_scale=768)
    s, _ = forward(x)
    full = backward(x, s)
    du, dr = torch.empty_like(x["u"]), torch.empty_like(x["u"])
    PeakGemm.rms_norm_residual_bwd(du, dr, x["dy"], x["ds"], s, x["u"], **params(x))
    assert torch.equal(du, full["du"]) and torch.equal(dr, full["dresidual"])
    y = dict(x, ds=None)
    check_backward(y, s, backward(y, s))
    # without norms and without the gate's gradient neither s nor u is needed
    PeakGemm.rms_norm_residual_bwd(du, dr, None, x["ds"], None, None, gate=x["gate"])
    g = x["gate"].double().repeat_interleave(35, 0)
    assert torch.equal(dr, x["ds"]) and torch.equal(du, (g * x["ds"].double()).to(BF16))


def test_gradients_against_differences(cuda):
    """Directional derivatives of the float64 definition by central differences.  The kernel's gradients start from s as
    stored (rounded to 16 bits) and are rounded themselves: each of the three roundings moves a gradient element by at
    most 2^-9 of itself (fp16 2^-12, taken here), the norm's Jacobian passes a relative change of s on at most threefold
    (shat, the mean and rstd), so a derivative of sum |g v| is within 8 * 2^-11 of sum |g v|."""
    x = make(12, 192, F16, 70, gates=4, res_scale=192)
    s, _ = forward(x)
    out = backward(x, s)
    d = {k: v.double() for k, v in x.items()}

    def loss(z):
        a, b, _, _ = oracle.rmsnorm_residual_fwd(z["u"], z["residual"], *(z[k] for k in PARAMS))
        return (a * d["ds"]).sum() + (b * d["dy"]).sum()

    g = torch.Generator().manual_seed(71)
    for name in ("u", "residual") + PARAMS:
        v = torch.randn(x[name].shape, generator=g).cuda().double()
        h = 1e-6
        diff = (loss({**d, name: d[name] + h * v}) - loss({**d, name: d[name] - h * v})) / (2 * h)
        got = out["d" + name].double()
        assert abs((got * v).sum() - diff) <= 2.0 ** -8 * (got * v).abs().sum() + 1e-6, name


def test_leading_dims_streams_and_graph_replay(cuda):
    """[batch, tokens, h] views, a stream that is not the default one, capture into a graph and replay on new values."""
    x = make(60, 512, BF16, 72, gates=4, res_scale=1)
    s, y = forward(x)
    out = backward(x, s)
    b = {k: v.view(4, 15, 512) if v is not None and v.dim() == 2 and v.shape[0] == 60 else v for k, v in x.items()}
    b["gate"] = x["gate"].view(4, 1, 512)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s3, y3 = forward(b)
        out3 = backward(b, s3)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(s3.view(60, 512), s) and torch.equal(y3.view(60, 512), y)
    for k in out:
        assert torch.equal(out3[k].reshape(out[k].shape), out[k]), k
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s4, y4 = torch.empty_like(s), torch.empty_like(y)
        forward(x, s4, y4)
        out4 = backward(x, s4, torch.empty_like(s), torch.empty_like(s))
    new = make(60, 512, BF16, 73, gates=4, res_scale=1)
    for k in x:
        x[k].copy_(new[k])
    graph.replay()
    torch.cuda.synchronize()
    s5, y5 = forward(new)
    out5 = backward(new, s5)
    assert torch.equal(s4, s5) and torch.equal(y4, y5)
    for k in out5:
        assert torch.equal(out4[k], out5[k]), k


def test_two_calls_at_once(cuda):
    """Backward passes on two streams, each with its own scratch."""
    xs = [make(2000, 1024, BF16, 74 + i, gates=8, res_scale=1) for i in range(2)]
    ss = [forward(x)[0] for x in xs]
    ref = [backward(x, s) for x, s in zip(xs, ss)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = []
    for i, st in enumerate(streams):
        with torch.cuda.stream(st):
            for _ in range(4):
                got.append((i, backward(xs[i], ss[i])))
    torch.cuda.synchronize()
    for i, o in got:
        for k in o:
            assert torch.equal(o[k], ref[i][k]), k
