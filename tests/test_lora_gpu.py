"""GPU: gemm_peak_lora against its definition in float64.

Bound (oracle.gemm_lora, derived before any run): every element is the 16-bit rounding (half a step) of a number within
the fp32 sums' slack of the exact value, the down projection's result rounded once to 16 bits.  The reference project
has no adapters (parity unpinned).
"""
import pytest
import torch

import oracle
from tests import helpers

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def make(m, n, k, adapters, rank, dtype, seed, ids="mixed", terms=False):
    x = oracle.gemm_lora_inputs(m, n, k, adapters, rank, dtype, seed, ids)
    if terms:
        x.update(oracle.gemm_lora_terms(m, n, dtype, seed + 1))
    return {key: v.cuda() for key, v in x.items()}


def call(x, d=None):
    import PeakGemm

    m, n = x["a"].shape[0], x["b"].shape[0]
    d = helpers.garbage_like((m, n), x["a"].dtype, "cuda") if d is None else d
    kw = {key: x[key] for key in ("scale", "row_scale", "bias", "residual") if key in x}
    PeakGemm.gemm_peak_lora(d, x["a"], x["b"], x["lora_a"], x["lora_b"], x["ids"], **kw)
    return d


def check(x, d, rows=slice(None)):
    from peakgemm_b200 import capi

    torch.cuda.synchronize()
    assert capi.device_status() == 0, "a kernel abandoned a bounded wait"
    y = {key: (v[rows] if key in ("a", "ids", "row_scale", "residual") else v) for key, v in x.items()}
    ref, bound = oracle.gemm_lora(**y)
    d = d[rows]
    assert torch.isfinite(d.float()).all()
    ok = helpers.elementwise_ok(d, ref.float(), (bound + 2.0 ** -24 * ref.abs()).float())
    assert ok.all(), f"{int((~ok).sum())} of {ok.numel()} elements off, worst {(d.double() - ref).abs()[~ok].max().item():.3g}"


# one token to several tiles of every kernel the product may take, sizes around the tiles' edges
ROWS = [1, 2, 15, 16, 17, 32, 33, 64, 65, 100, 128, 129, 200, 256, 257, 300, 513, 1003]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("m", ROWS)
def test_rows(cuda, m, dtype):
    for n, k, rank, ids in ((520, 264, 16, "mixed"), (264, 1032, 24, "runs")):
        x = make(m, n, k, 7, rank, dtype, 81, ids, terms=m % 2 == 0)
        check(x, call(x))


@pytest.mark.parametrize("rank", [8, 16, 24, 40, 56, 64, 72, 128, 200, 512])
@pytest.mark.parametrize("m", [3, 64, 130, 700])
def test_ranks(cuda, m, rank):
    x = make(m, 392, 520, 5, rank, BF16, 82)
    check(x, call(x))


@pytest.mark.parametrize("m", [1, 5, 64, 128, 300, 600])
@pytest.mark.parametrize("ids", ["mixed", "runs", "one", "none"])
@pytest.mark.parametrize("adapters", [1, 3, 64, 200])
def test_which_rows_use_which_adapter(cuda, m, ids, adapters):
    x = make(m, 264, 136, adapters, 8, F16, 83, ids)
    check(x, call(x))


@pytest.mark.parametrize("n,k", [(8, 8), (8, 4096), (4096, 8), (136, 72), (4104, 5128)])
@pytest.mark.parametrize("m", [1, 40, 130, 520])
def test_narrow_and_odd_matrices(cuda, m, n, k):
    x = make(m, n, k, 4, 16, BF16, 84, terms=True)
    check(x, call(x))


# sizes at which the product takes each of its kernels (few tokens, split over k, pairs, pairs with two row blocks)
@pytest.mark.parametrize("m,n,k", [(16, 4096, 4096), (40, 14336, 2048), (128, 4096, 4096), (100, 2048, 8192),
                                   (256, 4096, 4096), (512, 4096, 4096), (1024, 4096, 1024), (4096, 4096, 512),
                                   (8192, 3328, 256), (8000, 3304, 136)])
@pytest.mark.parametrize("ids", ["mixed", "runs"])
def test_large(cuda, m, n, k, ids):
    x = make(m, n, k, 12, 16, BF16, 85, ids, terms=True)
    check(x, call(x))


# few tokens with more rank elements than dot products are for, more tokens with a pool they are for
@pytest.mark.parametrize("m,k,adapters,rank", [(17, 8192, 3, 512), (40, 4104, 5, 512), (64, 8200, 9, 128), (1, 131080, 1, 512),
                                               (65, 1032, 20, 16), (130, 520, 64, 24), (513, 264, 17, 8)])
@pytest.mark.parametrize("ids", ["mixed", "runs"])
def test_both_down_projections(cuda, m, k, adapters, rank, ids):
    x = make(m, 264, k, adapters, rank, F16, 92, ids, terms=m % 2 == 0)
    check(x, call(x))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("m", [1, 17, 64, 100, 200, 300, 600])
@pytest.mark.parametrize("rank", [8, 16, 24, 32, 40, 72, 512])
def test_down_projection_keeps_its_bits(cuda, m, rank, dtype):
    """The down projection's sums go into the second product as two 16-bit terms, within (eps / 2)^2 of themselves, not as
    one.  Adapters that outweigh the product: there one term shows."""
    x = make(m, 392, 264, 5, rank, dtype, 97)
    x["b"] *= 2.0 ** -6
    d = call(x)
    torch.cuda.synchronize()
    ref, bound = oracle.gemm_lora(**x, v_terms=2)
    ok = helpers.elementwise_ok(d, ref.float(), (bound + 2.0 ** -24 * ref.abs()).float())
    assert ok.all(), f"{int((~ok).sum())} of {ok.numel()} elements off, worst {(d.double() - ref).abs()[~ok].max().item():.3g}"


@pytest.mark.parametrize("terms", ["scale", "row_scale", "bias", "residual", ""])
@pytest.mark.parametrize("m", [5, 130, 600])
def test_each_term_alone(cuda, m, terms):
    x = make(m, 264, 264, 4, 16, BF16, 86, terms=True)
    for key in ("scale", "row_scale", "bias", "residual"):
        if key != terms:
            del x[key]
    check(x, call(x))


@pytest.mark.parametrize("m", [1, 33, 130, 600])
def test_residual_may_be_the_output(cuda, m):
    x = make(m, 520, 264, 4, 16, BF16, 87, terms=True)
    d = x["residual"].clone()
    call(dict(x, residual=d), d)
    check(x, d)


@pytest.mark.parametrize("m", [6, 70, 300])
def test_ids_outside_the_pool_mean_none(cuda, m):
    x = make(m, 264, 264, 4, 16, F16, 88)
    x["ids"][:] = torch.tensor([0, 4, -1, 3, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32).repeat(m // 6 + 1)[:m].cuda()
    check(x, call(x))


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("m", [12, 70, 128, 300, 600])
def test_one_request_does_not_touch_another(cuda, m, value):
    """Infinities or NaN in an adapter that no row uses, in one that a single row uses, and in a row of the batch leave
    all other rows as exact as they are without them."""
    x = make(m, 392, 264, 6, 16, BF16, 89)
    x["ids"][x["ids"] >= 3] = 1
    x["ids"][4], x["ids"][9] = 3, 4
    x["lora_a"][5], x["lora_b"][5] = value, value            # no row uses it
    x["lora_b"][3, 100:140] = value
    x["lora_a"][4, 2] = value
    x["a"][7, 11] = value
    d = call(x)
    keep = [t for t in range(m) if t not in (4, 7, 9)]
    check({k: v for k, v in x.items()}, d, keep)
    assert not torch.isfinite(d[4, 100:140].float()).any() and torch.isfinite(d[4, :100].float()).all()
    assert not torch.isfinite(d[7].float()).any() and not torch.isfinite(d[9].float()).any()


@pytest.mark.parametrize("m", [12, 32, 64, 100, 300, 700])
def test_an_adapter_without_a_finite_value(cuda, m):
    """One request's adapter is NaN altogether, at a long k: the other rows stay exact, no wait runs out, and the call takes
    no longer than without it over 64 rows (some tens of microseconds), up to 64 rows about twice as long."""
    x = make(m, 1032, 8192, 6, 16, BF16, 98)
    x["ids"][x["ids"] == 2] = 1
    x["ids"][3] = 2
    call(x)
    x["lora_b"][2] = float("nan")
    x["lora_b"][5, ::7] = float("inf")
    x["a"][6] = float("nan")
    torch.cuda.synchronize()
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    d = call(x, torch.empty(m, 1032, dtype=BF16, device="cuda"))
    end.record()
    keep = [t for t in range(m) if t not in (3, 6) and x["ids"][t] != 5]
    check(x, d, keep)
    assert d[3].isnan().all() and d[6].isnan().all()
    assert start.elapsed_time(end) < 1.0


@pytest.mark.parametrize("m,n,k", [(8192, 3328, 256), (3000, 4096, 512), (2500, 8200, 136)])
@pytest.mark.parametrize("without", ["first", "last", "between"])
def test_tiles_without_adapters_beside_tiles_with(cuda, m, n, k, without):
    """Kernels that take several tiles one after the other: the first, the last or every other tile row has no adapter."""
    x = make(m, n, k, 5, 24, BF16, 100, "mixed")
    row = torch.arange(m, device="cuda")
    none = {"first": row < 5 * m // 8, "last": row >= 3 * m // 8, "between": row // 512 % 2 == 0}[without]
    x["ids"][none] = -1
    for _ in range(3):
        check(x, call(x))


@pytest.mark.parametrize("m,n,k,adapters,rank", [(8192, 3328, 256, 700, 8), (1100, 520, 264, 600, 40), (300, 264, 136, 1000, 16)])
def test_hundreds_of_adapters_in_a_tile(cuda, m, n, k, adapters, rank):
    x = make(m, n, k, adapters, rank, BF16, 99)
    check(x, call(x))


def test_scratch_does_not_grow_with_the_pool(cuda):
    """Twice V's bits for every row (rank 64: 256 bytes), and a few words for each adapter that the rows of a tile can use."""
    from peakgemm_b200 import capi

    for m, n, k in ((128, 4096, 4096), (1000, 4096, 4096), (4096, 14336, 4096), (32768, 4096, 4096)):
        for pool in (1, 512, 100000):
            table = (m // 128 + 4) * (min(pool, 512) + 4) * (4 + 512 // 8)
            assert 0 < capi.hgemm_lora_workspace_bytes(m, n, k, pool, 64) <= m * 64 * 4 + table + 512
    for m in (1, 16, 64):                       # the tokens of a small batch once for each adapter they can use
        assert capi.hgemm_lora_workspace_bytes(m, 4096, 4096, 100000, 64) <= 64 * 64 * 64 * 4 + 1024


def test_no_scratch_for_a_call_that_is_refused(cuda):
    """A rank or a matrix that is no multiple of 8, an index of 2^31 or more: pg_hgemm_lora refuses, and the query says 0."""
    from peakgemm_b200 import capi

    size = capi.hgemm_lora_workspace_bytes
    assert size(64, 64, 64, 4, 16) > 0
    for a in ((64, 64, 64, 4, 12), (64, 60, 64, 4, 16), (64, 64, 60, 4, 16), (64, 64, 64, 2 ** 27, 16), (64, 64, 64, 2 ** 25 + 1, 64),
              (2 ** 31, 64, 64, 4, 16), (64, 2 ** 31, 64, 4, 16), (64, 64, 2 ** 31, 4, 16)):
        assert size(*a) == 0, a


@pytest.mark.parametrize("m", [9, 130, 600])
def test_pitches_and_untouched_surroundings(cuda, m):
    """Matrices that are blocks of wider ones; columns beside the output and rows behind it stay as they were."""
    from peakgemm_b200 import capi

    n, k = 264, 200
    x = make(m, n, k, 4, 24, BF16, 90, terms=True)
    wide = {key: torch.full((x[key].shape[0] + 3, x[key].shape[1] + 40), 7.0, dtype=BF16, device="cuda") for key in ("a", "b", "residual")}
    for key in wide:
        wide[key][:x[key].shape[0], 16:16 + x[key].shape[1]] = x[key]
        x[key + "_w"] = wide[key][:x[key].shape[0], 16:16 + x[key].shape[1]]
    out = torch.full((m + 5, n + 48), 3.0, dtype=BF16, device="cuda")
    ws = torch.empty(capi.hgemm_lora_workspace_bytes(m, n, k, 4, 24), dtype=torch.uint8, device="cuda").fill_(255)
    capi.hgemm_lora(out[:m, 24:24 + n], x["a_w"], x["b_w"], x["lora_a"], x["lora_b"], x["ids"], ws, scale=x["scale"],
                    row_scale=x["row_scale"], bias=x["bias"], residual=x["residual_w"])
    x = {key: v for key, v in x.items() if not key.endswith("_w")}
    check(x, out[:m, 24:24 + n].contiguous())
    assert (out[m:] == 3).all() and (out[:, :24] == 3).all() and (out[:, 24 + n:] == 3).all()


@pytest.mark.parametrize("m", [3, 64, 128, 700])
def test_same_bits_on_every_call(cuda, m):
    x = make(m, 1032, 2048, 9, 16, BF16, 91)
    first = call(x)
    for _ in range(4):
        assert torch.equal(call(x), first)


def test_operator_refuses(cuda):
    import PeakGemm

    x = make(4, 16, 8, 2, 8, BF16, 130)
    good = [torch.empty(4, 16, dtype=BF16, device="cuda"), *(x[key] for key in ("a", "b", "lora_a", "lora_b", "ids"))]
    PeakGemm.gemm_peak_lora(*good)
    bf = lambda *s: torch.zeros(*s, dtype=BF16, device="cuda")      # noqa: E731
    for i, t in ((0, bf(5, 16)), (0, bf(4, 24)), (2, bf(16, 16)), (3, bf(2, 8, 16)), (3, x["lora_a"].half()), (4, bf(2, 16, 16)),
                 (4, bf(3, 16, 8)), (4, x["lora_b"].cpu()), (4, bf(2, 8, 16).mT), (5, x["ids"][:3]), (5, x["ids"].long())):
        with pytest.raises((RuntimeError, NotImplementedError)):
            PeakGemm.gemm_peak_lora(*good[:i], t, *good[i + 1:])
    for kw in (dict(scale=x["scale"][:1]), dict(scale=x["scale"].double()), dict(row_scale=x["scale"]), dict(bias=bf(8)),
               dict(residual=bf(4, 8))):
        with pytest.raises(RuntimeError):
            PeakGemm.gemm_peak_lora(*good, **kw)
    with pytest.raises(RuntimeError, match="UNSUPPORTED"):
        PeakGemm.gemm_peak_lora(*good[:3], bf(2, 12, 8), bf(2, 16, 12), x["ids"])             # rank % 8
    torch.cuda.synchronize()


def test_no_rows_no_adapters(cuda):
    import PeakGemm

    x = make(5, 64, 64, 2, 8, BF16, 92)
    e = {key: (v[:0] if key in ("a", "ids") else v) for key, v in x.items()}
    assert call(e).shape == (0, 64)
    none = dict(x, lora_a=x["lora_a"][:0], lora_b=x["lora_b"][:0], scale=x["scale"][:0])
    d, plain = call(none), torch.empty(5, 64, dtype=BF16, device="cuda")
    PeakGemm.gemm_peak_fused(plain, x["a"], x["b"])
    assert torch.equal(d, plain)


@pytest.mark.parametrize("m", [8, 128, 600])
def test_streams_and_graph_replay(cuda, m):
    """A stream that is not the default one; capture, then replay with other values and other ids."""
    x = make(m, 264, 520, 6, 16, BF16, 93, terms=True)
    ref = call(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        d = call(x)
    side.synchronize()
    assert torch.equal(d, ref)
    graph = torch.cuda.CUDAGraph()
    out = torch.empty_like(ref)
    with torch.cuda.graph(graph):
        call(x, out)
    for seed in (94, 95):
        new = make(m, 264, 520, 6, 16, BF16, seed, terms=True)
        for key in x:
            x[key].copy_(new[key])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call(new))


def test_back_to_back_calls_on_changing_inputs(cuda):
    """No call may read the scratch of the one before: the same buffers, values of very different scale."""
    xs = [make(48, 1024, 1024, 5, 16, BF16, 96 + i) for i in range(12)]
    for i, x in enumerate(xs):
        x["a"] *= 4.0 ** (i % 5)
    refs = []
    for x in xs:
        refs.append(call(x))
        torch.cuda.synchronize()
    for r, d in zip(refs, [call(x) for x in xs]):
        assert torch.equal(r, d)


def test_two_calls_at_once(cuda):
    xs = [make(600, 1032, 1024, 8, 16, BF16, 110 + i) for i in range(2)]
    refs = [call(x) for x in xs]
    torch.cuda.synchronize()
    got, streams = [], [torch.cuda.Stream() for _ in xs]
    for _ in range(6):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got.append((i, call(xs[i])))
    torch.cuda.synchronize()
    for i, d in got:
        assert torch.equal(d, refs[i])


@pytest.mark.parametrize("m", [1, 64, 300])
def test_a_block_with_adapters(cuda, m):
    """The operators as a network runs them: rstd, a projection with adapters over the raw stream, then the norm after
    the block, its gate, the residual and the next norm.  Each step against its own definition on the step's inputs."""
    import PeakGemm

    h = 512
    x = make(m, h, h, 6, 16, BF16, 120)
    t = {key: v.cuda() if v is not None else None
         for key, v in oracle.rmsnorm_residual_inputs(m, h, BF16, 121, gates=1, res_scale=1).items()}
    stream, gamma = t["residual"], t["gamma_pre"]
    w = PeakGemm.fold_gamma(x["b"], gamma)
    la = PeakGemm.fold_gamma(x["lora_a"].view(-1, h), gamma).view_as(x["lora_a"])
    rstd = torch.empty(m, device="cuda")
    torch.ops.PeakGemm.rms_norm_rstd(rstd, stream, 1e-6)
    u = torch.empty(m, h, dtype=BF16, device="cuda")
    PeakGemm.gemm_peak_lora(u, stream, w, la, x["lora_b"], x["ids"], scale=x["scale"], row_scale=rstd)
    s, y = torch.empty_like(u), torch.empty_like(u)
    terms = {key: t[key] for key in ("gamma_post", "gate", "res_scale", "gamma_pre")}
    PeakGemm.rms_norm_residual_fwd(s, y, u, stream, **terms)
    check(dict(a=stream, b=w, lora_a=la, lora_b=x["lora_b"], ids=x["ids"], scale=x["scale"], row_scale=rstd), u)
    # against the unfolded definition: folding rounds W and A once more (half a step each, on sums of h products)
    norm = stream.double() * torch.rsqrt(stream.double().pow(2).mean(-1, keepdim=True) + 1e-6) * gamma.double()
    ref, bound = oracle.gemm_lora(norm, x["b"].double(), x["lora_a"].double(), x["lora_b"].double(), x["ids"], x["scale"])
    slack = 2.0 ** -8 * (norm.abs() @ x["b"].double().abs().t()) + bound
    for i in range(6):
        k = (x["ids"] == i).nonzero()[:, 0]
        slack[k] += 2.0 ** -7 * float(x["scale"][i]) * (norm[k].abs() @ x["lora_a"][i].double().abs().t()) @ x["lora_b"][i].double().abs().t()
    assert ((u.double() - ref).abs() <= slack + 2.0 ** -8 * ref.abs() + 1e-6).all()
    rs, ry, es, ey = oracle.rmsnorm_residual_fwd(u, stream, **terms)
    assert helpers.elementwise_ok(s, rs.float(), (es + 2.0 ** -24 * rs.abs()).float()).all()
    assert helpers.elementwise_ok(y, ry.float(), (ey + 2.0 ** -24 * ry.abs()).float()).all()
