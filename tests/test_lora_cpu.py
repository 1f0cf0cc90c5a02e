"""CPU: refusals of gemm_peak_lora before any CUDA call, its schema, and its oracle against a direct evaluation."""
import pytest
import torch

import oracle

P = 4096          # a fake, aligned, never dereferenced address


def call(**kw):
    from peakgemm_b200 import capi

    a = dict(d=P, a=P, b=P, m=64, n=64, k=64, lda=64, ldb=64, ldd=64, lora_a=P, lora_b=P, ids=P, adapters=4, rank=16,
             scale=P, row_scale=P, bias=P, residual=P, ldr=64, dtype=1, workspace=P, workspace_bytes=1 << 40, stream=None)
    a.update(kw)
    return capi.lib().pg_hgemm_lora(*a.values())


@pytest.mark.parametrize("kw,status", [
    (dict(m=0), 0), (dict(n=0), 0), (dict(m=-1), 1), (dict(adapters=-1), 1), (dict(dtype=7), 1), (dict(d=None), 1),
    (dict(a=None), 1), (dict(lda=32), 1), (dict(ldr=32), 1), (dict(lora_a=None), 1), (dict(lora_b=None), 1),
    (dict(ids=None), 1), (dict(rank=0), 1), (dict(workspace=None), 1), (dict(workspace_bytes=16), 4),
    (dict(k=0), 3), (dict(n=60, ldd=60), 3), (dict(k=60, lda=60), 3), (dict(ldd=68), 3), (dict(rank=12), 3),
    (dict(rank=520), 3), (dict(adapters=2 ** 27), 3), (dict(adapters=2 ** 25 + 1), 3), (dict(m=2 ** 31), 3),
    (dict(d=P + 2), 2), (dict(lora_a=P + 8), 2), (dict(lora_b=P + 8), 2), (dict(ids=P + 2), 2), (dict(scale=P + 2), 2),
    (dict(workspace=P + 128), 2), (dict(bias=P + 2), 2),
])
def test_refusals(kw, status):
    assert call(**kw) == status


def test_workspace_of_no_work():
    from peakgemm_b200 import capi

    for a in ((0, 64, 64, 4, 16), (64, 0, 64, 4, 16), (64, 64, 0, 4, 16), (64, 64, 64, 0, 16), (64, 64, 64, 4, 0),
              (64, 64, 64, 4, 1024), (-1, 64, 64, 4, 16)):
        assert capi.hgemm_lora_workspace_bytes(*a) == 0


def test_operator_refuses_and_traces():
    from torch._subclasses.fake_tensor import FakeTensorMode

    import PeakGemm

    op = torch.ops.PeakGemm.gemm_peak_lora.default
    assert "Tensor(a!) d" in str(op._schema) and op._schema.is_mutable
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)      # noqa: E731
    good = [bf(4, 16), bf(4, 8), bf(16, 8), bf(2, 8, 8), bf(2, 16, 8), torch.zeros(4, dtype=torch.int32)]
    with pytest.raises((RuntimeError, NotImplementedError)):
        PeakGemm.gemm_peak_lora(*good)                                                   # no CPU path
    with pytest.raises(AssertionError):
        PeakGemm.gemm_peak_lora(good[0], torch.zeros(4, 8), *good[2:])                   # float32
    with FakeTensorMode():
        e = lambda *s, **kw: torch.empty(*s, device="cuda", **kw)      # noqa: E731
        f = dict(dtype=torch.bfloat16)
        PeakGemm.gemm_peak_lora(e(2, 2, 16, **f), e(2, 2, 8, **f), e(16, 8, **f), e(2, 8, 8, **f), e(2, 16, 8, **f),
                                e(2, 2, dtype=torch.int32), scale=e(2), row_scale=e(2, 2), residual=e(2, 2, 16, **f))


def test_oracle_is_the_definition():
    x = oracle.gemm_lora_inputs(9, 24, 16, 3, 8, torch.float16, 80)
    t = oracle.gemm_lora_terms(9, 24, torch.float16, 81)
    x["ids"][:3] = torch.tensor([0, 3, -1])
    d, bound = oracle.gemm_lora(**x, **t)
    for i in range(9):
        y = x["b"].double() @ x["a"][i].double()
        if 0 <= x["ids"][i] < 3:
            a = int(x["ids"][i])
            y = y + x["scale"][a].double() * (x["lora_b"][a].double() @ (x["lora_a"][a].double() @ x["a"][i].double()))
        y = t["row_scale"][i].double() * y + t["bias"].double() + t["residual"][i].double()
        torch.testing.assert_close(d[i], y, rtol=1e-12, atol=1e-12)
    assert (bound > 0).all()
