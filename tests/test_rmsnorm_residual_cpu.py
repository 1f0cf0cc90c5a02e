"""CPU: refusals of rms_norm_residual_fwd / _bwd before any CUDA call, their schemas, and the oracle's gradients."""
import pytest
import torch

import oracle

P = 4096          # a fake, aligned, never dereferenced address


def fwd(**kw):
    from peakgemm_b200 import capi

    a = dict(s=P, y=P, u=P, residual=P, gamma_post=P, gate=P, gate_rows=2, res_scale=P, res_scale_len=64, gamma_pre=P,
             rows=4, h=64, eps=1e-6, dtype=1, stream=None)
    a.update(kw)
    return capi.lib().pg_rmsnorm_residual_fwd(*a.values())


def bwd(**kw):
    from peakgemm_b200 import capi

    a = dict(du=P, dresidual=P, dgamma_post=P, dgate=P, dres_scale=P, dgamma_pre=P, dy=P, ds=P, s=P, u=P, residual=P,
             gamma_post=P, gate=P, gate_rows=2, res_scale=P, res_scale_len=64, gamma_pre=P, rows=4, h=64, eps=1e-6,
             dtype=1, workspace=P, workspace_bytes=1 << 30, stream=None)
    a.update(kw)
    return capi.lib().pg_rmsnorm_residual_bwd(*a.values())


@pytest.mark.parametrize("call", [fwd, bwd])
@pytest.mark.parametrize("kw,status", [
    (dict(rows=-1), 1), (dict(h=0), 1), (dict(dtype=2), 1), (dict(gate_rows=-1), 1),
    (dict(gate=None), 1), (dict(gate_rows=0), 1), (dict(gate_rows=3), 1),              # 3 does not divide 4
    (dict(res_scale=None), 1), (dict(res_scale_len=0), 1), (dict(res_scale_len=8), 1),  # neither 1 nor h
    (dict(h=60, res_scale_len=60), 3), (dict(rows=2 ** 31), 3),
    (dict(gamma_post=P + 4), 2), (dict(gate=P + 2), 2), (dict(res_scale=P + 8), 2), (dict(u=P + 2), 2),
    (dict(u=None), 1), (dict(gamma_pre=None), 1),
])
def test_shared_refusals(call, kw, status):
    assert call(**kw) == status


def test_refusals_of_each_direction():
    assert fwd(rows=0, s=None, u=None) == 0
    assert fwd(y=None) == 1 and fwd(s=None) == 1 and fwd(residual=None) == 1
    assert fwd(s=P + 8) == 2 and fwd(y=P + 8) == 2
    assert bwd(dy=None) == 1 and bwd(ds=None, dy=None, gamma_pre=None, dgamma_pre=None) == 1
    assert bwd(s=None) == 1 and bwd(residual=None) == 1 and bwd(workspace=None) == 1
    assert bwd(gamma_post=None) == 1                                  # dgamma_post without gamma_post
    assert bwd(gate=None, gate_rows=0) == 1 and bwd(res_scale=None, res_scale_len=0) == 1
    assert bwd(gamma_pre=None, dy=None) == 1                          # dgamma_pre without gamma_pre
    assert bwd(workspace=P + 16) == 2 and bwd(dgate=P + 2) == 2 and bwd(dres_scale=P + 4) == 2
    from peakgemm_b200 import capi

    for rows, h, gates in ((0, 64, 0), (4, 60, 0), (-1, 64, 0), (4, 64, -1), (2 ** 31, 64, 1)):
        assert capi.rmsnorm_residual_bwd_workspace_bytes(rows, h, gates) == 0


def test_operators_refuse_and_trace():
    from torch._subclasses.fake_tensor import FakeTensorMode

    import PeakGemm

    ops = torch.ops.PeakGemm
    assert "Tensor(a!) s, Tensor(b!)? y" in str(ops.rms_norm_residual_fwd.default._schema)
    assert ops.rms_norm_residual_bwd.default._schema.is_mutable
    x, g = torch.zeros(4, 64, dtype=torch.bfloat16), torch.ones(64)
    with pytest.raises((RuntimeError, NotImplementedError)):
        PeakGemm.rms_norm_residual_fwd(x, x.clone(), x, x, gamma_pre=g)              # no CPU path
    with pytest.raises(AssertionError):
        PeakGemm.rms_norm_residual_fwd(x, None, x, x, gamma_pre=g)                   # gamma_pre without y
    with pytest.raises(AssertionError):
        PeakGemm.rms_norm_residual_fwd(x.float(), None, x.float(), x.float())
    with FakeTensorMode():
        x, g = torch.empty(4, 8, 64, dtype=torch.bfloat16, device="cuda"), torch.empty(64, device="cuda")
        PeakGemm.rms_norm_residual_fwd(x.clone(), x.clone(), x, x, gamma_post=g, gamma_pre=g)
        PeakGemm.rms_norm_residual_bwd(x.clone(), x.clone(), x, x, x, x, gamma_post=g, gamma_pre=g, dgamma_post=g.clone())


@pytest.mark.parametrize("post,pre,gates,res", [(True, True, 3, 16), (True, True, 0, 1), (False, True, 6, 0), (True, False, 1, 16)])
def test_oracle_gradients_match_autograd(post, pre, gates, res):
    x = oracle.rmsnorm_residual_inputs(6, 16, torch.float16, 60, post=post, pre=pre, gates=gates, res_scale=res)
    names = [k for k in ("u", "residual", "gamma_post", "gate", "res_scale", "gamma_pre") if x[k] is not None]
    z = {k: x[k].double().requires_grad_(True) for k in names}
    p = {k: z.get(k) for k in ("gamma_post", "gate", "res_scale", "gamma_pre")}
    s, y, _, _ = oracle.rmsnorm_residual_fwd(z["u"], z["residual"], **p)
    loss = (s * x["ds"].double()).sum() + ((y * x["dy"].double()).sum() if pre else 0)
    loss.backward()
    out = oracle.rmsnorm_residual_bwd(x["dy"], x["ds"], s.detach(), x["u"], x["residual"],
                                      **{k: x[k] for k in ("gamma_post", "gate", "res_scale", "gamma_pre")})
    for k in names:
        torch.testing.assert_close(out["d" + k][0], z[k].grad, rtol=1e-10, atol=1e-12)
