"""Calls of the operators over logits at the limits of what they take: no rows."""
import pytest
import torch

from service_account_auth_improvements_amd import ops


def _no_rows(device, V, lse):
    x = torch.zeros(0, V, dtype=torch.bfloat16, device=device)
    ids, z = torch.zeros(0, 3, dtype=torch.long, device=device), torch.zeros(0, 3, device=device)
    L = torch.zeros(0, device=device) if lse else None
    loss, d = ops.distill_topk_fused(x, ids, z, 1.0, 1.0, L)
    assert loss.shape == (0,) and d.shape == (0, V)
    st = ops.distill_topk_stats(x, ids, z, 1.0, L)
    assert st.shape[0] == 0
    loss, d = ops.distill_topk_grad(x, ids, z, ops.distill_topk_join(st[None]), 1.0, 1.0, L)
    assert loss.shape == (0,) and d.shape == (0, V)
    xv = x.clone().requires_grad_()
    (d,) = torch.autograd.grad(ops.distill_topk(xv, ids, z, 1.0, L), xv, torch.zeros(0, device=device))
    assert d.shape == (0, V)
    xv, tok = x.clone().requires_grad_(), torch.zeros(0, dtype=torch.long, device=device)
    logp, ent, top, tlp = ops.token_logprobs(xv, tok, 1.0, min(2, V))
    (d,) = torch.autograd.grad([logp, ent], xv, [torch.zeros(0, device=device)] * 2)
    assert d.shape == (0, V) and top.shape == tlp.shape == (0, min(2, V))


@pytest.mark.parametrize("lse", [False, True])
@pytest.mark.parametrize("V", [1, 100])
def test_no_rows(V, lse):
    _no_rows("cpu", V, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("lse", [False, True])
@pytest.mark.parametrize("V", [1, 100, 300001])
def test_no_rows_gpu(V, lse):
    _no_rows("cuda:0", V, lse)
