"""The dense operators refuse tensors with a forward-mode tangent, which they
would drop, and take them where forward mode is off."""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("requires_grad", [False, True])
def test_tangents_are_refused(spmm_npu, requires_grad):
    def rand(*s):
        return torch.randn(*s, device="cuda").requires_grad_(requires_grad)

    x, w, b, m = rand(6, 16), rand(16), rand(16), rand(2, 16, 16)
    off = torch.tensor([0, 2, 6], dtype=torch.int32, device="cuda")
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        calls = [lambda: spmm_npu.layer_norm(dual(x), w, b), lambda: spmm_npu.layer_norm(x, dual(w), b),
                 lambda: spmm_npu.layer_norm(x, None, dual(b)), lambda: spmm_npu.grouped_matmul(dual(x), m, off),
                 lambda: spmm_npu.grouped_matmul(x, dual(m), off)]
        if not requires_grad:
            calls.append(lambda: spmm_npu.orthogonalize(dual(m)))
        for call in calls:
            with pytest.raises(RuntimeError, match="forward-mode derivatives are not supported"):
                call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            spmm_npu.orthogonalize(dual(m))


def test_tensors_without_a_tangent_pass(spmm_npu):
    x = torch.randn(6, 16, device="cuda")
    with forward_ad.dual_level():
        plain = spmm_npu.layer_norm(x)
        with forward_ad._set_fwd_grad_enabled(False):
            off = spmm_npu.layer_norm(forward_ad.make_dual(x, torch.ones_like(x)))
    assert torch.equal(plain, off)
