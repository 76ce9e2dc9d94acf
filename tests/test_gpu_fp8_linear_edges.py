"""More of the 8-bit linear layers on the GPU: calls that the documentation allows at the edges of what tests/test_gpu_fp8_linear.py
runs. Bounds as there."""
import pytest
import torch

from nanochat_amd import fp8_linear as fl
from tests.test_gpu_fp8_linear import bf, form, weight

pytestmark = pytest.mark.gpu


def at_the_end(scale, wider):
    """The same scales as the last columns of wider rows, at the very end of their storage."""
    rows, blocks = scale.shape
    pad = -(-blocks // 4) * 4
    whole = torch.zeros(rows, pad + wider, dtype=torch.uint8, device=scale.device)
    whole[:, wider:wider + blocks] = scale.contiguous().view(torch.uint8)
    return whole.view(fl.SCALE)[:, wider:wider + blocks]


@pytest.mark.parametrize("rows,n,k", [(8, 528, 2048), (70, 1296, 512), (600, 4112, 512), (4100, 4112, 1024)])
def test_scales_that_end_with_their_storage(device, rows, n, k):
    """Few results, small, half and full tiles."""
    gen = torch.Generator().manual_seed(rows + k)
    codes, scale, _ = form(gen, device, rows, k)
    w, _ = weight(gen, device, n, k)
    want = fl.fp8_matmul(codes, scale, w)
    for wider in (4, 48):
        assert torch.equal(fl.fp8_matmul(codes, at_the_end(scale, wider), fl.Fp8Weight(w.codes, at_the_end(w.scale, wider))), want)
    dy = bf(gen, rows, 144).to(device)
    assert torch.equal(fl.checkpoint_weight_grad(dy, codes, at_the_end(scale, 48)), fl.checkpoint_weight_grad(dy, codes, scale))


def test_buffers_of_layers_without_a_gradient(device):
    """Neither the input nor the weights require one: what the buffers are given is what a parameter would get."""
    gen = torch.Generator().manual_seed(20)
    x, dy = bf(gen, 70, 256).to(device), bf(gen, 70, 144).to(device)
    w, fc, proj = (torch.randn(*s, generator=gen).to(device) / 16 for s in ((144, 256), (640, 256), (144, 640)))
    buffers = [torch.zeros_like(t) for t in (w, fc, proj)]
    fl.checkpointed_linear(x, w, grad=buffers[0]).backward(dy)
    fl.checkpointed_mlp(x, fc, proj, fc_grad=buffers[1], proj_grad=buffers[2]).backward(dy)
    asked = [t.clone().requires_grad_() for t in (w, fc, proj)]
    fl.checkpointed_linear(x, asked[0]).backward(dy)
    fl.checkpointed_mlp(x, *asked[1:]).backward(dy)
    # the same sums, added to zeros
    assert all(torch.equal(b, t.grad) for b, t in zip(buffers, asked)) and all(t.grad is None for t in (w, fc, proj))
