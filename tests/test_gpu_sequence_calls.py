"""The sequence operators (genie/sequence.py) in the surroundings a training or serving program puts them into, on the GPU: hooks on saved tensors, empty batches, the C entries'
own workspaces, versions of tensors that are updated in place, values that are not finite.  Numerics: tests/test_gpu_sequence.py."""
import pytest
import torch

import util  # noqa: F401  (paths)

pytestmark = pytest.mark.gpu


def _gf():
    from genie import functional
    return functional


def _randn(*shape, seed, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator(device='cuda').manual_seed(seed), device='cuda') * scale).to(torch.bfloat16)


def _cu(lens):
    return torch.tensor([0] + list(lens), dtype=torch.int32, device='cuda').cumsum(0).to(torch.int32)


def _apart(t):
    """The same values, nothing of them contiguous."""
    wide = torch.empty((*t.shape, 2), dtype=t.dtype, device=t.device)
    wide[..., 0] = t
    return wide[..., 0]


def _shifted(t):
    """The same values at an address off 16 bytes."""
    flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape)
    return flat.copy_(t)


@pytest.mark.parametrize('hook', ['on the host', 'apart', 'shifted'])
@pytest.mark.parametrize('lens', [[20, 1, 50], [400, 300]], ids=str)
def test_gradients_after_a_round_trip_of_the_saved_tensors(lens, hook):
    """Slices of a fused projection come back dense, in a layout of their own or off 16 bytes: the gradients are those of the plain call, to the bit."""
    gf, rows, h, d = _gf(), sum(lens), 4, 64
    fused = _randn(rows, 3 * h, d, seed=1).requires_grad_(True)
    g, ld, cu = _randn(rows, h, d, seed=2), -torch.linspace(0.01, 0.5, h, device='cuda'), _cu(lens)
    s0 = torch.randn((len(lens), h, d, d), generator=torch.Generator(device='cuda').manual_seed(3), device='cuda')

    def context():
        if hook == 'on the host':
            return torch.autograd.graph.save_on_cpu()
        return torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), _apart if hook == 'apart' else _shifted)

    for call in (lambda q, k, v: gf.packed_attention(q, k[:, :2], v[:, :2], cu), lambda q, k, v: gf.decay_attention(q, k, v, ld, cu),
                 lambda q, k, v: gf.decay_attention(q, k, v, ld, cu, initial_state=s0)):
        want = torch.autograd.grad(call(*fused.split(h, 1)), fused, g)[0]
        with context():
            out = call(*fused.split(h, 1))
        assert torch.equal(torch.autograd.grad(out, fused, g)[0], want)
