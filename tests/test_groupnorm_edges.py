"""Group norm with very many groups in all.  References and tolerances are those of test_norm_attention."""
import pytest
import torch

from comfyui_propainter_nodes_amd import ops
from test_norm_attention import F16, F32, U, _groupnorm_case


def test_more_groups_than_waves_of_the_finishing_launch(backend):
    """140 images of 64 groups: the launch between the sums and the values goes over them more than once."""
    _groupnorm_case(backend, F32, (140, 3, 1, 64), 64, "none")
    _groupnorm_case(backend, F16, (140, 3, 1, 64), 64, "silu", skip=True)


@pytest.mark.gpu
def test_groups_past_the_size_of_a_launch(hip_lib):
    """2^26 groups in all: a wave for each would be more threads than a launch holds."""
    n, c = (1 << 20) + 5, 64
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(8)
    x = torch.randn(n, 2, 1, c, device=dev, generator=g).to(F16)
    y = torch.full_like(x, 7.0)
    ops.groupnorm(x, y, c, eps=1e-2)
    # a group is two values a, b: mean (a + b) / 2, standard deviation |a - b| / 2
    half = (x[:, 0].float() - x[:, 1].float()) / 2
    want = half / (half * half + 1e-2).sqrt()
    for i, sign in ((0, 1.0), (1, -1.0)):
        tol = 16 * 2.0 ** -24 + U[F16] * want.abs() + 2.0 ** -25
        assert bool(((y[:, i, 0].float() - sign * want[:, 0]).abs() <= tol[:, 0]).all())
