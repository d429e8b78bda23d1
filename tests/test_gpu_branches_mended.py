"""Several continuations of one prompt: calls that once went wrong, and the ones beside them."""
import pytest
import torch

from hira_b200 import HiraCacheLayer, patch_attention
from test_patched_layers_host import D, HIDDEN, _Layer, _neighbours

pytestmark = pytest.mark.gpu


def _cache_of_one_layer():
    layer = HiraCacheLayer("cuda_only", 4, dict(num_levels=2, max_iterations=1, branching_factor=8), {})

    class One:
        def update(self, k, v, idx):
            return layer.update(k, v)
    return One()


@torch.no_grad()
@pytest.mark.parametrize("rotary", [D, 8])
@pytest.mark.parametrize("odd", ["", "table_halves"])
def test_interleaved_layers_rotate_as_their_own_forward_does(odd, rotary):
    """Tables by channel, and tables that hold a pair's value at i and i + R/2."""
    layer = _Layer(odd, pairs=_neighbours, rotary=rotary).cuda()
    model = torch.nn.ModuleList([layer])
    model.register_buffer("inv_freq", torch.ones(rotary // 2))
    n, gen = 20, torch.Generator().manual_seed(5)
    x = (torch.randn((1, n, HIDDEN), generator=gen) * 20).cuda()
    angle = torch.randn((1, n, rotary // 2), generator=gen).cuda() * 6
    angle = torch.cat([angle, angle], -1) if odd else angle.repeat_interleave(2, -1)
    mask = torch.full((1, 1, n, n), torch.finfo(torch.float32).min, device="cuda").triu(1)
    want = layer(x, (angle.cos(), angle.sin()), mask)[0]
    assert patch_attention(model, interleaved=True) == 1
    got = layer(x, position_embeddings=(angle.cos(), angle.sin()), past_key_values=_cache_of_one_layer())[0]
    torch.testing.assert_close(got, want, atol=1e-4, rtol=1e-3)
