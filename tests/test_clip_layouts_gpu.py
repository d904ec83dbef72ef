"""Clipping of gradients into results of other layouts, on both host paths."""
import itertools

import pytest
import torch

from test_grad_norm_gpu import TYPES, _check_clipped, _check_norm, _norm64, _rand, path      # noqa: F401
from turbodeberta_amd.ops.grad_norm import clip_grads

pytestmark = pytest.mark.gpu

LAYOUTS = {
    "contiguous": lambda t: t.contiguous(),
    "channels_last": lambda t: t.to(memory_format=torch.channels_last),
    "transposed": lambda t: t.permute(3, 2, 1, 0).contiguous().permute(3, 2, 1, 0),
    "halfway": lambda t: t.transpose(2, 3).contiguous().transpose(2, 3),
    "gapped": lambda t: torch.stack([t, t], -1)[..., 0],
    "padded rows": lambda t: torch.nn.functional.pad(t, (1, 2))[..., 1:-2],
}


@pytest.mark.parametrize("to", TYPES)
@pytest.mark.parametrize("dtype", TYPES)
def test_pairs_of_layouts(dtype, to, path):       # noqa: F811
    """Each pair by itself and all of them in one call; the values are all different."""
    values = _rand(1, 6, 5, 4, 7, dtype=dtype)
    pairs = list(itertools.product(LAYOUTS.values(), LAYOUTS.values()))
    grads = [a(values) for a, _ in pairs]
    nan = torch.full((6, 5, 4, 7), torch.nan, dtype=to, device="cuda")
    for some in [[n] for n in range(len(pairs))] + [range(len(pairs))]:
        mine = [grads[n] for n in some]
        norm = _norm64(mine, 2.0)
        out = [pairs[n][1](nan.clone()) for n in some]
        got, same = clip_grads(mine, 0.25 * norm, out=out)
        _check_norm(got, mine, 2.0)
        assert all(a is b for a, b in zip(same, out))
        _check_clipped(out, mine, norm, 0.25 * norm)
        assert all(torch.equal(g, values) for g in mine)


def test_a_weight_s_transpose(path):       # noqa: F811
    """As an optimizer keeps the master gradient of a layer whose weight it holds transposed."""
    grads = [_rand(2, 300, 70, dtype=torch.bfloat16), _rand(3, 70, dtype=torch.bfloat16)]
    norm = _norm64(grads, 2.0)
    out = [torch.empty(70, 300, device="cuda").t(), torch.empty(70, device="cuda")]
    clip_grads(grads, 0.5 * norm, out=out)
    _check_clipped(out, grads, norm, 0.5 * norm)
