"""Where clipping reads and writes gradients and results of every pair of layouts, without a GPU: the two launches, which take memory as it lies, are stood in for."""
import itertools

import pytest
import torch

import turbodeberta_amd.ops.grad_norm as G

LAYOUTS = {
    "contiguous": lambda *s: torch.zeros(s),
    "transposed": lambda *s: torch.zeros(s[::-1]).permute(*range(len(s))[::-1]),
    "halfway": lambda *s: torch.zeros(s[:-2] + (s[-1], s[-2])).transpose(-1, -2),
    "gapped": lambda *s: torch.zeros(s[:-1] + (2 * s[-1],))[..., ::2],
    "gapped transposed": lambda *s: torch.zeros(s[::-1][:-1] + (2 * s[0],))[..., ::2].permute(*range(len(s))[::-1]),
    "padded rows": lambda *s: torch.zeros(s[:-1] + (s[-1] + 3,))[..., 1:1 + s[-1]],
}


def _memory(t):
    """What the kernels see: values from the first address on."""
    return torch.as_strided(t, (t.numel(),), (1,), t.storage_offset())


@pytest.fixture
def launches(monkeypatch):
    def norm(flat, kind):
        for t in flat:
            assert torch.ops.aten.is_non_overlapping_and_dense(t)
        return [_memory(t).clone() for t in flat], torch.tensor(1.0), None

    def clip(a, out, max_norm, dev):
        for o, values in zip(out, a):
            assert torch.ops.aten.is_non_overlapping_and_dense(o)
            _memory(o).copy_(values * 0.5)
    monkeypatch.setattr(G, "_norm", norm)
    monkeypatch.setattr(G, "_clip", clip)


@pytest.mark.parametrize("shape", [(5, 3), (2, 3, 4, 5), (4, 1), (1, 6)])
def test_pairs_of_layouts(shape, launches):
    for a, b in itertools.product(LAYOUTS, LAYOUTS):
        t, o = LAYOUTS[a](*shape), LAYOUTS[b](*shape)
        t.copy_(torch.arange(1.0, t.numel() + 1).view(shape))
        kept = t.clone()
        G._scaled([t], [o], 0.5, 2, False)
        assert torch.equal(o, kept * 0.5) and torch.equal(t, kept), (a, b)


@pytest.mark.parametrize("layout", LAYOUTS)
def test_in_place(layout, launches):
    t = LAYOUTS[layout](5, 3)
    t.copy_(torch.arange(15.0).view(5, 3))
    kept, version = t.clone(), t._version
    G._scaled([t], [t], 0.5, 2, False)
    assert torch.equal(t, kept * 0.5) and t._version > version


def test_a_gradient_into_its_own_transpose(launches):
    """Both views of one memory, where the values move."""
    base = torch.arange(16.0).view(4, 4)
    kept = base.clone()
    G._scaled([base.t()], [base], 0.5, 2, False)
    assert torch.equal(base, kept.t() * 0.5)
