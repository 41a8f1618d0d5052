"""Arguments of the layer's Python functions that fit each other but no kernel: refused by
name before any call of the library.  Host tensors stand in for the GPU's here."""

import pytest
import torch

import gmmxx_amd
from gmmxx_amd import experts


@pytest.fixture(autouse=True)
def host_tensors(monkeypatch):
    monkeypatch.setattr(experts, "_tensor", lambda t, name: t)


def routing(n, k, e=3):
    ints = dict(dtype=torch.int32)
    return gmmxx_amd.Routing(torch.zeros((n, k), **ints), torch.zeros(n, k), torch.zeros(e + 1, **ints),
                             torch.zeros(n * k, **ints), torch.zeros((n, k), **ints))


@pytest.mark.parametrize("n", [0, 3])
@pytest.mark.parametrize("k", [0, experts.MAX_TOP_K + 1])
def test_top_k_out_of_range(n, k):
    """Without choices there is nothing to add up: a forward pass that answered had a backward pass that failed."""
    x = torch.zeros((n, 4), requires_grad=True)
    with pytest.raises(ValueError, match="top_k"):
        gmmxx_amd.grouped_matmul(x, torch.zeros(3, 4, 5), routing(n, k))
    with pytest.raises(ValueError, match="top_k"):
        gmmxx_amd.combine_rows(torch.zeros(n * k, 5), routing(n, k))


WIDE = (1 << 22) + 1


@pytest.mark.parametrize("rows", [0, 2])
@pytest.mark.parametrize("which", ["D", "F"])
def test_matrices_too_wide(rows, which):
    """The library's limit, by the argument's own name."""
    x = torch.zeros(1, 1).expand(rows, WIDE if which == "D" else 4)
    w = torch.zeros(1, 1, 1).expand(3, x.shape[1], WIDE if which == "F" else 4)
    with pytest.raises(ValueError, match="4194304"):
        gmmxx_amd.grouped_matmul(x, w, torch.zeros(4, dtype=torch.int32))
    with pytest.raises(ValueError, match="4194304"):
        gmmxx_amd.combine_rows(torch.zeros(1, 1).expand(rows, WIDE), routing(rows, 1))
