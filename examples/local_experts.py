"""Local linear experts gated by a fitted mixture.

    python examples/local_experts.py

A Gaussian mixture is fitted to the inputs; every row goes to its two most
responsible components, each of which has a linear map of its own, and the two
results are added up by responsibility.  The maps (and the scale the rows are
brought to first) are trained by gradient descent, then the layer answers single
rows as a server would.
"""

import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import gmmxx_amd  # noqa: E402


class LocalExperts(torch.nn.Module):
    """norm -> mixture's responsibilities -> experts -> sum."""

    def __init__(self, mixture, width, outputs, top_k=2, dtype=torch.float32):
        super().__init__()
        device, experts = mixture.means_.device, mixture.means_.shape[0]
        self.mixture, self.top_k = mixture, top_k
        self.scale = torch.nn.Parameter(torch.ones(width, device=device, dtype=dtype))
        self.shift = torch.nn.Parameter(torch.zeros(width, device=device, dtype=dtype))
        self.maps = torch.nn.Parameter(torch.zeros(experts, width, outputs, device=device, dtype=dtype))
        self.offsets = torch.nn.Parameter(torch.zeros(experts, outputs, device=device, dtype=dtype))

    def forward(self, x):
        # log(0) = -inf: a component without responsibility is no candidate
        scores = torch.log(self.mixture.predict_proba(x))
        routing = gmmxx_amd.route_rows(scores, self.top_k)
        h = gmmxx_amd.layer_norm(x.to(self.scale.dtype), self.scale, self.shift)
        return gmmxx_amd.combine_rows(gmmxx_amd.grouped_matmul(h, self.maps, routing, bias=self.offsets), routing)


def make_data(rows, width, outputs, clusters, device, seed=0):
    """Clustered rows, and a target that is another linear map of the normalised row in every cluster."""
    g = torch.Generator().manual_seed(seed)
    centers = 4.0 * torch.randn((clusters, width), generator=g)
    maps = torch.randn((clusters, width, outputs), generator=g) / width ** 0.5
    label = torch.randint(0, clusters, (rows,), generator=g)
    x = centers[label] + torch.randn((rows, width), generator=g)
    h = torch.nn.functional.layer_norm(x, (width,))
    y = torch.matmul(h[:, None, :], maps[label])[:, 0]
    return x.to(device), y.to(device)


def run(rows=20_000, width=32, outputs=16, clusters=12, steps=200, device="cuda:0", dtype=torch.float32):
    """Trains the layer; returns the mean squared errors and the trained layer."""
    x, y = make_data(rows, width, outputs, clusters, device)
    mixture = gmmxx_amd.GMMXX(n_components=clusters, covariance_type="diag", max_iter=20, device=device).fit(x)
    layer = LocalExperts(mixture, width, outputs, dtype=dtype)
    optimiser = torch.optim.Adam(layer.parameters(), lr=2e-2)
    errors = []
    for _ in range(steps):
        optimiser.zero_grad()
        error = (layer(x).float() - y).square().mean()
        error.backward()
        optimiser.step()
        errors.append(error.detach())
    return [float(e) for e in errors], layer, x


def main():
    errors, layer, x = run()
    print(f"mean squared error {errors[0]:.4f} -> {errors[-1]:.4f} in {len(errors)} steps")
    with torch.no_grad():
        one = layer(x[:1])
    print("one row:", [round(v, 3) for v in one[0, :4].tolist()], "...")


if __name__ == "__main__":
    main()
