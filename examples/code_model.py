"""What code comes next: a mixture's labels as tokens.

    python examples/code_model.py

A Gaussian mixture is fitted to rows that wander between clusters; each row's label is a
token.  A small model reads a token and answers with scores over the next one: an embedding,
a layer of experts with dropout around it, and a head.  It is trained on the log probabilities of the tokens that
came, with a little entropy kept; then it answers single tokens with the head in 8-bit integers.
"""

import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import gmmxx_amd  # noqa: E402


class CodeModel(torch.nn.Module):
    """token -> embedding -> norm -> experts, dropped and added -> norm -> scores of the next token."""

    def __init__(self, tokens, width=64, experts=4, top_k=2, dropout=0.1, dtype=torch.bfloat16, device="cuda:0", seed=0):
        super().__init__()
        g = torch.Generator().manual_seed(seed)

        def weight(*shape, scale):
            return torch.nn.Parameter((scale * torch.randn(shape, generator=g)).to(dtype).to(device))

        self.top_k, self.dropout, self.scale = top_k, dropout, width ** 0.5
        self.table = weight(tokens, width, scale=width ** -0.5)
        self.gate = weight(width, experts, scale=width ** -0.5)
        self.maps = weight(experts, width, width, scale=width ** -0.5)
        self.head = weight(tokens, width, scale=width ** -0.5)
        self.steps = torch.zeros(1, dtype=torch.int64, device=device)       # the dropout's seed

    def hidden(self, tokens):
        h = gmmxx_amd.embed_rows(self.table, tokens, scale=self.scale)
        x = gmmxx_amd.layer_norm(h)
        routing = gmmxx_amd.route_rows(x @ self.gate, self.top_k)
        branch = gmmxx_amd.combine_rows(gmmxx_amd.grouped_matmul(x, self.maps, routing), routing)
        if self.training:
            h = gmmxx_amd.dropout(branch, self.dropout, self.steps, residual=h)
        else:
            h = h + branch
        return gmmxx_amd.layer_norm(h)

    def loss(self, tokens, following, entropy=0.01):
        p = gmmxx_amd.log_probs(self.hidden(tokens) @ self.head.t(), following)
        counted = (following >= 0).sum()
        return -(p.chosen.sum() + entropy * p.entropy.sum()) / counted

    @torch.no_grad()
    def quantized_head(self):
        """The head as it is now, for ``answer``."""
        return gmmxx_amd.quantize_rows(self.head)

    @torch.no_grad()
    def answer(self, tokens, top_k=3, head=None):
        """The likeliest next tokens and their log probabilities.  ``head``: a trained model's ``quantized_head()``,
        made once for many answers; without it the head is brought into 8 bits here."""
        scores = gmmxx_amd.quantized_matmul(self.hidden(tokens), self.quantized_head() if head is None else head)
        return gmmxx_amd.log_probs(scores, torch.full_like(tokens, -1), top_k=top_k)


def make_codes(rows=20_000, width=8, clusters=20, device="cuda:0", seed=0):
    """Rows that go from one cluster to its next one, or sometimes anywhere; a mixture's labels of them."""
    g = torch.Generator().manual_seed(seed)
    centers = 6.0 * torch.randn((clusters, width), generator=g)
    jump, anywhere = torch.rand(rows, generator=g) < 0.2, torch.randint(0, clusters, (rows,), generator=g)
    at, path = 0, []
    for r in range(rows):
        at = int(anywhere[r]) if jump[r] else (at + 1) % clusters
        path.append(at)
    x = (centers[torch.tensor(path)] + torch.randn((rows, width), generator=g)).to(device)
    mixture = gmmxx_amd.GMMXX(n_components=clusters, covariance_type="diag", max_iter=20, device=device).fit(x)
    return mixture.predict(x)


def run(rows=20_000, clusters=20, steps=150, dtype=torch.bfloat16, device="cuda:0"):
    codes = make_codes(rows, clusters=clusters, device=device)
    tokens, following = codes[:-1], codes[1:]
    model = CodeModel(clusters, dtype=dtype, device=device)
    optimiser = torch.optim.Adam(model.parameters(), lr=1e-2)
    losses = []
    for _ in range(steps):
        optimiser.zero_grad()
        loss = model.loss(tokens, following)
        loss.backward()
        optimiser.step()
        model.steps += 1
        losses.append(loss.detach())
    model.eval()
    return [float(v) for v in losses], model, codes


def main():
    losses, model, codes = run()
    print(f"loss {losses[0]:.3f} -> {losses[-1]:.3f} in {len(losses)} steps")
    head = model.quantized_head()
    answer = model.answer(codes[:1], head=head)
    print(f"after {int(codes[0])}:", ", ".join(f"{int(t)} ({float(p):.2f})" for t, p in
                                               zip(answer.top_index[0], answer.top[0])))


if __name__ == "__main__":
    main()
