"""Trains a small text encoder with the encoder operators, then searches with it.

    python cuda-vector-search_amd/examples/train_encoder.py [--steps 200] [--seed 0]

Documents are token sequences of differing lengths about synthetic topics; a query is a few of
a document's tokens in another order and in another language (tokens of its own).  The encoder's layers (attention with a learned
bias by relative position, a feed-forward pair, layer norms) run ``encoder.attention``,
``encoder.linear`` and ``encoder.layer_norm``, forward and backward; the loss is the softmax
over the batch's documents of each query's cosine with them.  Before and after training
every document is embedded, put into an ``Index``, and the queries look for theirs.
(No counterpart in the reference, whose corpora are embedded elsewhere.)
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch
from torch import nn

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from cuda_vector_search import Index, encoder  # noqa: E402

TYPE = torch.bfloat16


class Layer(nn.Module):
    """One encoder layer, norms after the residuals; parameters in float32, used in bfloat16."""

    def __init__(self, width: int, heads: int, buckets: int = 32):
        super().__init__()
        self.heads = heads

        def weight(out, inp):
            return nn.Parameter(torch.randn(out, inp) * inp**-0.5)

        self.qkv, self.qkv_bias = weight(3 * width, width), nn.Parameter(torch.zeros(3 * width))
        self.out, self.out_bias = weight(width, width), nn.Parameter(torch.zeros(width))
        self.up, self.up_bias = weight(4 * width, width), nn.Parameter(torch.zeros(4 * width))
        self.down, self.down_bias = weight(width, 4 * width), nn.Parameter(torch.zeros(width))
        self.norms = nn.ParameterList([torch.ones(width), torch.zeros(width), torch.ones(width), torch.zeros(width)])
        self.table = nn.Parameter(torch.zeros(buckets, heads))

    def forward(self, x, lengths):
        b, l, width = x.shape
        p = {n: t.to(TYPE) for n, t in self.named_parameters()}
        qkv = encoder.linear(x, p["qkv"], p["qkv_bias"]).view(b, l, 3, self.heads, width // self.heads)
        a = encoder.attention(qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2], p["table"], lengths, lengths)
        x = encoder.linear(a.view(b, l, width), p["out"], p["out_bias"], residual=x)
        x = encoder.layer_norm(x, p["norms.0"], p["norms.1"])
        h = encoder.linear(x, p["up"], p["up_bias"], "gelu")
        x = encoder.linear(h, p["down"], p["down_bias"], residual=x)
        return encoder.layer_norm(x, p["norms.2"], p["norms.3"])


class Encoder(nn.Module):
    """Tokens [b, l] of which the first lengths[b] count -> unit vectors [b, width]."""

    def __init__(self, vocabulary: int, width: int = 128, heads: int = 4, layers: int = 2):
        super().__init__()
        self.tokens = nn.Parameter(torch.randn(vocabulary, width) * 0.5)
        self.layers = nn.ModuleList(Layer(width, heads) for _ in range(layers))

    def forward(self, tokens, lengths):
        x = self.tokens[tokens].to(TYPE)
        for layer in self.layers:
            x = layer(x, lengths)
        counts = torch.arange(tokens.shape[1], device=tokens.device) < lengths[:, None]
        pooled = (x.float() * counts[..., None]).sum(1)
        return nn.functional.normalize(pooled, dim=1)


def documents(n: int, vocabulary: int, longest: int, g: torch.Generator):
    """(tokens, lengths): each document draws from a handful of tokens of its topic and from all."""
    topics = torch.randint(0, vocabulary, (max(8, n // 8), 40), generator=g)
    lengths = torch.randint(longest // 4, longest + 1, (n,), generator=g)
    own = topics[torch.randint(0, len(topics), (n,), generator=g)]
    pick = own.gather(1, torch.randint(0, 40, (n, longest), generator=g))
    any_ = torch.randint(0, vocabulary, (n, longest), generator=g)
    return torch.where(torch.rand(n, longest, generator=g) < 0.7, pick, any_), lengths


def queries(tokens, lengths, size: int, vocabulary: int, g: torch.Generator):
    """A few tokens of each document, in another order, translated: by `vocabulary` further on."""
    at = (torch.rand(len(tokens), size, generator=g) * lengths[:, None]).long()
    return vocabulary + tokens.gather(1, at), torch.full((len(tokens),), size)


def recall(model, docs, q) -> float:
    """Share of the queries whose document is among the ten that the index finds."""
    with torch.no_grad():
        index = Index(model(*docs), metric="cosine")
        _, ids = index.search(model(*q).half(), 10)
    return float((ids == torch.arange(len(ids), device=ids.device)[:, None]).any(1).float().mean())


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--seed", type=int, default=0)
    args = ap.parse_args(argv)
    g = torch.Generator().manual_seed(args.seed)
    torch.manual_seed(args.seed)
    vocabulary = 600
    model = Encoder(2 * vocabulary).cuda()

    def on_gpu(pair):
        return pair[0].cuda(), pair[1].to(torch.int32).cuda()

    text = documents(1024, vocabulary, 96, g)
    docs, held = on_gpu(text), on_gpu(queries(*text, 16, vocabulary, g))
    before = recall(model, docs, held)
    optimiser = torch.optim.AdamW(model.parameters(), lr=2e-3)
    for step in range(args.steps):
        some = torch.randperm(len(text[0]), generator=g)[:128]
        batch = text[0][some], text[1][some]
        d, q = model(*on_gpu(batch)), model(*on_gpu(queries(*batch, 16, vocabulary, g)))
        loss = nn.functional.cross_entropy(q @ d.T / 0.05, torch.arange(len(d), device=d.device))
        optimiser.zero_grad(set_to_none=True)
        loss.backward()
        optimiser.step()
        if step % 50 == 0 or step + 1 == args.steps:
            print(f"step {step}: loss {loss.item():.3f}", flush=True)
    after = recall(model, docs, held)
    print(f"recall@10 of {len(held[0])} queries: {before:.3f} before training, {after:.3f} after", flush=True)
    return before, after


if __name__ == "__main__":
    main()
