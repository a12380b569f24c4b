"""A small causal encoder whose sequences are told apart by their embeddings, trained and then served token by token.

Training: packed projections, rotary positions, causal attention over shared key heads, mean pooling over each sequence's own length,
cosine similarities between two noisy views of every sequence as logits.  Serving: the same layer takes one token at a time with
its keys and values in a cache, and arrives at the embeddings that the whole sequence gives.

    python examples/attention_retrieval.py [--steps 60]
"""
import argparse
import sys
from pathlib import Path

import torch
import torch.nn.functional as F

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
import torchpairwise_b200 as tpw  # noqa: E402

HEADS, KEY_HEADS, WIDTH, LONGEST = 8, 2, 64, 256


class Encoder(torch.nn.Module):
    """One attention layer over embedded tokens: weights in 32 bits, attention in `dtype`."""

    def __init__(self, dtype, words=512, features=256):
        super().__init__()
        self.dtype = dtype
        self.words = torch.nn.Embedding(words, features)
        self.project = torch.nn.Linear(features, (HEADS + 2 * KEY_HEADS) * WIDTH, bias=False)
        self.out = torch.nn.Linear(HEADS * WIDTH, features, bias=False)
        cos, sin = tpw.rotary_table(LONGEST, WIDTH)
        self.register_buffer("cos", cos)
        self.register_buffer("sin", sin)

    def parts(self, tokens, positions):
        qkv = self.project(self.words(tokens)).to(self.dtype).unflatten(-1, (-1, WIDTH))
        q, k, v = qkv.split((HEADS, KEY_HEADS, KEY_HEADS), 2)   # views of one projection
        q, k = tpw.rotary_embedding(q, k, self.cos, self.sin, positions)
        return q, k, v

    def hidden(self, tokens):
        """Outputs of every token, each sequence padded at its end; a causal token sees no padding."""
        q, k, v = self.parts(tokens, None)
        return self.out(tpw.attention(q, k, v, causal=True).flatten(2).float())

    def forward(self, tokens, lengths):
        h = self.hidden(tokens)
        inside = torch.arange(tokens.size(1), device=tokens.device) < lengths[:, None]
        return (h * inside[..., None]).sum(1) / lengths[:, None]

    @torch.no_grad()
    def serve(self, tokens, lengths):
        """The same embeddings from one token at a time: the new token's keys and values join the cache, its query reads it."""
        batch, longest = tokens.shape
        keys = torch.empty(batch, longest, KEY_HEADS, WIDTH, dtype=self.dtype, device=tokens.device)
        values = torch.empty_like(keys)
        total = torch.zeros(batch, self.out.out_features, dtype=torch.float32, device=tokens.device)
        for t in range(longest):
            q, k, v = self.parts(tokens[:, t:t + 1], torch.tensor([t], device=tokens.device))
            keys[:, t:t + 1], values[:, t:t + 1] = k, v
            held = torch.full((batch,), t + 1, dtype=torch.int32, device=tokens.device)
            h = self.out(tpw.attention(q, keys, values, causal=True, key_lengths=held).flatten(2).float())[:, 0]
            total += torch.where((t < lengths)[:, None], h, torch.zeros_like(h))
        return total / lengths[:, None]


def views(generator, sequences, words, device):
    """Two views of random sequences of ragged lengths: a fifth of the words is the sequence's own and in both, from the first quarter of the
    vocabulary; the others are filler, drawn anew."""
    lengths = torch.randint(20, LONGEST + 1, (sequences,), generator=generator)
    shape = (sequences, LONGEST)
    kept = torch.rand(shape, generator=generator) < 0.2
    own = torch.randint(0, words // 4, shape, generator=generator)
    out = [torch.where(kept, own, torch.randint(words // 4, words, shape, generator=generator)).to(device) for _ in range(2)]
    return out[0], out[1], lengths.to(device)


def main(steps=60, sequences=64, dtype=torch.bfloat16, device="cuda", seed=0, report=print):
    torch.manual_seed(seed)
    generator = torch.Generator().manual_seed(seed)
    model = Encoder(dtype).to(device=device)
    optimiser = torch.optim.AdamW(model.parameters(), lr=1e-3)
    losses = []
    for step in range(steps):
        a, b, lengths = views(generator, sequences, 512, device)
        similarity = tpw.cosine_similarity(model(a, lengths), model(b, lengths))   # [sequences, sequences]
        loss = F.cross_entropy(similarity * 10, torch.arange(sequences, device=device))
        optimiser.zero_grad(set_to_none=True)
        loss.backward()
        optimiser.step()
        losses.append(float(loss.detach()))
        if step % 10 == 0 or step == steps - 1:
            report(f"step {step:3d}  loss {losses[-1]:.4f}")
    tokens, _, lengths = views(generator, 8, 512, device)
    with torch.no_grad():
        whole = model(tokens, lengths)
    served = model.serve(tokens, lengths)
    apart = float((whole - served).norm() / whole.norm())
    report(f"embeddings served token by token are {apart:.2e} from those of whole sequences")
    return losses, apart


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=60)
    main(ap.parse_args().steps)
