"""Trains a small decoder on packed batches: several documents per sequence that do not see each other, each counting from zero and with an image
inside that is positioned by time, height and width, scores capped, gradients clipped by their global norm.

    python examples/packed_documents.py [--steps 20] [--seq-length 1024] [--device cuda]
"""
from __future__ import annotations

import argparse
import os
import random
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from lightron_b200.config import ModelArgs  # noqa: E402
from lightron_b200.models import LightronTransformer, init_weights  # noqa: E402
from lightron_b200.ops import functional as OF  # noqa: E402


def packed_batch(rng: random.Random, batch: int, length: int, vocab: int):
    """(tokens, targets, documents, prefix, positions): documents of a prompt with an image of 4 columns, and an answer that repeats after a few tokens."""
    tokens, documents = torch.zeros(batch, length, dtype=torch.long), torch.full((batch, length), -1, dtype=torch.int32)
    targets, prefix = torch.full((batch, length), -100), torch.zeros(batch, length, dtype=torch.bool)
    positions = torch.zeros(3, batch, length, dtype=torch.int32)
    for b in range(batch):
        at, doc = 0, 0
        while length - at >= 24:
            n, image, period = min(length - at, rng.randint(24, 300)), 4 * rng.randint(1, 4), rng.randint(2, 7)
            prompt = image + 2
            word = [rng.randrange(vocab) for _ in range(period)]
            tokens[b, at:at + n] = torch.tensor([word[i % period] for i in range(n)])
            documents[b, at:at + n] = doc
            prefix[b, at:at + prompt] = True
            targets[b, at + prompt:at + n - 1] = tokens[b, at + prompt + 1:at + n]
            i = torch.arange(n, dtype=torch.int32)
            text = i - image + max(image // 4, 4)                 # text goes on behind the largest position of the image
            for axis, inside in enumerate((torch.zeros_like(i), i // 4, i % 4)):
                positions[axis, b, at:at + n] = torch.where(i < image, inside, text)
            at, doc = at + n, doc + 1
    return tokens, targets, documents, prefix, positions


def main(argv=None) -> list:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--batch", type=int, default=4)
    ap.add_argument("--seq-length", type=int, default=1024)
    ap.add_argument("--dim", type=int, default=512)
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--device", default="cuda" if torch.cuda.is_available() else "cpu")
    a = ap.parse_args(argv)
    dtype = torch.bfloat16 if a.device == "cuda" else torch.float32
    head = 64 if a.dim >= 256 else 16
    args = ModelArgs(dim=a.dim, n_layers=a.layers, n_heads=a.dim // head, n_kv_heads=a.dim // head // 2, vocab_size=1024, intermediate_size=2 * a.dim, max_seq_len=a.seq_length,
                     attn_softcap=50.0, rope_sections=(head // 8, 3 * head // 16, 3 * head // 16))
    model = LightronTransformer(args, dtype=dtype, device=a.device)
    init_weights(model, 0)
    opt = torch.optim.AdamW(model.parameters(), lr=1e-3, weight_decay=0.0)
    rng, losses = random.Random(0), []
    for step in range(a.steps):
        tokens, targets, documents, prefix, positions = (t.to(a.device) for t in packed_batch(rng, a.batch, a.seq_length, args.vocab_size))
        mask = OF.attention_mask(documents=documents, prefix=prefix)          # once per batch, for all layers
        opt.zero_grad()
        loss = model.loss(tokens, targets, positions=positions, mask=mask, n_tokens=int((targets >= 0).sum()))
        loss.backward()
        norm = OF.clip_grad_norm([p.grad for p in model.parameters()], 1.0)
        opt.step()
        losses.append(float(loss.detach()))
        print(f"step {step + 1}: loss {losses[-1]:.4f}, gradient norm {float(norm):.3f}", flush=True)
    return losses


if __name__ == "__main__":
    main()
