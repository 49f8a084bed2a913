#!/usr/bin/env python3
"""A small decoder served with an 8-bit key/value cache, whose idle cache is parked
with the codec and restored bit for bit.

Random weights; per layer: residual sum and norm into 8 bits (add_rms_norm), the
projections, the new keys and values into the pages (kv_write), attention of the
chunk over the pages (KvAttention).  Prompts go in as ragged chunks, tokens then
one by one.  Half way the cache's tensors are compressed (compress_many), cleared
and decoded again (decode_many): the program goes on as if nothing had happened.

Usage: python examples/park_cache.py [--tokens 16] [--layers 2]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import checkers_amd as ck  # noqa: E402

HIDDEN, HEADS, KV_HEADS, DIM, VOCAB, PAGE, UNIT = 1024, 16, 4, 64, 4096, 64, 65536


class Layer:
    def __init__(self, n_pages, rng, dev):
        def w(a, b):
            return (torch.randn(a, b, generator=rng, device=dev) * a ** -0.5).to(torch.bfloat16)
        self.norm_in = torch.ones(HIDDEN, dtype=torch.bfloat16, device=dev)
        self.norm_out = torch.ones(HIDDEN, dtype=torch.bfloat16, device=dev)
        self.qkv, self.o = w(HIDDEN, (HEADS + 2 * KV_HEADS) * DIM), w(HEADS * DIM, HIDDEN)
        self.up, self.down = w(HIDDEN, 2 * HIDDEN), w(2 * HIDDEN, HIDDEN)
        self.cache = ck.KvCache.empty(n_pages, PAGE, KV_HEADS, DIM, ck.F8, device=dev)


def project(x8, scales, weight):
    """A product of 8-bit rows: their codes are exact in bfloat16, a row's scale is applied after it."""
    return (x8.to(torch.bfloat16) @ weight).float() * scales[:, None]


class Server:
    """Sequences of at most `longest` tokens, each with its own pages."""

    def __init__(self, n_seqs, longest, layers, seed=0, device="cuda"):
        dev = torch.device(device)
        rng = torch.Generator(device=dev).manual_seed(seed)
        per = -(-longest // PAGE)
        self.table = torch.randperm(n_seqs * per, generator=rng, device=dev).to(torch.int32).view(n_seqs, per)
        self.layers = [Layer(n_seqs * per, rng, dev) for _ in range(layers)]
        self.embed = torch.randn(VOCAB, HIDDEN, generator=rng, device=dev).to(torch.bfloat16)
        self.head = torch.randn(HIDDEN, VOCAB, generator=rng, device=dev)
        self.norm = torch.ones(HIDDEN, dtype=torch.bfloat16, device=dev)
        self.lens = [0] * n_seqs
        self.longest = longest
        self.plan = ck.KvAttention(HEADS, KV_HEADS, DIM, n_seqs, n_seqs * longest, longest, longest, device=dev)

    def step(self, chunks):
        """Take each sequence's new tokens (a list of token lists); the next token of each."""
        dev = self.embed.device
        new = [len(c) for c in chunks]
        offsets = torch.tensor([0] + new).cumsum(0)
        batch = ck.KvBatch(self.table, torch.tensor(self.lens, dtype=torch.int32, device=dev),
                           offsets.to(torch.int32).to(dev), sum(new), max(new), max(a + b for a, b in zip(self.lens, new)))
        n = batch.n_tokens
        x = self.embed[torch.tensor([t for c in chunks for t in c], device=dev)]
        delta = torch.zeros_like(x)
        for la in self.layers:
            x8, s, x = ck.add_rms_norm(delta, x, la.norm_in, dtype=ck.F8)
            qkv = project(x8, s, la.qkv).to(torch.bfloat16).view(n, HEADS + 2 * KV_HEADS, DIM)
            ck.kv_write(la.cache, batch, qkv[:, HEADS:HEADS + KV_HEADS], qkv[:, HEADS + KV_HEADS:])
            a = self.plan.run(la.cache, batch, qkv[:, :HEADS])
            x8, s, x = ck.add_rms_norm((a.view(n, -1) @ la.o), x, la.norm_out, dtype=ck.F8)
            delta = (torch.nn.functional.silu(project(x8, s, la.up)).to(torch.bfloat16) @ la.down)
        y, _, _ = ck.add_rms_norm(delta, x, self.norm)
        self.lens = [a + b for a, b in zip(self.lens, new)]
        last = (offsets[1:] - 1).to(dev)
        return (y[last].float() @ self.head).argmax(-1).tolist()

    def tensors(self):
        """The cache's tensors as the codec takes them: bytes and float32 scales."""
        return [t.view(torch.uint8) if t.element_size() == 1 else t for la in self.layers for t in la.cache.tensors()]


def park(tensors):
    """The tensors compressed, losslessly: (encoders, encoded)."""
    tags = [ck.I8 if t.element_size() == 1 else ck.F32 for t in tensors]
    encoders = [ck.Encoder(t.numel(), tag, UNIT, device=t.device) for t, tag in zip(tensors, tags)]
    return encoders, ck.compress_many(encoders, tensors)


def restore(encoders, encoded, tensors):
    decoders = [ck.Decoder(e.n_elems, e.dtype, e.unit_bytes, device=t.device) for e, t in zip(encoders, tensors)]
    bad = ck.decode_many(decoders, encoded, tensors)
    if any(bad):
        raise RuntimeError(f"parked cache is damaged: {bad}")


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--tokens", type=int, default=16)
    ap.add_argument("--layers", type=int, default=2)
    a = ap.parse_args(argv)
    prompts = [[(7 * i + 13 * s) % VOCAB for i in range(n)] for s, n in enumerate((200, 3, 77, 450))]
    runs = []
    for parked in (False, True):
        srv = Server(len(prompts), max(map(len, prompts)) + a.tokens + 1, a.layers)
        half = [p[: len(p) // 2] for p in prompts]
        srv.step(half)                                         # prompts in two chunks
        nxt = srv.step([p[len(h):] for p, h in zip(prompts, half)])
        out = [nxt]
        for i in range(a.tokens):
            if parked and i == a.tokens // 2:
                ts = srv.tensors()
                kept = [t.clone() for t in ts]
                encoders, encoded = park(ts)
                size = sum(t.numel() * t.element_size() for t in ts)
                small = sum(e.total + (e.sidecar.numel() if e.sidecar is not None else 0) for e in encoded)
                for t in ts:
                    t.zero_()
                restore(encoders, encoded, ts)
                same = all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(ts, kept))
                print(f"parked {size} bytes of cache in {small} ({size / small:.2f}x), restored {'bit for bit' if same else 'WRONG'}")
                if not same:
                    return 1
            nxt = srv.step([[t] for t in nxt])
            out.append(nxt)
        runs.append(out)
    ok = runs[0] == runs[1]
    print(f"{a.tokens} tokens of {len(prompts)} sequences: with the cache parked half way {'the same' if ok else 'DIFFERENT'}")
    return 0 if ok else 1


if __name__ == "__main__":
    sys.exit(main())
