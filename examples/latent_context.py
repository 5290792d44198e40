"""A context model beside the codec: attention from the feature tokens of each
packet to those of earlier packets.

Encodes a seeded synthetic sequence (one I packet, then P packets of 8 frames)
with the seeded random-init models, and after each packet takes the codec's
reference features (Q9 integers, one token per 8 x 8 pixels) through two
attention layers with random weights:

* rotary positions over (packet, row, column);
* keys and values of every packet in the 8-bit paged cache, with a window of a
  few packets and the first packet's first tokens always visible;
* two trial codings of the last packet, at different QPs, that branch off the
  same decoded state -- their full pages shared, their own tokens apart;
* pages behind the window dropped, the trials released, the pool compacted.

    python examples/latent_context.py --width 128 --height 128 --packets 3

prints one JSON line.  The weights are random: what is shown is the use of the
operators, not a trained model.
"""
from __future__ import annotations

import argparse
import json
import os
import sys

import numpy as np
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)

import __graft_entry__ as entry  # noqa: E402

FEATURES, HEADS, KV_HEADS, DIM, LAYERS, PAGE = 512, 8, 2, 64, 2, 32


class ContextModel:
    """Pre-norm attention layers over a KVCache, random weights, bfloat16 products."""

    def __init__(self, ufb, rows, columns, slots, packets, device):
        self.ufb, self.device, self.tokens = ufb, device, rows * columns
        gen = torch.Generator(device=device).manual_seed(5)
        w = lambda i, o: (torch.randn(i, o, generator=gen, device=device) * i ** -0.5).bfloat16()  # noqa: E731
        self.qkv = [w(FEATURES, (HEADS + 2 * KV_HEADS) * DIM) for _ in range(LAYERS)]
        self.out = [w(HEADS * DIM, FEATURES) for _ in range(LAYERS)]
        self.rotary = ufb.Rotary((8, 12, 12), (4096, rows, columns), (10000.0, 100.0, 100.0), device=device)
        width = -(-self.tokens * packets // PAGE) + 1
        self.cache = ufb.KVCache(LAYERS, slots * width, KV_HEADS, DIM, PAGE, slots, width, device=device)
        i = torch.arange(self.tokens, device=device)
        self.grid = torch.stack([torch.zeros_like(i), i // columns, i % columns], 1).to(torch.int32)

    def step(self, slots, packets, features, window, sinks):
        """One packet's features [streams, tokens, FEATURES] of each listed stream
        at its packet index -> features after attention, float32."""
        n = len(slots)
        plan = self.cache.plan(slots, [self.tokens] * n)
        positions = self.grid.repeat(n, 1)
        positions[:, 0] = torch.tensor(packets, dtype=torch.int32, device=self.device).repeat_interleave(self.tokens)
        x = features.reshape(n * self.tokens, FEATURES)
        self.cache.extend(plan)
        for layer in range(LAYERS):
            y = (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)).bfloat16()
            qkv = (y @ self.qkv[layer]).view(-1, HEADS + 2 * KV_HEADS, DIM)
            q, k = self.rotary.apply(positions, qkv[:, :HEADS], qkv[:, HEADS:HEADS + KV_HEADS])
            self.cache.append(layer, plan, k, qkv[:, HEADS + KV_HEADS:])
            # the tokens of a packet are there together: no order among them
            o = self.cache.attend(layer, plan, q, window=window, sinks=sinks, causal=False)
            x = x + (o.flatten(1) @ self.out[layer]).float()
        return x.view(n, self.tokens, FEATURES)


def features_of(codec, device):
    """The codec's reference features (Q9) as tokens [1, H/8 * W/8, 512]."""
    state = codec.state("reference")
    if state.shape[1] != FEATURES:   # after an I packet: the unshuffled frame, fewer channels
        state = np.concatenate([state] * (-(-FEATURES // state.shape[1])), 1)[:, :FEATURES]
    t = torch.from_numpy(state).to(device).float() / 512.0
    return t.flatten(2).transpose(1, 2)


def main(argv=None) -> dict:
    p = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    p.add_argument("--width", type=int, default=128)
    p.add_argument("--height", type=int, default=128)
    p.add_argument("--packets", type=int, default=3, help="P packets")
    p.add_argument("--window-packets", type=int, default=2)
    p.add_argument("--sinks", type=int, default=16)
    a = p.parse_args(argv)
    ufb, syn = entry.load_package(), entry.load_synthetic()
    device = torch.device("cuda:0")
    rows, columns = -(-a.height // 16) * 2, -(-a.width // 16) * 2
    tokens = rows * columns

    image = ufb.Codec(ufb.Model("image", syn.prepared("image", 1)), 1)
    video_model = ufb.Model("htl", syn.prepared("htl", 2))
    trials = [ufb.Codec(video_model, 1) for _ in range(2)]
    for c in [image] + trials:
        c.set_skip_threshold(0.2)
    frames = syn.synthetic_video(a.width, a.height, 1 + 8 * a.packets, 3)
    image.compress(syn.frames_to_chunk(frames[:1]), 0)
    for c in trials:
        c.set_reference_from(image)

    model = ContextModel(ufb, rows, columns, 3, a.packets + 2, device)
    cache, window = model.cache, a.window_packets * tokens
    model.step([0], [0], features_of(trials[0], device), window, a.sinks)
    one = cache.plan([0], [0])
    sizes = []
    for packet in range(a.packets):
        chunk = syn.frames_to_chunk(frames[1 + 8 * packet: 9 + 8 * packet])
        last = packet == a.packets - 1
        if last:
            # two trial codings of the last packet branch off the decoded state
            cache.fork(cache.fork_plan([0, 0], [1, 2]))
        qps = (20, 40) if last else (20, 20)
        for codec, qp in zip(trials, qps):
            sizes.append(len(codec.compress(chunk, qp, True)[0][0]))
        if last:
            x = torch.cat([features_of(c, device) for c in trials])
            result = model.step([1, 2], [packet + 1] * 2, x, window, a.sinks)
        else:
            model.step([0], [packet + 1], features_of(trials[0], device), window, a.sinks)
            cache.trim(one, window, a.sinks)
    used = int((cache.refs > 0).sum())
    cache.release(cache.plan([0, 2], [0, 0]))
    cache.compact()
    kept = int((cache.refs > 0).sum())
    event = {"event": "latent_context", "tokens_per_packet": tokens, "bytes": sizes, "lengths": cache.lengths.tolist(),
             "pages_used": used, "pages_kept": kept, "pages_lowest": bool((cache.refs[:kept] > 0).all()),
             "finite": bool(torch.isfinite(result).all()),
             "trials_differ": float((result[0] - result[1]).abs().mean()), "status": ufb.device_status(0)}
    print(json.dumps(event))
    return event


if __name__ == "__main__":
    main()
