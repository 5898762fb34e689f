"""Serving several prompts from one pool of 8-bit pages: packed prefill, shared samples, decode steps, housekeeping.

    python examples/paged_serving.py [--layers 4] [--steps 32]

A small random-weight decoder (attention only; no weights are shipped with this repository) runs as a server
would run it: the prompts are packed without padding and attend causally in one call per layer
(kvb.prefill_attention), their keys and values go into 8-bit pages (PagePool.write), each prompt is forked into
several samples that share its full pages (PagePool.fork), the samples decode token by token (extend, write, attend),
one of them ends (free), the pool closes the holes (compact), and a follow-up question continues a finished sample
by a chunk after its prefix (read, then prefill_attention with more keys than queries).
"""

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "kv-project_b200"))
import kvb  # noqa: E402

HQ, HKV, D, HIDDEN, VOCAB, PAGE = 32, 8, 128, 1024, 4096, 64


class Decoder:
    """Random-weight layers: RMS norm, one projection to q, k and v, attention, output projection."""

    def __init__(self, layers, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def weight(a, b):
            return (torch.randn(a, b, generator=g, device="cuda") / a ** 0.5).bfloat16()

        self.embed = weight(VOCAB, HIDDEN) * VOCAB ** 0.5
        self.qkv = [weight(HIDDEN, (HQ + 2 * HKV) * D) for _ in range(layers)]
        self.out = [weight(HQ * D, HIDDEN) for _ in range(layers)]

    def split(self, x, layer):
        h = x * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + 1e-6).bfloat16()
        y = (h @ self.qkv[layer]).view(-1, HQ + 2 * HKV, D)
        return y[:, :HQ], y[:, HQ:HQ + HKV], y[:, HQ + HKV:]

    def next_token(self, x):
        return (x @ self.embed.t()).float().argmax(-1)


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def offsets(lens):
    return ints([0] + torch.tensor(lens).cumsum(0).tolist())


def prompt(model, pools, slots, tokens, lens):
    """Packed prompts into empty sequences; the last position's token of each."""
    cu, start = offsets(lens), pools[0].extend(slots, ints(lens))
    x = model.embed[tokens]
    for i, pool in enumerate(pools):
        q, k, v = model.split(x, i)
        pool.write(slots, start, cu, k, v)
        x = x + kvb.prefill_attention(q, k, v, cu).flatten(1) @ model.out[i]
    return model.next_token(x[cu[1:].long() - 1])


def step(model, pools, slots, tokens, cu, one):
    """One decode step: every sequence's next token."""
    start = pools[0].extend(slots, one)
    x = model.embed[tokens]
    for i, pool in enumerate(pools):
        q, k, v = model.split(x, i)
        pool.write(slots, start, cu, k, v)
        x = x + pool.attend(q[:, :, None], slots).view(len(slots), -1) @ model.out[i]
    return model.next_token(x)


def follow_up(model, pools, slot, length, tokens):
    """A chunk of new tokens after a sequence's cached prefix."""
    n = len(tokens)
    start = pools[0].extend(slot, ints([n]))
    x, zero, cu, cu_all = model.embed[tokens], ints([0]), offsets([n]), offsets([length + n])
    for i, pool in enumerate(pools):
        q, k, v = model.split(x, i)
        pool.write(slot, start, cu, k, v)
        k, v = pool.read(slot, zero, cu_all, length + n)
        x = x + kvb.prefill_attention(q, k, v, cu, cu_all).flatten(1) @ model.out[i]
    return model.next_token(x[-1:])


def serve(layers=4, steps=32, lens=(700, 33, 1500), samples=4, seed=0):
    """Runs the example; returns the sampled tokens (sequences, steps) and the tokens of the follow-up."""
    model = Decoder(layers, seed)
    blocks = sum(-(-(n + steps + 64) // PAGE) for n in lens) * (samples + 1)
    pools = [kvb.PagePool.create(blocks, HKV, D, PAGE, n_slots=len(lens) * (samples + 1), max_blocks=blocks)]
    pools += [pools[0].add_layer() for _ in range(layers - 1)]
    g = torch.Generator(device="cuda").manual_seed(seed + 1)

    parents = ints(range(len(lens)))
    first = prompt(model, pools, parents, torch.randint(VOCAB, (sum(lens),), generator=g, device="cuda"), list(lens))

    children = ints(range(len(lens), len(lens) * (samples + 1)))
    pools[0].fork(parents.repeat_interleave(samples), children)
    pools[0].free(parents)                              # the samples hold the prompts' pages now

    n = len(children)
    one, cu = torch.ones_like(children), offsets([1] * n)
    # the samples begin with different tokens, as sampling would give them
    token = (first.repeat_interleave(samples) + torch.arange(samples, device="cuda").repeat(len(lens))) % VOCAB
    told = []
    for _ in range(steps):
        token = step(model, pools, children, token, cu, one)
        told.append(token)

    pools[0].free(children[1:2])
    live = pools[0].compact()
    last = follow_up(model, pools, children[:1], lens[0] + steps, torch.randint(VOCAB, (50,), generator=g, device="cuda"))
    told = torch.stack(told, 1)
    torch.cuda.synchronize()
    if kvb.device_status() != 0:
        raise RuntimeError("device status word set")
    print(f"{len(lens)} prompts of {list(lens)} tokens, {samples} samples each, {steps} steps, {layers} layers; "
          f"{int(live)} of {blocks} pages live after compaction")
    print("first sample:", told[0].tolist()[:16], "follow-up:", last.tolist())
    return told, last


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--steps", type=int, default=32)
    a = ap.parse_args()
    with torch.no_grad():
        serve(a.layers, a.steps)
