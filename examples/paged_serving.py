"""Serving with a paged K / V cache: prompts, parallel answers, single-token steps, release.

A toy decoder (embedding, attention layers with grouped heads and a residual, greedy head, all
with random weights) runs as a server would: the prompts are packed and go through
``gqa_attn.prefill``, their keys and values into pages (``kv_pages.reserve`` / ``append``); each
prompt is forked into several answers that share its pages; every step writes one token per
sequence and reads the cache with ``gqa_attn.decode``; finished sequences are freed and the
pages that are left move together.

    python -m examples.paged_serving        (from the repository's root)
"""

import torch

import mzoo_b200
from mzoo_b200 import gqa_attn, kv_pages

HQ, HKV, D, PAGE = 8, 2, 64, 16


class Model:
    def __init__(self, layers=2, vocab=512, device="cuda", seed=0):
        g = torch.Generator().manual_seed(seed)
        width = HQ * D

        def weight(*shape):
            return (torch.randn(*shape, generator=g) / shape[0] ** 0.5).to(torch.bfloat16).to(device)
        self.embed = weight(vocab, width) * vocab ** 0.5
        self.qkv = [weight(width, (HQ + 2 * HKV) * D) for _ in range(layers)]
        self.out = [weight(width, width) for _ in range(layers)]
        self.head = weight(width, vocab)

    def layer_qkv(self, i, x):
        x = torch.nn.functional.rms_norm(x, x.shape[-1:])
        return (x @ self.qkv[i]).view(-1, HQ + 2 * HKV, D).split([HQ, HKV, HKV], 1)  # views of one projection

    def after(self, i, x, o):
        return x + o.reshape(x.shape) @ self.out[i]

    def logits(self, x):
        return torch.nn.functional.rms_norm(x, x.shape[-1:]) @ self.head


class Cache:
    """Pages of every layer's K and V, and which sequence (slot) owns which."""

    def __init__(self, model, slots, pages, width, device="cuda"):
        shape = (pages, HKV, PAGE, D)
        self.pools = [torch.zeros(shape, dtype=torch.bfloat16, device=device) for _ in range(2 * len(model.qkv))]
        self.table = torch.full((slots, width), -1, dtype=torch.int32, device=device)
        self.lens = torch.zeros(slots, dtype=torch.int32, device=device)
        self.refs = torch.zeros(pages, dtype=torch.int32, device=device)

    def room(self, n_new):
        return kv_pages.reserve(self.table, self.lens, self.refs, n_new, page_size=PAGE)


def prompts(model, cache, tokens, cu, n_new):
    """Packed prompts (one per slot, n_new[slot] tokens) -> logits after each prompt's last token."""
    starts = cache.room(n_new)
    x = model.embed[tokens]
    for i in range(len(model.qkv)):
        q, k, v = model.layer_qkv(i, x)
        kv_pages.append(k, v, cache.pools[2 * i], cache.pools[2 * i + 1], cache.table[:len(cu) - 1], starts[:len(cu) - 1], cu)
        x = model.after(i, x, gqa_attn.prefill(q, k, v, cu)[0])
    return model.logits(x[cu[1:].long() - 1])


def step(model, cache, tokens):
    """One token for every slot -> logits."""
    starts = cache.room(torch.ones_like(cache.lens))
    x = model.embed[tokens]
    for i in range(len(model.qkv)):
        q, k, v = model.layer_qkv(i, x)
        kv_pages.append(k, v, cache.pools[2 * i], cache.pools[2 * i + 1], cache.table, starts)
        x = model.after(i, x, gqa_attn.decode(q, cache.pools[2 * i], cache.pools[2 * i + 1], cache.table, cache.lens)[0])
    return model.logits(x)


@torch.no_grad()
def serve(lengths=(5, 40, 17), answers=3, steps=20, device="cuda"):
    """-> (model, token lists of all sequences, their last logits, cache) after `steps` greedy steps."""
    model = Model(device=device)
    n, slots = len(lengths), len(lengths) * answers
    width = -(-(max(lengths) + steps) // PAGE)
    cache = Cache(model, slots, slots * width, width, device)
    g = torch.Generator().manual_seed(1)
    texts = [torch.randint(0, 512, (m,), generator=g) for m in lengths]
    cu = torch.tensor([0, *lengths]).cumsum(0).to(torch.int32).to(device)
    n_new = torch.tensor([*lengths] + [0] * (slots - n), dtype=torch.int32, device=device)
    logits = prompts(model, cache, torch.cat(texts).to(device), cu, n_new)
    # answer a of prompt p lives in slot a * n + p; the first one is the prompt's own slot
    src = torch.arange(n, dtype=torch.int32, device=device).repeat(answers - 1)
    kv_pages.fork(cache.pools, cache.table, cache.lens, cache.refs, src,
                  torch.arange(n, slots, dtype=torch.int32, device=device), page_size=PAGE)
    # the answers start with the best, second best, ... token
    token = logits.topk(answers, -1).indices.T.reshape(-1)
    made = [token]
    for _ in range(steps):
        logits = step(model, cache, token)
        token = logits.argmax(-1)
        made.append(token)
    mzoo_b200.check_errors()
    made = torch.stack(made[:-1], 1).cpu()  # the last one has not been run
    return model, [torch.cat([texts[s % n], made[s]]) for s in range(slots)], logits, cache


@torch.no_grad()
def whole(model, texts, device="cuda"):
    """Last logits of the same sequences without a cache: one packed prefill."""
    cu = torch.tensor([0] + [len(t) for t in texts]).cumsum(0).to(torch.int32).to(device)
    x = model.embed[torch.cat(texts).to(device)]
    for i in range(len(model.qkv)):
        x = model.after(i, x, gqa_attn.prefill(*model.layer_qkv(i, x), cu)[0])
    return model.logits(x[cu[1:].long() - 1])


def main():
    model, texts, logits, cache = serve()
    far = (logits.float() - whole(model, texts).float()).abs().max()
    used = int((cache.refs > 0).sum())
    print(f"{len(texts)} sequences of {min(map(len, texts))} to {max(map(len, texts))} tokens on {used} pages; "
          f"logits against one packed run without a cache: largest difference {float(far):.4f}")
    gone = torch.arange(0, len(texts), 2, dtype=torch.int32, device="cuda")
    kv_pages.free(cache.table, cache.lens, cache.refs, gone)
    cache.table, cache.refs = kv_pages.compact(cache.pools, cache.table, cache.refs)
    mzoo_b200.check_errors()
    print(f"after {len(gone)} sequences were freed: {int((cache.refs > 0).sum())} pages, "
          f"the highest in use is number {int(cache.refs.nonzero().max())}")


if __name__ == "__main__":
    main()
