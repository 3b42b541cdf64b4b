"""Requests of different lengths decoded together over the paged 8-bit K/V cache.

A small decoder on MX linears (grouped K/V heads, rotary embedding, SwiGLU) with
synthetic weights.  One step: kv_plan gives every new token its place, each layer
appends its K/V rows to its cache and attends over it, and token_logprobs gives
the sampled tokens' log probabilities, the entropy and the alternatives.
Requests join with whole prompts while others decode; when one ends kv_release
gives its pages to the next.  The update at the end takes the policy gradient to the
logits of the tokens that were generated.

    python examples/paged_serving.py
"""
import os
import sys
from dataclasses import dataclass

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from cpu_model_b200 import mx  # noqa: E402


@dataclass
class Config:
    layers: int = 4
    dim: int = 1024
    heads: int = 8
    kv_heads: int = 2
    head_dim: int = 128
    ffn: int = 2816
    vocab: int = 32000
    page: int = 64
    pages: int = 256          # of the pool
    slots: int = 8            # requests at a time
    max_pages: int = 32       # pages a request
    theta: float = 10000.0


class PagedDecoder:
    def __init__(self, cfg, seed=0, device="cuda"):
        self.cfg = cfg
        g = torch.Generator(device=device).manual_seed(seed)
        rnd = lambda n, k: torch.randn((n, k), device=device, generator=g) * k ** -0.5
        weight = lambda n, k: mx.MXWeight.from_float(rnd(n, k), mx.FMT_INT8)
        rows = (cfg.heads + 2 * cfg.kv_heads) * cfg.head_dim
        self.layers = [dict(qkv=weight(rows, cfg.dim), out=weight(cfg.dim, cfg.heads * cfg.head_dim), gate=weight(cfg.ffn, cfg.dim),
                            up=weight(cfg.ffn, cfg.dim), down=weight(cfg.dim, cfg.ffn),
                            cache=mx.KVCache.empty(cfg.pages, cfg.page, cfg.kv_heads, cfg.head_dim, device))
                       for _ in range(cfg.layers)]
        self.head = weight(cfg.vocab, cfg.dim)
        self.embedding = torch.randn((cfg.vocab, cfg.dim), device=device, generator=g)
        half = cfg.head_dim // 2
        self.freq = cfg.theta ** (-torch.arange(half, device=device) / half)
        # the requests' state, on the device
        i32 = dict(dtype=torch.int32, device=device)
        self.lengths = torch.zeros(cfg.slots, **i32)
        self.table = torch.full((cfg.slots, cfg.max_pages), -1, **i32)
        self.free = torch.arange(cfg.pages, **i32)
        self.free_count = torch.tensor([cfg.pages], **i32)

    def _norm(self, x):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5)

    def _rotate(self, x, positions):
        a = positions.clamp(min=0).float()[:, None, None] * self.freq
        lo, hi = x.chunk(2, -1)
        return torch.cat([lo * a.cos() - hi * a.sin(), hi * a.cos() + lo * a.sin()], -1)

    def step(self, tokens, new, max_new):
        """tokens int32 [N], request by request; new int32 [slots] tokens of
        each (0: none).  Returns every token's logits and the step's plan."""
        c = self.cfg
        plan = mx.kv_plan(self.lengths, new, c.page, self.table, self.free, self.free_count, tokens.numel(), in_place=True)
        x = self.embedding[tokens.long()]
        q_dim, kv_dim = c.heads * c.head_dim, c.kv_heads * c.head_dim
        for w in self.layers:
            qkv = mx.mx_linear(self._norm(x), w["qkv"])
            q, k, v = (t.unflatten(1, (-1, c.head_dim)) for t in qkv.split([q_dim, kv_dim, kv_dim], 1))
            mx.kv_append(w["cache"], self._rotate(k, plan.positions), v, plan.slots)
            att, _ = mx.kv_attention(self._rotate(q, plan.positions), w["cache"], self.table, plan.ctx_len, plan.cu, max_new=max_new,
                                     want_lse=False)
            x = x + mx.mx_linear(att.flatten(1), w["out"])
            x = x + mx.gated_mlp_step(self._norm(x), w["gate"], w["up"], w["down"])
        return mx.mx_linear(self._norm(x), self.head), plan

    def release(self, done):
        mx.kv_release(done, self.lengths, self.cfg.page, self.table, self.free, self.free_count)


def generate(model, prompts, length, top_k=5):
    """Greedy continuations of `length` tokens; requests wait for a free slot.
    Returns, for each prompt, (tokens, log probabilities, entropies, alternatives)."""
    cfg, device = model.cfg, model.lengths.device
    waiting, running, results = list(range(len(prompts))), {}, {i: ([], [], [], []) for i in range(len(prompts))}
    feed = {}                                             # slot -> tokens to feed next
    while waiting or running:
        for slot in range(cfg.slots):
            if slot not in running and waiting:
                running[slot] = waiting.pop(0)
                feed[slot] = list(prompts[running[slot]])
        new = torch.tensor([len(feed.get(s, ())) for s in range(cfg.slots)], dtype=torch.int32, device=device)
        tokens = torch.tensor([t for s in range(cfg.slots) for t in feed.get(s, ())], dtype=torch.int32, device=device)
        logits, plan = model.step(tokens, new, max(len(f) for f in feed.values()))
        slots = sorted(running)
        last = logits[plan.cu[1:][slots].long() - 1]      # each request's last row
        best = last.argmax(1).to(torch.int32)
        r = mx.token_logprobs(last, best, top_k)
        assert int(plan.short) == 0, "the pool is out of pages"
        done = torch.zeros(cfg.slots, dtype=torch.bool, device=device)
        for i, slot in enumerate(slots):
            out = results[running[slot]]
            for dst, src in zip(out, (best, r.logp, r.entropy, r.top_ids)):
                dst.append(src[i].tolist())
            feed[slot] = [int(best[i])]
            if len(out[0]) == length:
                done[slot] = True
                del running[slot], feed[slot]
        if done.any():
            model.release(done)
    return results


def score(model, sequences):
    """Log probabilities and entropies of whole sequences (one slot each), as a
    rollout's update needs them, with the logits they came from."""
    cfg, device = model.cfg, model.lengths.device
    assert len(sequences) <= cfg.slots
    new = torch.tensor([len(s) for s in sequences] + [0] * (cfg.slots - len(sequences)), dtype=torch.int32, device=device)
    tokens = torch.tensor([t for s in sequences for t in s], dtype=torch.int32, device=device)
    logits, _ = model.step(tokens, new, max(map(len, sequences)))
    targets = torch.tensor([t for s in sequences for t in list(s[1:]) + [-1]], dtype=torch.int32, device=device)   # -1: no next token
    model.release(new > 0)
    return logits, targets


def main():
    cfg = Config()
    model = PagedDecoder(cfg)
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, cfg.vocab, (n,), generator=g).tolist() for n in (5, 300, 33, 1, 120, 64, 17, 250, 31, 90, 700)]
    results = generate(model, prompts, 24)
    for i, (tokens, logp, entropy, _) in results.items():
        print("request %2d: prompt %3d, first tokens %s, mean logp %.3f, mean entropy %.3f"
              % (i, len(prompts[i]), tokens[:4], sum(logp) / len(logp), sum(entropy) / len(entropy)))
    assert int(model.free_count) == cfg.pages             # every page came back
    # one policy-gradient step on the logits of what was generated
    logits, targets = score(model, [prompts[i] + results[i][0] for i in range(4)])
    logits.requires_grad_(True)
    logp, entropy = mx.token_logp(logits, targets)
    advantage = torch.randn(logp.shape, device=logp.device)
    (-(advantage * logp).sum() - 0.01 * entropy.sum()).backward()
    print("policy gradient: |dlogits| = %.4f over %d tokens" % (float(logits.grad.norm()), logits.shape[0]))


if __name__ == "__main__":
    main()
