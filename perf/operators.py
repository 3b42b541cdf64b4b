"""Timed cases of the serving operators: block tables and slot maps from request lengths (kv_plan), the paged 8-bit K/V
cache (kv_append, kv_read), attention over it (kv_attention) and the log probabilities of given tokens with their gradient
(token_logprobs, token_logprobs_grad).

`run` computes a case in plain torch operations in 32 bits, or, where `own` is true, with the library's own entry points.
The cache layout is the library's: int8 values in blocks of 32 tokens and one E8M0 scale (2^(byte - 127)) for each block
and head; K [page][head][block][32][D], V [page][head][block][D/2][4][2][8] with token 8j + 2c + b and dimension d of a
block at ((d / 2) * 4 + c, d % 2, 2j + b).
"""
import math
import random

import torch

own = False

BLOCK = 32
DEV = "cuda"


# ------------------------------------------------------------------ cases ---
def listed():
    return [
        # one decode step's block tables for a small serving batch: every launch of it is latency
        dict(name="plan_step32", op="plan", requests=32, past_lo=1, past_hi=2303, new_lo=1, new_hi=1, page=64, lens=11),
        # a full scheduler step: thousands of decoding requests with prompts among them
        dict(name="plan_mixed4096", op="plan", requests=4096, past_lo=1, past_hi=8191, new_lo=1, new_hi=97, page=32, lens=12),
        # the new K/V rows of a 32-sequence decode step of the 32-head decoder (fp32 rows, as the linears write them)
        dict(name="append_step32", op="append", requests=32, past_lo=1, past_hi=2303, new_lo=1, new_hi=1, kv_heads=32,
             head_dim=128, group=1, page=64, dtype="float32", lens=13),
        # prompts being cached: some whole, some continuing inside a block
        dict(name="append_prompts", op="append", requests=12, past_lo=0, past_hi=700, new_lo=700, new_hi=2300, kv_heads=8,
             head_dim=128, group=4, page=64, dtype="bfloat16", lens=14),
        # one user, one token: the smallest attention call
        dict(name="attend_one", op="attend", requests=1, ctx_lo=517, ctx_hi=517, new_lo=1, new_hi=1, kv_heads=32,
             head_dim=128, group=1, page=64, dtype="float32", lens=15),
        # the 32-head decoder's batch-32 decode step after a 2048-token prompt
        dict(name="attend_step32", op="attend", requests=32, ctx_lo=2049, ctx_hi=2304, new_lo=1, new_hi=1, kv_heads=32,
             head_dim=128, group=1, page=64, dtype="float32", lens=16),
        # a serving batch of very unequal requests, four query heads to a K/V head
        dict(name="attend_ragged192", op="attend", requests=192, ctx_lo=16, ctx_hi=8191, new_lo=1, new_hi=1, kv_heads=8,
             head_dim=128, group=4, page=32, dtype="bfloat16", lens=17),
        # two long documents being continued: few rows, a long axis to split
        dict(name="attend_long2", op="attend", requests=2, ctx_lo=100003, ctx_hi=131071, new_lo=1, new_hi=1, kv_heads=2,
             head_dim=64, group=8, page=128, dtype="float16", lens=18),
        # prompt chunks that continue cached prefixes
        dict(name="attend_prompts4", op="attend", requests=4, ctx_lo=1500, ctx_hi=4096, new_lo=900, new_hi=2048, kv_heads=8,
             head_dim=128, group=4, page=64, dtype="bfloat16", lens=19),
        # one sampled token of one request: its log probability, the entropy and the alternatives to show
        dict(name="logp_one", op="logp", rows=1, vocab=32000, pad=0, top_k=20, dtype="float32"),
        # rollout scoring: 16 rollouts of 512 tokens; the logits share their rows with a value head (stride vocab + 1)
        dict(name="logp_rollout", op="logp", rows=8192, vocab=32000, pad=1, top_k=5, dtype="float32"),
        # the policy update's gradient to the logits of as many tokens as 8 rollouts have
        dict(name="logp_grad", op="logp_grad", rows=4096, vocab=32000, pad=0, top_k=0, dtype="bfloat16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(max(lo, 1)), math.log(max(hi, 1)))))))) if hi > lo else lo


def draw(rng):
    op = rng.choice(["plan", "append", "attend", "attend", "logp", "logp_grad"])
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    page = rng.choice([32, 64, 128])
    lens = rng.randrange(1 << 20)
    if op == "plan":
        return dict(op=op, requests=_log_int(rng, 1, 4096), past_lo=0, past_hi=_log_int(rng, 32, 8191), new_lo=1,
                    new_hi=_log_int(rng, 1, 97), page=page, lens=lens)
    group, dim = rng.choice([1, 2, 4, 5, 8]), rng.choice([64, 128])
    if op == "append":
        kv_heads = rng.choice([1, 2, 4, 8, 32]) if rng.random() < 0.5 else rng.randint(1, 16)
        if rng.random() < 0.5:
            return dict(op=op, requests=_log_int(rng, 1, 512), past_lo=0, past_hi=2303, new_lo=1, new_hi=1, kv_heads=kv_heads,
                        head_dim=dim, group=group, page=page, dtype=dtype, lens=lens)
        return dict(op=op, requests=_log_int(rng, 1, 12), past_lo=0, past_hi=700, new_lo=2, new_hi=_log_int(rng, 3, 2300),
                    kv_heads=min(kv_heads, 8), head_dim=dim, group=min(group, 4), page=page, dtype=dtype, lens=lens)
    if op == "attend":
        kind = rng.choice(["step", "step", "few", "prompt"])
        if kind == "prompt":
            new = _log_int(rng, 33, 2048)
            return dict(op=op, requests=_log_int(rng, 1, 4), ctx_lo=new, ctx_hi=_log_int(rng, new, 4096), new_lo=max(1, new // 3),
                        new_hi=new, kv_heads=rng.randint(1, 8), head_dim=dim, group=rng.choice([1, 2, 4]), page=page, dtype=dtype, lens=lens)
        kv_heads = rng.choice([1, 2, 4, 8]) if group > 1 else rng.choice([4, 8, 16, 32])
        hi = _log_int(rng, 64, 16384)
        most = (32 * 2176 * 32) // (hi * kv_heads)
        return dict(op=op, requests=_log_int(rng, 1, max(1, min(256, most))), ctx_lo=max(8, hi // rng.choice([1, 2, 16, 256])), ctx_hi=hi,
                    new_lo=1, new_hi=1 if kind == "step" else rng.randint(2, 8), kv_heads=kv_heads, head_dim=dim, group=group,
                    page=page, dtype=dtype, lens=lens)
    vocab = rng.choice([32000, 32001, rng.randint(80, 2048), _log_int(rng, 4096, 131072)])
    size = 4 if dtype == "float32" else 2
    rows = _log_int(rng, 1, min(8192, (1 << 30) // (vocab * size) if op == "logp" else (1 << 28) // (vocab * size // 2)))
    return dict(op=op, rows=max(1, rows), vocab=vocab, pad=rng.choice([0, 0, 1]), top_k=rng.choice([0, 1, 5, 20]) if op == "logp" else 0,
                dtype=dtype)


def _lengths(case):
    """(past, new) of each request: they belong to the case, so that its work is known without the inputs."""
    r = random.Random(case["lens"])
    past, new = [], []
    for _ in range(case["requests"]):
        n = _log_int(r, case["new_lo"], case["new_hi"])
        if case["op"] == "attend":
            c = max(n, _log_int(r, case["ctx_lo"], case["ctx_hi"]))
            past.append(c - n)
        else:
            past.append(_log_int(r, case["past_lo"], case["past_hi"]))
        new.append(n)
    return past, new


def _size(dtype):
    return 4 if dtype == "float32" else 2


def _read_back(past, new):
    """Slots' positions that an append is read back at: every token of the touched blocks up to the last new one."""
    return [(r, t) for r, (p, n) in enumerate(zip(past, new)) for t in range(p // BLOCK * BLOCK, p + n)]


def work(case):
    op = case["op"]
    if op in ("plan", "append", "attend"):
        past, new = _lengths(case)
        n = sum(new)
    if op == "plan":
        p = case["page"]
        pages = sum(-(-(a + b) // p) - -(-a // p) for a, b in zip(past, new))
        old = sum(1 for a in past if a % p)
        return {"bytes": 4.0 * (2 * len(past) + pages * 2 + old + 2 * len(past) + 1 + 3 * n + 3), "flops": 0}
    if op == "append":
        values = 2 * case["kv_heads"] * case["head_dim"]
        back = len(_read_back(past, new))
        # rows in, 8-bit values out, and the read-back's 8-bit values in and 16-bit values out
        return {"bytes": float(n * values * (_size(case["dtype"]) + 1) + back * values * 3 + 4 * (n + back)), "flops": 0}
    if op == "attend":
        hq = case["kv_heads"] * case["group"]
        d = case["head_dim"]
        cached = sum(a + b for a, b in zip(past, new))
        blocks = sum(-(-(a + b) // BLOCK) for a, b in zip(past, new))
        pairs = sum(b * a + b * (b + 1) // 2 for a, b in zip(past, new))
        return {"bytes": float(cached * case["kv_heads"] * 2 * d + blocks * case["kv_heads"] * 2 + 2 * n * hq * d * _size(case["dtype"])
                               + 4 * n * hq),
                "flops": 4.0 * hq * d * pairs}
    e = case["rows"] * case["vocab"] * _size(case["dtype"])
    return {"bytes": float(e * (1 if op == "logp" else 2) + case["rows"] * (16 + 8 * case["top_k"])), "flops": 0}


# ----------------------------------------------------------------- inputs ---
def _pages(case, past, new, gen, upto_new):
    """A block table for the given lengths over a shuffled page pool, and what is left of the pool."""
    p = case["page"]
    held = [-(-(a + (b if upto_new else 0)) // p) for a, b in zip(past, new)]
    most = max(1, max(-(-(a + b) // p) for a, b in zip(past, new)))
    need = sum(-(-(a + b) // p) for a, b in zip(past, new))
    n_pages = need + 3
    pool = torch.randperm(n_pages, device=DEV, generator=gen).to(torch.int32)
    counts = torch.tensor(held, device=DEV)
    start = counts.cumsum(0) - counts
    col = torch.arange(most, device=DEV)
    idx = (start[:, None] + col).clamp(max=n_pages - 1)
    table = torch.where(col < counts[:, None], pool[idx], torch.full_like(pool[idx], -1))
    free = pool[sum(held):]
    return table.contiguous(), free, n_pages


def _dtype(case):
    return {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}[case["dtype"]]


def _cache(case, n_pages, gen):
    """A cache in use: values of normal K/V rows, scales that differ from block to block."""
    h, d, nb = case["kv_heads"], case["head_dim"], case["page"] // BLOCK
    out = {}
    for name, shape in (("k", (n_pages, h, nb, BLOCK, d)), ("v", (n_pages, h, nb, d // 2, 4, 2, 8))):
        x = torch.empty(shape, dtype=torch.int8, device=DEV)
        flat = x.view(n_pages, -1)
        step = max(1, (1 << 26) // flat.shape[1])
        for i in range(0, n_pages, step):
            part = flat[i:i + step]
            part.copy_((torch.randn(part.shape, device=DEV, generator=gen) * 31).round_().clamp_(-127, 127))
        out[name] = x
        out[name + "_scale"] = torch.randint(121, 124, (n_pages, h, nb), device=DEV, generator=gen, dtype=torch.uint8)
    return out


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed * 7919 + 17)
    st = {"case": dict(case)}
    op = case["op"]
    if op in ("plan", "append", "attend"):
        past, new = _lengths(case)
        st["past"] = torch.tensor(past, dtype=torch.int32, device=DEV)
        st["new"] = torch.tensor(new, dtype=torch.int32, device=DEV)
        st["n"] = sum(new)
        st["max_new"] = max(new)
        st["table"], free, n_pages = _pages(case, past, new, gen, op != "plan")
    if op == "plan":
        st["free"] = torch.cat([free, torch.full((n_pages - free.numel(),), -1, dtype=torch.int32, device=DEV)])
        st["free_count"] = torch.tensor([free.numel()], dtype=torch.int32, device=DEV)
        st["table"] = torch.where(st["table"] < 0, torch.full_like(st["table"], -1), st["table"])
        return st
    if op in ("append", "attend"):
        st["cache"] = _cache(case, n_pages, gen)
        hkv, hq, d = case["kv_heads"], case["kv_heads"] * case["group"], case["head_dim"]
        st["cu"] = torch.tensor([0] + new, device=DEV).cumsum(0).to(torch.int32)
        st["ctx"] = st["past"] + st["new"]
        if op == "attend":
            st["max_ctx"] = max(a + b for a, b in zip(past, new))
            st["q"] = torch.randn((st["n"], hq, d), device=DEV, generator=gen).to(_dtype(case))
            return st
        # the linear's fused [q | k | v] rows: K and V are strided views
        qkv = torch.randn((st["n"], (hq + 2 * hkv) * d), device=DEV, generator=gen)
        qkv *= torch.exp(0.5 * torch.randn((st["n"], 1), device=DEV, generator=gen))
        qkv = qkv.to(_dtype(case))
        st["k"] = qkv[:, hq * d:(hq + hkv) * d].unflatten(1, (hkv, d))
        st["v"] = qkv[:, (hq + hkv) * d:].unflatten(1, (hkv, d))
        req = torch.repeat_interleave(torch.arange(len(new), device=DEV), st["new"].long())
        pos = torch.arange(st["n"], device=DEV) - st["cu"][req] + st["past"][req]
        p = case["page"]
        st["slots"] = (st["table"][req, pos // p] * p + pos % p).to(torch.int32)
        first = st["past"].long() // BLOCK * BLOCK
        count = st["past"].long() + st["new"].long() - first
        req = torch.repeat_interleave(torch.arange(len(new), device=DEV), count)
        pos = torch.arange(req.numel(), device=DEV) - (count.cumsum(0) - count)[req] + first[req]
        st["back"] = (st["table"][req, pos // p] * p + pos % p).to(torch.int32)
        return st
    rows, vocab = case["rows"], case["vocab"]
    buf = torch.empty((rows, vocab + case["pad"]), dtype=_dtype(case), device=DEV)
    x = buf[:, :vocab]
    step = max(1, (1 << 27) // vocab)
    for i in range(0, rows, step):
        x[i:i + step] = torch.randn((min(step, rows - i), vocab), device=DEV, generator=gen) * 2
    st["targets"] = torch.randint(3, vocab, (rows,), device=DEV, generator=gen).to(torch.int32)
    sure = torch.rand((rows,), device=DEV, generator=gen) < 0.5     # half of the tokens are likely ones
    r = torch.arange(rows, device=DEV)
    x[r, st["targets"].long()] += torch.where(sure, 9.0, 0.0).to(x.dtype)
    x[:, :3] = -float("inf")                                        # tokens that may not be sampled
    if case["pad"]:
        buf[:, vocab:] = torch.randn((rows, case["pad"]), device=DEV, generator=gen).to(x.dtype)
    st["logits"] = x
    if op == "logp_grad":                                           # what the forward pass left, and the loss's gradients
        lse, ent = torch.empty(rows, device=DEV), torch.empty(rows, device=DEV)
        for i in range(0, rows, step):
            part = x[i:i + step].double()
            z = torch.logsumexp(part, 1)
            q = torch.exp(part - z[:, None])
            lse[i:i + step] = z.float()
            ent[i:i + step] = (z - (q * torch.where(q > 0, part, torch.zeros_like(part))).sum(1)).float()
        st["lse"], st["entropy"] = lse, ent
        st["dlogp"] = torch.randn(rows, device=DEV, generator=gen)
        st["dentropy"] = torch.randn(rows, device=DEV, generator=gen) * 0.01
    return st


# ---------------------------------------------------------------- a pass ---
def run(st):
    op = st["case"]["op"]
    if own:
        from cpu_model_b200 import mx
        return {"plan": _own_plan, "append": _own_append, "attend": _own_attend, "logp": _own_logp,
                "logp_grad": _own_grad}[op](mx, st)
    return {"plan": _plain_plan, "append": _plain_append, "attend": _plain_attend, "logp": _plain_logp,
            "logp_grad": _plain_grad}[op](st)


def _own_plan(mx, st):
    p = mx.kv_plan(st["past"], st["new"], st["case"]["page"], st["table"], st["free"], st["free_count"], st["n"])
    return {"table": st["table"], "ctx": p.ctx_len, "cu": p.cu, "slots": p.slots, "positions": p.positions,
            "requests": p.requests, "free_count": p.free_count, "short": p.short}


def _own_cache(mx, st):
    c = st["cache"]
    return mx.KVCache(c["k"], c["v"], c["k_scale"], c["v_scale"])


def _own_append(mx, st):
    cache = _own_cache(mx, st)
    mx.kv_append(cache, st["k"], st["v"], st["slots"])
    k, v = mx.kv_read(cache, st["back"], torch.bfloat16)
    return {"k": k, "v": v}


def _own_attend(mx, st):
    out, lse = mx.kv_attention(st["q"], _own_cache(mx, st), st["table"], st["ctx"], st["cu"], max_new=st["max_new"])
    return {"out": out, "lse": lse}


def _own_logp(mx, st):
    r = mx.token_logprobs(st["logits"], st["targets"], st["case"]["top_k"])
    out = {"logp": r.logp, "entropy": r.entropy, "lse": r.lse}
    if st["case"]["top_k"]:
        out |= {"top_logp": r.top_logp, "top_ids": r.top_ids}
    return out


def _own_grad(mx, st):
    return mx.token_logprobs_grad(st["logits"], st["targets"], st["lse"], st["entropy"], st["dlogp"], st["dentropy"])


def _plain_plan(st):
    p, table, free, count = st["case"]["page"], st["table"], st["free"], st["free_count"]
    n, r, width = st["n"], st["past"].numel(), st["table"].shape[1]
    past, new = st["past"].long(), st["new"].long().clamp(min=0)
    ctx = past + new
    have, full = (past + p - 1) // p, (ctx + p - 1) // p
    want = full.clamp(max=width) - have.clamp(max=width)
    first = want.cumsum(0) - want
    col = torch.arange(width, device=DEV)
    j = col - have[:, None]
    mine = (j >= 0) & (j < want[:, None])
    at = count.long() - 1 - (first[:, None] + j)
    page = torch.where(at >= 0, free[at.clamp(0, free.numel() - 1)], torch.full_like(table, -1))
    table.copy_(torch.where(mine, page, table))
    taken = torch.minimum(want.sum(), count.long()[0])
    ends = new.cumsum(0)
    cu = torch.cat([torch.zeros(1, dtype=torch.int64, device=DEV), ends])
    i = torch.arange(n, device=DEV)
    req = torch.searchsorted(ends, i, right=True)
    real = req < r
    req = req.clamp(max=r - 1)
    pos = i - cu[req] + past[req]
    page = torch.where(pos // p < width, table[req, (pos // p).clamp(max=width - 1)], torch.full_like(req, -1).int())
    slot = torch.where(real & (page >= 0), page * p + pos % p, torch.full_like(pos, -1))
    none = torch.full_like(pos, -1)
    return {"table": table, "ctx": ctx.int(), "cu": cu.int(), "slots": slot.int(), "positions": torch.where(real, pos, none).int(),
            "requests": torch.where(real, req, none).int(), "free_count": (count - taken).int(),
            "short": ((full - have).sum() - taken).int().reshape(1)}


def _pack_v(x):
    """[..., 32, D] -> [..., D/2, 4, 2, 8], the order of a V block."""
    s = x.shape[:-2]
    y = x.reshape(*s, 4, 4, 2, x.shape[-1] // 2, 2)
    k = len(s)
    return y.permute(*range(k), k + 3, k + 1, k + 4, k, k + 2).reshape(*s, x.shape[-1] // 2, 4, 2, 8)


def _unpack_v(x):
    """[..., D/2, 4, 2, 8] -> [..., 32, D]."""
    s = x.shape[:-4]
    y = x.reshape(*s, x.shape[-4], 4, 2, 4, 2)
    k = len(s)
    return y.permute(*range(k), k + 3, k + 1, k + 4, k, k + 2).reshape(*s, 32, x.shape[-4] * 2)


def _two(e):
    """2^e in 32 bits, e >= -149."""
    return torch.ldexp(torch.ones((), device=DEV), e)


def _plain_append(st):
    c, slots = st["cache"], st["slots"].long()
    nb, h, d, n = st["case"]["page"] // BLOCK, st["case"]["kv_heads"], st["case"]["head_dim"], st["n"]
    blk = slots // BLOCK
    lead = torch.cat([torch.ones(1, dtype=torch.bool, device=DEV), blk[1:] != blk[:-1]])
    grp = lead.cumsum(0) - 1
    head = torch.nonzero(lead).reshape(-1)
    g = head.numel()
    gblk = blk[head]
    page, b = gblk // nb, gblk % nb
    fresh = slots[head] % BLOCK == 0
    back = st["back"].long()
    res = {}
    for name in ("k", "v"):
        x = st[name].float()
        top = torch.zeros((g, h), device=DEV).index_reduce_(0, grp, x.abs().amax(-1), "amax")
        m, e = torch.frexp(top)
        e = torch.where(top > 0, torch.where(m <= 0.9921875, e - 7, e - 6).clamp(min=-127), torch.full_like(e, -127))
        old = c[name + "_scale"][page, :, b].int() - 127
        e = torch.where(fresh[:, None], e, torch.maximum(e, old))
        vals = c[name][page, :, b]                              # [g][h][block]
        vals = (_unpack_v(vals) if name == "v" else vals).float()
        vals = torch.round(vals * _two((old - e).clamp(-140, 0))[:, :, None, None])
        vals[grp, :, slots % BLOCK] = torch.round(x * _two(-e)[grp][:, :, None])
        q = vals.to(torch.int8)
        c[name][page, :, b] = _pack_v(q) if name == "v" else q
        c[name + "_scale"][page, :, b] = (e + 127).to(torch.uint8)
        rb = back // BLOCK
        # the cache read back at every token of the touched blocks up to the last new one
        got = c[name][rb // nb, :, rb % nb]
        got = (_unpack_v(got) if name == "v" else got)[torch.arange(rb.numel(), device=DEV), :, back % BLOCK].float()
        res[name] = (got * _two(c[name + "_scale"][rb // nb, :, rb % nb].int() - 127)[:, :, None]).to(torch.bfloat16)
    return res


def _plain_attend(st):
    c, case = st["cache"], st["case"]
    q, cu, ctx = st["q"], st["cu"].long(), st["ctx"].long()
    p, hkv, grp, d, t = case["page"], case["kv_heads"], case["group"], case["head_dim"], st["max_new"]
    r, n = ctx.numel(), q.shape[0]
    pages = st["table"][:, :-(-st["max_ctx"] // p)].long().clamp(min=0)
    length = pages.shape[1] * p

    def rows(name):
        v = c[name][pages]                                     # [r][pages][h][blocks][...]
        v = (_unpack_v(v) if name == "v" else v).float()
        v *= _two(c[name + "_scale"][pages].int() - 127)[..., None, None]
        return v.permute(0, 2, 1, 3, 4, 5).reshape(r, hkv, length, d)

    new = cu[1:] - cu[:-1]
    tt = torch.arange(t, device=DEV)
    at = (cu[:-1, None] + tt).clamp(max=n - 1)
    qr = q[at].float().reshape(r, t, hkv, grp, d).permute(0, 2, 1, 3, 4).reshape(r, hkv, t * grp, d)
    s = torch.matmul(qr, rows("k").transpose(2, 3)) * (1.0 / math.sqrt(d))
    last = (ctx - new)[:, None] + tt                           # the last key that a row sees
    seen = torch.arange(length, device=DEV) <= last.repeat_interleave(grp, 1)[:, None, :, None]
    s = torch.where(seen, s, torch.full((), -float("inf"), device=DEV))
    m = s.amax(-1, keepdim=True)
    s = torch.exp(s - m)
    z = s.sum(-1, keepdim=True)
    o = torch.matmul(s, rows("v")) / z
    lse = (m + torch.log(z))[..., 0]
    valid = tt < new[:, None]
    o = o.reshape(r, hkv, t, grp, d).permute(0, 2, 1, 3, 4).reshape(r, t, hkv * grp, d)[valid]
    lse = lse.reshape(r, hkv, t, grp).permute(0, 2, 1, 3).reshape(r, t, hkv * grp)[valid]
    return {"out": o.to(q.dtype), "lse": lse}


def _plain_logp(st):
    x, k = st["logits"].float(), st["case"]["top_k"]
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(1, keepdim=True)
    lse = (m + torch.log(z))[:, 0]
    ent = lse - (e * torch.where(e > 0, x, torch.zeros_like(x))).sum(1) / z[:, 0]
    out = {"logp": x.gather(1, st["targets"].long()[:, None])[:, 0] - lse, "entropy": ent, "lse": lse}
    if k:
        top, ids = torch.sort(x, dim=1, descending=True, stable=True)
        out |= {"top_logp": top[:, :k] - lse[:, None], "top_ids": ids[:, :k].int()}
    return out


def _plain_grad(st):
    x = st["logits"].float() - st["lse"][:, None]
    p = torch.exp(x)
    hit = torch.arange(x.shape[1], device=DEV) == st["targets"][:, None]
    g = st["dlogp"][:, None] * (hit.float() - p)
    g -= st["dentropy"][:, None] * p * (torch.where(p > 0, x, torch.zeros_like(x)) + st["entropy"][:, None])
    return g.to(st["logits"].dtype)


# --------------------------------------------------------- in 64 bits -----
def exact(case, seed):
    op = case["op"]
    if op == "plan":
        return None                                            # whole numbers only
    st = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "logp": _exact_logp, "logp_grad": _exact_grad}[op](st)


def _exact_append(st):
    """Block by block, on the values themselves: what each block holds, rounded to its own step."""
    case, c = st["case"], st["cache"]
    nb, p, h, d = case["page"] // BLOCK, case["page"], case["kv_heads"], case["head_dim"]
    past, new = _lengths(case)
    res = {"k": [], "v": []}
    table = st["table"].tolist()
    tok = torch.arange(BLOCK, device=DEV)
    dim = torch.arange(d, device=DEV)
    where_v = (((dim // 2)[None, :] * 4 + (tok // 2 % 4)[:, None]) * 2 + (dim % 2)[None, :]) * 8 + (tok // 8 * 2 + tok % 2)[:, None]
    at = 0
    for r, (a, n) in enumerate(zip(past, new)):
        for b in range(a // BLOCK, (a + n - 1) // BLOCK + 1):
            lo, hi = max(a, b * BLOCK) - b * BLOCK, min(a + n, (b + 1) * BLOCK) - b * BLOCK
            pg, sub = table[r][b * BLOCK // p], b % nb
            for name in ("k", "v"):
                rows = st[name][at:at + hi - lo].double().transpose(0, 1)          # [h][new][d]
                m, x = torch.frexp(rows.abs().amax((1, 2)) / 127.0)
                e = torch.where(m == 0.5, x - 1, x).clamp(min=-127)
                held = c[name][pg, :, sub].reshape(h, -1)
                held = (held[:, where_v] if name == "v" else held.reshape(h, BLOCK, d)).double()[:, :lo]
                if lo:
                    was = c[name + "_scale"][pg, :, sub].int() - 127
                    held = held * torch.exp2(was.double())[:, None, None]
                    e = torch.maximum(e, was)
                step = torch.exp2(e.double())[:, None, None]
                both = torch.cat([held, rows], 1)
                res[name].append((torch.round(both / step) * step).transpose(0, 1))
            at += hi - lo
    return {n: torch.cat(v) for n, v in res.items()}


def _exact_attend(st):
    case, c = st["case"], st["cache"]
    past, new = _lengths(case)
    grp, d, p = case["group"], case["head_dim"], case["page"]
    outs, lses, at = [], [], 0
    d_ = torch.arange(d, device=DEV)
    t_ = torch.arange(BLOCK, device=DEV)
    where_v = (((d_ // 2)[None, :] * 4 + (t_ // 2 % 4)[:, None]) * 2 + (d_ % 2)[None, :]) * 8 + (t_ // 8 * 2 + t_ % 2)[:, None]
    for r, (a, n) in enumerate(zip(past, new)):
        ids = st["table"][r, :-(-(a + n) // p)].long()
        out = torch.empty((n, case["kv_heads"] * grp, d), dtype=torch.float64, device=DEV)
        lse = torch.empty((n, case["kv_heads"] * grp), dtype=torch.float64, device=DEV)
        for h in range(case["kv_heads"]):
            ks = torch.exp2(c["k_scale"][ids, h].double() - 127)[..., None, None]
            vs = torch.exp2(c["v_scale"][ids, h].double() - 127)[..., None, None]
            k = (c["k"][ids, h].double() * ks).reshape(-1, d)[:a + n]
            v = (c["v"][ids, h].flatten(2)[:, :, where_v].double() * vs).reshape(-1, d)[:a + n]
            for i in range(0, n, 256):
                q = st["q"][at + i:at + min(n, i + 256), h * grp:(h + 1) * grp].double()
                s = torch.einsum("tgd,ld->tgl", q, k) / math.sqrt(d)
                row = torch.arange(a + i, a + i + q.shape[0], device=DEV)
                s.masked_fill_(torch.arange(a + n, device=DEV)[None, None, :] > row[:, None, None], -float("inf"))
                lse[i:i + q.shape[0], h * grp:(h + 1) * grp] = torch.logsumexp(s, -1)
                out[i:i + q.shape[0], h * grp:(h + 1) * grp] = torch.softmax(s, -1) @ v
        outs.append(out)
        lses.append(lse)
        at += n
    return {"out": torch.cat(outs), "lse": torch.cat(lses)}


def _exact_logp(st):
    x, k = st["logits"], st["case"]["top_k"]
    step = max(1, (1 << 27) // x.shape[1])
    got = []
    for i in range(0, x.shape[0], step):
        lp = torch.log_softmax(x[i:i + step].double(), 1)
        t = st["targets"][i:i + step].long()[:, None]
        ent = -torch.special.xlogy(lp.exp(), lp.exp()).sum(1)
        got.append((lp.gather(1, t)[:, 0], ent, torch.logsumexp(x[i:i + step].double(), 1),
                    torch.topk(lp, k, dim=1).values if k else None))
    logp, ent, lse = (torch.cat([g[j] for g in got]) for j in range(3))
    out = {"logp": logp, "entropy": ent, "lse": lse}
    if k:
        out |= {"top_logp": torch.cat([g[3] for g in got]), "top_ids": None}
    return out


def _exact_grad(st):
    x = st["logits"]
    step = max(1, (1 << 26) // x.shape[1])
    out = []
    for i in range(0, x.shape[0], step):
        lp = torch.log_softmax(x[i:i + step].double(), 1)
        p = lp.exp()
        lp = torch.where(p > 0, lp, torch.zeros_like(lp))
        ent = -(p * lp).sum(1, keepdim=True)
        g = -p * st["dlogp"][i:i + step].double()[:, None]
        g.scatter_add_(1, st["targets"][i:i + step].long()[:, None], st["dlogp"][i:i + step].double()[:, None])
        out.append(g - st["dentropy"][i:i + step].double()[:, None] * p * (lp + ent))
    return torch.cat(out)
