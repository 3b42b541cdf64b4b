"""Attention over the paged 8-bit cache against the formula in 64 bits.

Tolerances, from the number formats.  fp32 rows: the products are exact sums
of integers; what rounds is the query's fixed point (2^-23 of its largest
element), a score (a few 2^-24 of |s| <= 50 gives 1e-5 in exp at most) and
the probabilities (2^-23 of a block's largest): relative 2-norm 1e-5, the
bound of the other fp32 results.  bf16 / fp16 rows: the result's own rounding is below
2^-9 / 2^-12 in the 2-norm (2^-8 / 2^-11 at most of an element, evenly spread); the probabilities' second digit adds 2^-16 and the
query's 15 bits an error of s below 2^-16 max|q| sum|k| scale, about 1e-4 here:
2^-9 + 2e-4 and 2^-12 + 4e-4.  lse: 2e-6 |lse| + 2e-6 in fp32, that error
of s (5e-4 bounds it) in 16 bits."""
import ctypes

import numpy as np
import pytest
import torch

from cpu_model_b200 import mx, synth

pytestmark = pytest.mark.gpu

TOL = {torch.float32: 1e-5, torch.bfloat16: 2.0 ** -9 + 2e-4, torch.float16: 2.0 ** -12 + 4e-4}


def v_index(D):
    t, d = torch.arange(32)[:, None], torch.arange(D)[None, :]
    return ((d >> 1) * 4 + (t >> 1) % 4) * 16 + (d & 1) * 8 + (t >> 3) * 2 + (t & 1)


class Case:
    def __init__(self, spans, Hkv, G, D, P, dtype, seed=1, extra_rows=0, wide=0, q_pad=0, spread=3):
        """spans: (ctx, new) of each request."""
        g = synth.rng(seed)
        self.D, self.Hkv, self.G, self.P, self.dtype = D, Hkv, G, P, dtype
        self.ctx = [c for c, _ in spans]
        self.new = [n for _, n in spans]
        nb = P // 32
        pages = [max(0, -(-c // P)) for c in self.ctx]
        n_pages = max(1, sum(pages) + 2)
        ids = g.permutation(n_pages)
        width = max(1, max(pages) + wide)
        table = np.full((len(spans), width), -1, np.int32)
        at = 0
        for r, n in enumerate(pages):
            table[r, :n] = ids[at:at + n]
            at += n
        gen = torch.Generator(device="cuda").manual_seed(seed)
        rnd = lambda *s: torch.randn(s, device="cuda", generator=gen)
        self.k = (rnd(n_pages, Hkv, nb, 32, D) * 31).round().clamp(-127, 127).to(torch.int8)
        self.v = (rnd(n_pages, Hkv, nb, D // 2, 4, 2, 8) * 31).round().clamp(-127, 127).to(torch.int8)
        self.ks = torch.randint(124 - spread, 124, (n_pages, Hkv, nb), device="cuda", generator=gen, dtype=torch.uint8)
        self.vs = torch.randint(124 - spread, 124, (n_pages, Hkv, nb), device="cuda", generator=gen, dtype=torch.uint8)
        self.table = torch.as_tensor(table, device="cuda")
        n = sum(self.new) + extra_rows
        buf = rnd(n, Hkv * G * D + q_pad).to(dtype)
        self.q = buf[:, q_pad:].unflatten(1, (Hkv * G, D))
        self.cu = torch.tensor([0] + list(np.cumsum(self.new)), dtype=torch.int32, device="cuda")
        self.ctx_len = torch.tensor(self.ctx, dtype=torch.int32, device="cuda")

    def cache(self):
        return mx.KVCache(self.k, self.v, self.ks, self.vs)

    def run(self, ctx, **kw):
        kw.setdefault("max_new", max(1, max(self.new)))
        return mx.kv_attention(self.q, self.cache(), self.table, self.ctx_len, self.cu, ctx=ctx, **kw)

    def dense(self, r, h, length):
        """K, V of a request and head in 64 bits; pages that are not there are marked."""
        D, P = self.D, self.P
        ids = self.table[r, :-(-length // P)].long()
        there = ((ids >= 0) & (ids < self.k.shape[0])).repeat_interleave(P)[:length]
        ids = ids.clamp(0, self.k.shape[0] - 1)
        two = lambda s: torch.where(s == 255, torch.full((), float("nan"), dtype=torch.float64, device="cuda"), torch.exp2(s.double() - 127))
        k = (self.k[ids, h].double() * two(self.ks[ids, h])[..., None, None]).reshape(-1, D)[:length]
        v = self.v[ids, h].flatten(2)[:, :, v_index(D).cuda()].double() * two(self.vs[ids, h])[..., None, None]
        return k, v.reshape(-1, D)[:length], there

    def ref(self, scale=None):
        scale = self.D ** -0.5 if scale is None else scale
        n, Hq = self.q.shape[:2]
        out = torch.zeros((n, Hq, self.D), dtype=torch.float64, device="cuda")
        lse = torch.full((n, Hq), -float("inf"), dtype=torch.float64, device="cuda")
        for r, (c, t) in enumerate(zip(self.ctx, self.new)):
            if t == 0 or c <= 0:
                continue
            a = int(self.cu[r])
            last = torch.arange(c - t, c, device="cuda")
            for h in range(self.Hkv):
                k, v, there = self.dense(r, h, c)
                q = self.q[a:a + t, h * self.G:(h + 1) * self.G].double()
                s = torch.einsum("tgd,ld->tgl", q, k) * scale
                see = (torch.arange(c, device="cuda")[None, :] <= last[:, None]) & there
                s = torch.where(see[:, None, :], s, torch.full_like(s, -float("inf")))
                some = see.any(1)[:, None].expand(-1, self.G)
                p = torch.softmax(s, -1)
                p = torch.where(some[..., None], p, torch.zeros_like(p))
                v = torch.where(there[:, None], v, torch.zeros_like(v))
                out[a:a + t, h * self.G:(h + 1) * self.G] = p @ v
                lse[a:a + t, h * self.G:(h + 1) * self.G] = torch.where(some, torch.logsumexp(s, -1), torch.full_like(lse[:1, :1], -float("inf")))
        return out, lse

    def check(self, ctx, **kw):
        out, lse = self.run(ctx, **kw)
        ctx.synchronize()
        want, wl = self.ref(kw.get("scale"))
        assert out.dtype == self.dtype and out.shape == want.shape
        assert torch.isfinite(out).all()
        err = float((out.double() - want).norm() / max(float(want.norm()), 1e-300))
        assert err <= TOL[self.dtype], err
        assert ((lse == -float("inf")) == (wl == -float("inf"))).all()
        fin = torch.isfinite(wl)
        tol = 2e-6 * wl[fin].abs() + 2e-6 if self.dtype == torch.float32 else 5e-4
        assert ((lse[fin].double() - wl[fin]).abs() <= tol).all()
        # every element, not the norm alone: rows of the smallest norm too
        rows = want.flatten(0, 1).norm(dim=1)
        some = rows > 0
        by_row = (out.double() - want).flatten(0, 1).norm(dim=1)[some] / rows[some]
        if some.any():
            assert float(by_row.max()) <= 4 * TOL[self.dtype]
        assert (out.flatten(0, 1)[~some] == 0).all()
        return out, lse


DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("spans", [
    [(1, 1)], [(2, 1)], [(31, 1)], [(32, 1)], [(33, 1)], [(517, 1)], [(5, 5)], [(300, 1), (1, 1), (64, 1), (1000, 1)]])
@pytest.mark.parametrize("Hkv,G", [(1, 1), (2, 4), (3, 8)])
def test_single_tokens(ctx, spans, Hkv, G, D, dtype):
    Case(spans, Hkv, G, D, 32, dtype).check(ctx)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,P", [(64, 128), (128, 64)])
@pytest.mark.parametrize("Hkv,G,spans", [
    (2, 5, [(100, 2), (40, 3), (7, 7)]),             # an odd group, tiles that end inside a token's heads
    (1, 8, [(200, 2), (90, 1), (4, 4)]),
    (4, 1, [(70, 9), (70, 16), (70, 17), (33, 33)]),
    (2, 3, [(500, 40), (129, 129), (64, 1)]),
    (1, 16, [(333, 1), (64, 5)]),
    (2, 4, [(257, 257), (600, 100)])])
def test_several_new_tokens(ctx, Hkv, G, spans, D, P, dtype):
    Case(spans, Hkv, G, D, P, dtype, seed=3).check(ctx)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_unequal_requests(ctx, dtype):
    g = synth.rng(8)
    spans = [(int(np.exp(g.uniform(0, np.log(1500)))), 1) for _ in range(150)]
    Case(spans, 2, 4, 128, 64, dtype, seed=5).check(ctx)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_long_context_over_many_ctas(ctx, dtype):
    Case([(20011, 1), (9000, 2)], 1, 4, 64, 128, dtype, seed=6).check(ctx)


def test_heads_of_the_decoder(ctx):
    Case([(2304, 1), (2049, 1), (700, 1)], 32, 1, 128, 64, torch.float32, seed=7).check(ctx)


def test_prompt_chunks(ctx):
    for dtype in DTYPES:
        Case([(700, 300), (1000, 512), (130, 130)], 2, 4, 128, 64, dtype, seed=8).check(ctx)


# enough rows for the tensor cores' kernel (32 units of 256 rows a K/V head)
LONG = {
    "even": (8, 4, [(512, 512), (1024, 512)]),
    "ragged": (8, 4, [(700, 300), (1000, 513), (130, 130), (40, 3), (900, 1), (5, 5), (0, 0), (300, 17)]),
    "heads": (32, 1, [(300, 300), (77, 33)]),
    "odd_group": (4, 5, [(1500, 500), (333, 299)]),
    "wide_group": (2, 16, [(257, 257), (500, 129)]),
    "one_page": (16, 8, [(64, 64), (31, 31), (128, 127)])}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,P", [(128, 64), (64, 32), (128, 256)])
@pytest.mark.parametrize("name", sorted(LONG))
def test_prompts_on_the_tensor_cores(ctx, name, D, P, dtype):
    Hkv, G, spans = LONG[name]
    Case(spans, Hkv, G, D, P, dtype, seed=31, extra_rows=2, q_pad=64, wide=1).check(ctx)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_prompts_with_missing_pages_and_rows_without_keys(ctx, dtype):
    c = Case([(600, 400), (300, 500), (256, 256), (0, 90), (-3, 40)], 8, 4, 128, 32, dtype, seed=32)
    c.table[0, 3] = -1
    c.table[0, 18] = 10 ** 8
    c.table[2, 0] = -1                               # the first rows see no key at all
    c.table[2, 7] = -5
    c.check(ctx)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_prompts_with_scales(ctx, dtype):
    c = Case([(600, 600), (300, 200)], 8, 4, 64, 64, dtype, seed=33, spread=10)
    c.check(ctx)
    c.check(ctx, scale=0.0)
    c.check(ctx, scale=-0.125)
    c.vs[:, 1] = 0                                   # blocks of zeros have the smallest scale
    c.v[:, 1] = 0
    c.check(ctx)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_prompts_with_v_scales_too_far_apart_for_fp16(ctx, dtype):
    """Exponents of V more than 2^32 apart: that unit's P is bf16, 8 bits (2^-9
    in the 2-norm), beside the result's rounding."""
    c = Case([(600, 600), (300, 200)], 8, 4, 128, 64, dtype, seed=40)
    c.vs[:, 1, 1] -= 70                              # head 1: every other block tiny
    c.vs[int(c.table[1, 0]), 2, :] = 250             # head 2 of request 1: two blocks huge
    c.vs[int(c.table[1, 1]), 3, 0] = 1
    out, lse = c.run(ctx)
    want, wl = c.ref()
    assert torch.isfinite(lse).all() and ((lse.double() - wl).abs() <= 5e-4).all()
    tol = (TOL[dtype] ** 2 + 2.0 ** -18) ** 0.5
    for h in range(8):
        for a, b in ((0, 600), (600, 800)):
            g, w = out[a:b, 4 * h:4 * h + 4].double(), want[a:b, 4 * h:4 * h + 4]
            if dtype == torch.float16 and float(w.abs().max()) > 65504:
                continue
            assert float((g - w).norm() / w.norm()) <= tol, (h, a)


def test_prompts_with_nan_in_masked_places(ctx):
    c = Case([(512, 512)], 8, 8, 128, 128, torch.bfloat16, seed=34)
    want, wl = c.ref()
    pg = int(c.table[0, 2])                          # keys 256 .. 383
    c.ks[pg, 0, 1] = 255                             # head 0: keys 288 .. 319
    c.vs[pg, 1, 3] = 255                             # head 1: keys 352 .. 383
    out, lse = c.run(ctx)
    tol = TOL[torch.bfloat16]
    near = lambda a, b: float((a.double() - b).norm() / b.norm()) <= tol
    assert near(out[:288, :8], want[:288, :8]) and torch.isnan(out[319:, :8]).all() and torch.isnan(lse[319:, :8]).all()
    assert near(out[:352, 8:16], want[:352, 8:16]) and torch.isnan(out[384:, 8:16]).all()
    assert near(out[:, 16:], want[:, 16:])
    c = Case([(512, 512)], 8, 8, 128, 128, torch.float16, seed=35)
    want, _ = c.ref()
    c.q[100, 5, 7] = float("inf")
    out, lse = c.run(ctx)
    assert torch.isnan(out[100, 5]).all()
    keep = torch.ones((512, 64), dtype=torch.bool)
    keep[100, 5] = False
    assert float((out[keep].double() - want[keep]).norm() / want[keep].norm()) <= TOL[torch.float16]


def test_prompts_repeat_and_run_on_two_streams(ctx):
    cs = [Case([(900, 700), (1300, 1000 + i)], 8, 2, 128, 64, torch.bfloat16, seed=36 + i) for i in range(2)]
    want = [c.run(ctx) for c in cs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for i in range(12):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(cs[i % 2].run(ctx))
    torch.cuda.synchronize()
    for i, (o, l) in enumerate(outs):
        assert torch.equal(o, want[i % 2][0]) and torch.equal(l, want[i % 2][1])


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_that_see_nothing(ctx, dtype):
    """No new rows, no context, fewer keys than rows, rows of no request,
    pages that are not there."""
    c = Case([(0, 0), (50, 0), (0, 3), (40, 2), (3, 6), (-5, 1)], 2, 2, 64, 32, dtype, extra_rows=4, wide=2)
    c.check(ctx)
    c = Case([(100, 1), (160, 3)], 1, 4, 128, 32, dtype)
    c.table[0, 1] = -1
    c.table[1, 0] = 10 ** 6
    c.check(ctx)
    c.table[0, :] = -1                               # a request with no page at all
    c.check(ctx)
    c.table = c.table[:, :1].contiguous()            # a table narrower than the lengths
    out, lse = c.run(ctx)
    assert torch.isfinite(out).all() and (out[0] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_rows_and_offsets(ctx, dtype):
    Case([(90, 3), (200, 1)], 2, 2, 128, 64, dtype, q_pad=64, wide=3).check(ctx)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scale_and_wide_scores(ctx, dtype):
    """Scores far apart: the running maximum rises by hundreds, and falls away."""
    c = Case([(400, 1), (97, 4)], 2, 2, 64, 32, dtype, seed=12, spread=12)
    c.check(ctx, scale=0.01)
    c.check(ctx, scale=0.0)
    if dtype == torch.float32:
        out, lse = c.run(ctx, scale=2.0)             # |s| to 1e4: exp's argument keeps 2^-24 of it
        want, wl = c.ref(2.0)
        assert float((out.double() - want).norm() / want.norm()) <= 1e-2 and torch.isfinite(out).all()


def test_nan_and_infinity_in_masked_places(ctx):
    """Garbage in pages past a length, in keys after a row and in other heads'
    blocks does not reach a row; a NaN that a row attends to does."""
    c = Case([(45, 1), (64, 20)], 2, 2, 64, 64, torch.float32, seed=13)
    want, wl = c.ref()
    spare = [p for p in range(c.k.shape[0]) if p not in c.table.flatten().tolist()]
    c.ks[spare] = 255
    c.vs[spare] = 255
    out, lse = c.run(ctx)
    assert float((out.double() - want).norm() / want.norm()) <= 1e-5
    # request 1's second block (keys 32..63) is NaN for head 0 (K) and head 1 (V); rows 44 .. 63 see it, request 0 does not
    pg = int(c.table[1, 0])
    c.ks[pg, 0, 1] = 255
    c.vs[pg, 1, 1] = 255
    out, lse = c.run(ctx)
    assert torch.isnan(out[1:]).all() and torch.isnan(lse[1:, :2]).all() and torch.isfinite(lse[1:, 2:]).all()
    assert float((out[0].double() - want[0]).norm() / want[0].norm()) <= 1e-5
    # rows before the block are untouched by it
    c = Case([(64, 64)], 1, 2, 64, 64, torch.float32, seed=14)
    want, _ = c.ref()
    c.ks[int(c.table[0, 0]), 0, 1] = 255
    c.vs[int(c.table[0, 0]), 0, 1] = 255
    out, lse = c.run(ctx)
    assert float((out[:32].double() - want[:32]).norm() / want[:32].norm()) <= 1e-5 and torch.isnan(out[32:]).all()


def test_nan_in_a_query_row(ctx):
    c = Case([(100, 3)], 1, 2, 64, 32, torch.float32, seed=15)
    want, _ = c.ref()
    c.q[1, 1, 5] = float("inf")
    out, lse = c.run(ctx)
    assert torch.isnan(out[1, 1]).all() and torch.isnan(lse[1, 1])
    keep = torch.ones((3, 2), dtype=torch.bool)
    keep[1, 1] = False
    assert float((out[keep].double() - want[keep]).norm() / want[keep].norm()) <= 1e-5


def test_tiny_and_huge_values(ctx):
    """Scales at the ends of E8M0's range and query rows near fp32's."""
    c = Case([(70, 1)], 1, 2, 64, 32, torch.float32, seed=16)
    c.ks[:] = 7
    c.q.mul_(2.0 ** 100)
    c.vs[:] = 200
    c.check(ctx)
    c.ks[:] = 220
    c.q.mul_(2.0 ** -197)
    c.vs[:] = 30
    c.check(ctx)
    c.q.zero_()
    c.check(ctx)


def test_repeats_are_bit_identical(ctx):
    c = Case([(5000, 1), (37, 1), (900, 3)], 2, 4, 128, 64, torch.bfloat16, seed=17)
    a, la = c.run(ctx)
    for _ in range(5):
        b, lb = c.run(ctx)
        assert torch.equal(a, b) and torch.equal(la, lb)


def test_max_new_is_only_a_hint_above(ctx):
    c = Case([(500, 1), (37, 1)], 2, 4, 128, 64, torch.float32, seed=18)
    a, _ = c.run(ctx)
    b, _ = c.run(ctx, max_new=1000)
    assert float((a - b).norm() / a.norm()) <= 1e-5
    out, none = c.run(ctx, want_lse=False)
    assert none is None and torch.equal(out, a)


def test_on_two_streams(ctx):
    """Split tiles meet in a workspace: one for each stream."""
    cs = [Case([(9000 + 500 * i, 1)], 2, 2, 128, 64, torch.bfloat16, seed=20 + i) for i in range(2)]
    want = [c.run(ctx)[0] for c in cs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for i in range(40):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(cs[i % 2].run(ctx)[0])
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        assert torch.equal(o, want[i % 2])


def test_in_a_cuda_graph(ctx):
    c = Case([(3000, 1), (200, 1)], 2, 4, 128, 64, torch.bfloat16, seed=25)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        want = c.run(ctx)[0]                         # makes the stream's workspace
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out, _ = c.run(ctx)
    c.q.copy_(c.q.flip(0))
    g.replay()
    torch.cuda.synchronize()
    again = c.run(ctx)[0]
    assert torch.equal(out, again) and not torch.equal(out, want)


def test_append_then_attend(ctx):
    """Rows that were appended are the rows that are attended to: the result
    is that of the quantised rows, and near the unquantised one's."""
    g = synth.rng(30)
    P, H, G, D, T = 32, 2, 2, 64, 150
    cache = mx.KVCache.empty(8, P, H, D)
    k = torch.randn((T, H, D), device="cuda")
    v = torch.randn((T, H, D), device="cuda")
    q = torch.randn((T, H * G, D), device="cuda")
    table = torch.as_tensor(g.permutation(8)[:5][None].astype(np.int32), device="cuda")
    lens = torch.zeros(1, dtype=torch.int32, device="cuda")
    free, count = torch.zeros(8, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    full = torch.full((1, 5), -1, dtype=torch.int32, device="cuda")
    free[:5] = table[0].flip(0)
    count += 5
    outs = []
    for a, b in ((0, 100), (100, 101), (101, 102), (102, 150)):
        add = torch.tensor([b - a], dtype=torch.int32, device="cuda")
        p = mx.kv_plan(lens, add, P, full, free, count, b - a, in_place=True, ctx=ctx)
        mx.kv_append(cache, k[a:b], v[a:b], p.slots, ctx=ctx)
        outs.append(mx.kv_attention(q[a:b], cache, full, p.ctx_len, p.cu, ctx=ctx)[0])
    assert torch.equal(full, table)
    out = torch.cat(outs).double()
    kk, vv = k.double().repeat_interleave(G, 1), v.double().repeat_interleave(G, 1)
    s = torch.einsum("thd,lhd->htl", q.double(), kk) / 8.0
    s.masked_fill_(torch.ones(T, T, dtype=torch.bool, device="cuda").triu(1), -float("inf"))
    want = torch.einsum("htl,lhd->thd", torch.softmax(s, -1), vv)
    # int8 steps of 2^-5 (a block's maximum is below 4): values move by at most 2^-6,
    # scores by 2^-6 / sqrt(3) * |q| / 8 ~ 0.009 one sigma; a few per cent bound it
    assert float((out - want).norm() / want.norm()) <= 0.05


def test_refusals(ctx):
    c = Case([(40, 1)], 2, 2, 64, 32, torch.float32)
    ok = dict(q=c.q, cache=c.cache(), table=c.table, ctx_len=c.ctx_len, cu=c.cu)
    for change in (dict(q=c.q.double()), dict(q=c.q[:, :3]), dict(q=c.q[..., :32]), dict(table=c.table.long()),
                   dict(table=c.table[0]), dict(cu=c.cu[:1]), dict(ctx_len=c.ctx_len.float()), dict(q=c.q.cpu()),
                   dict(max_new=0), dict(scale=float("nan")),
                   dict(q=torch.zeros(1 + c.q.numel(), device="cuda")[1:].view(c.q.shape))):
        with pytest.raises(ValueError):
            mx.kv_attention(**{**ok, **change})
    out, lse = mx.kv_attention(c.q[:0], c.cache(), c.table, c.ctx_len, torch.zeros(2, dtype=torch.int32, device="cuda"))
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
def test_prompts_behind_a_long_prefix(ctx, D, dtype):
    """V's exponents of a whole prefix are searched before a unit's first
    probabilities: the softmax's wait for them is a long one, and ends the sleeping way."""
    Case([(20000, 300), (15001, 33)], 8, 4, D, 64, dtype, seed=51).check(ctx)


def capture(stream, f):
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        out = f()
    return g, out


SHARED = {
    "joined": lambda i: Case([(9000 + 500 * i, 1), (40, 1)], 2, 2, 128, 64, torch.bfloat16, seed=60 + i),
    "prompts": lambda i: Case([(900, 700), (1300, 1000 + i)], 8, 2, 128, 64, torch.bfloat16, seed=64 + i)}


@pytest.mark.parametrize("kind", sorted(SHARED))
def test_graphs_of_one_stream_replayed_on_two(ctx, kind):
    """Graphs captured on one stream run at the same time on others, and beside
    calls on the stream that they were captured on."""
    cs = [SHARED[kind](i) for i in range(3)]
    want = [c.run(ctx) for c in cs]
    s = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    graphs = [capture(s[0], lambda c=c: c.run(ctx)) for c in cs[:2]]
    for _ in range(3):
        eager = []
        for i in range(2):
            graphs[i][1][0].zero_()
            graphs[i][1][1].zero_()
        torch.cuda.synchronize()
        for _ in range(15):
            for i in range(2):
                with torch.cuda.stream(s[1 + i]):
                    graphs[i][0].replay()
            with torch.cuda.stream(s[0]):
                eager.append(cs[2].run(ctx))
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(graphs[i][1][0], want[i][0]) and torch.equal(graphs[i][1][1], want[i][1])
        for o, l in eager:
            assert torch.equal(o, want[2][0]) and torch.equal(l, want[2][1])


def test_first_call_in_a_capture():
    """A capture on a stream that has not been used before, by a context that has no workspace yet."""
    c = Case([(3000, 1), (200, 1)], 2, 4, 128, 64, torch.float32, seed=67)
    want, _ = c.ref()
    fresh = mx.MXContext(0)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, _ = c.run(fresh)
    g.replay()
    torch.cuda.synchronize()
    assert float((out.double() - want).norm() / want.norm()) <= TOL[torch.float32]
    a = c.run(fresh)[0]
    assert torch.equal(a, out)
    del g
    torch.cuda.synchronize()
    fresh.close()


def test_workspaces_of_graphs_and_streams_that_are_gone_are_used_again(ctx):
    """Forty graphs, and forty streams, one after another, do not keep a workspace each (13 MB)."""
    c = Case([(3000, 1), (200, 1)], 2, 4, 128, 64, torch.bfloat16, seed=68)
    want = c.run(ctx)[0]
    s = torch.cuda.Stream()

    def once():
        g, (out, _) = capture(s, lambda: c.run(ctx))
        with torch.cuda.stream(s):
            g.replay()
        s.synchronize()
        assert torch.equal(out, want)
        del g, out
        torch.cuda.synchronize()
        torch.cuda.empty_cache()

    def own_stream():
        rt, h = torch.cuda.cudart(), ctypes.c_void_p()
        assert int(rt.cudaStreamCreate(ctypes.addressof(h))) == 0
        with torch.cuda.stream(torch.cuda.ExternalStream(h.value)):
            out = c.run(ctx)[0]
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        ctx._bind()                                  # a context's stream outlives its use there
        assert int(rt.cudaStreamDestroy(h.value)) == 0
        return h.value

    for f in (once, own_stream):
        f()
        f()
        before = torch.cuda.mem_get_info()[0]
        handles = {f() for _ in range(40)}
        used = (before - torch.cuda.mem_get_info()[0]) / 2 ** 20
        assert used <= 13 * (len(handles) + 4), (f.__name__, used, len(handles))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [1, 3, 300])
def test_lengths_near_the_end_of_int32(ctx, new, dtype):
    """A request that says it is 2^31 - 1 tokens long, with pages for 96 of them: each of its rows sees those."""
    c = Case([(96, 96)] * 2, 8, 4, 64, 32, dtype, seed=53, extra_rows=2 * new)
    q = c.q[:2 * new]
    cu = torch.tensor([0, new, 2 * new], dtype=torch.int32, device="cuda")
    for length in (2 ** 31 - 1, 2 ** 31 - 31, 2 ** 31 - 65):
        lens = torch.tensor([length, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
        out, lse = mx.kv_attention(q, c.cache(), c.table, lens, cu, max_new=new, ctx=ctx)
        ctx.synchronize()
        for r in range(2):
            for h in range(8):
                k, v, _ = c.dense(r, h, 96)
                rows = slice(r * new, r * new + new)
                s = torch.einsum("tgd,ld->tgl", q[rows, 4 * h:4 * h + 4].double(), k) / 8
                want, got = torch.softmax(s, -1) @ v, out[rows, 4 * h:4 * h + 4].double()
                assert float((got - want).norm() / want.norm()) <= TOL[dtype]
                assert float((lse[rows, 4 * h:4 * h + 4].double() - torch.logsumexp(s, -1)).abs().max()) <= 5e-4


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("G", [1, 4])
@pytest.mark.parametrize("R", [500, 4095, 4096, 4130, 8192])
def test_thousands_of_requests(ctx, R, G, dtype):
    """As many requests as kv_plan takes, short ones and a few long enough to be cut."""
    g = synth.rng(R)
    lens = g.integers(1, 70, R)
    far = g.integers(0, R, 5)
    lens[far] = g.integers(2000, 6000, 5)
    c = Case([(int(n), 1) for n in lens], 1, G, 128, 32, dtype, seed=54)
    out, lse = c.run(ctx)
    ctx.synchronize()
    # the first 96 keys of every request at once, then the long ones by themselves
    ids = c.table[:, :3].long().clamp(min=0)
    two = lambda x: torch.exp2(x.double() - 127)[..., None, None]
    k = (c.k[ids, 0, 0].double() * two(c.ks[ids, 0, 0])).reshape(R, 96, 128)
    v = (c.v[ids, 0, 0].flatten(2)[:, :, v_index(128).cuda()].double() * two(c.vs[ids, 0, 0])).reshape(R, 96, 128)
    s = torch.einsum("rgd,rld->rgl", c.q.double(), k) * 128 ** -0.5
    s.masked_fill_(torch.arange(96, device="cuda") >= c.ctx_len[:, None, None], -float("inf"))
    want, wl = torch.softmax(s, -1) @ v, torch.logsumexp(s, -1)
    for r in set(far.tolist()):
        k, v, _ = c.dense(r, 0, int(lens[r]))
        s = torch.einsum("gd,ld->gl", c.q[r].double(), k) * 128 ** -0.5
        want[r], wl[r] = torch.softmax(s, -1) @ v, torch.logsumexp(s, -1)
    err = (out.double() - want).norm(dim=2) / want.norm(dim=2)
    assert float(err.max()) <= 4 * TOL[dtype] and float((out.double() - want).norm() / want.norm()) <= TOL[dtype]
    tol = 2e-6 * wl.abs() + 2e-6 if dtype == torch.float32 else 5e-4
    assert ((lse.double() - wl).abs() <= tol).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
def test_prompt_rows_with_an_infinity_or_nan(ctx, value, dtype):
    """Such a row is NaN, whatever the sign of the keys it sees: the first rows see one or two."""
    c = Case([(512, 512), (300, 300)], 8, 4, 128, 64, dtype, seed=55)
    want, wl = c.ref()
    bad = torch.zeros(want.shape[:2], dtype=torch.bool)
    for row, head, d in ((0, 0, 7), (0, 5, 100), (1, 3, 0), (2, 31, 127), (512, 9, 64), (513, 14, 1), (400, 2, 3)):
        c.q[row, head, d] = value
        bad[row, head] = True
    out, lse = c.run(ctx)
    assert torch.isnan(out[bad]).all() and torch.isnan(lse[bad]).all()
    keep = ~bad
    assert float((out[keep].double() - want[keep]).norm() / want[keep].norm()) <= TOL[dtype]
    assert ((lse[keep].double() - wl[keep]).abs() <= 5e-4).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_v_blocks_that_are_nan(ctx, dtype):
    """Rows that see such a block are NaN, also those whose probabilities there are 0; their log-sum-exp knows nothing of V."""
    c = Case([(512, 512), (200, 200)], 8, 4, 128, 64, dtype, seed=56)
    pg = int(c.table[0, 3])                          # keys 192 .. 255
    c.k[pg, 2, 0] = 0                                # head 2: keys 192 .. 223 have scores far below the others'
    c.ks[:, 2] = 140
    c.k[int(c.table[0, 0]), 2, 0, 0] = 100
    c.q[:512, 8:12] = c.q[:512, 8:12].abs()
    want, wl = c.ref()                               # of the values without the NaN: what the other rows are
    c.vs[pg, 1, 1] = 255                             # head 1: keys 224 .. 255
    c.vs[pg, 2, 0] = 255
    assert float(torch.exp(wl[300:512, 8:12].neg()).max()) == 0.0
    out, lse = c.run(ctx)
    nan = torch.zeros(want.shape[:2], dtype=torch.bool)
    nan[224:512, 4:8] = True
    nan[192:512, 8:12] = True
    assert torch.isnan(out[nan]).all() and torch.isfinite(out[~nan]).all()
    assert float((out[~nan].double() - want[~nan]).norm() / want[~nan].norm()) <= TOL[dtype]
    assert ((lse.double() - wl).abs() <= 5e-4 + 2e-6 * wl.abs()).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
def test_prompts_keep_their_bits_where_v_scales_are_far_apart(ctx, D, dtype):
    """Exponents of V more than 2^32 apart: P in two terms of 8 bits (2^-17 of
    an element), beside which the usual bound holds."""
    c = Case([(600, 600), (300, 200), (1000, 77)], 8, 4, D, 64, dtype, seed=57)
    c.vs[:, 1, 1] -= 70                              # head 1: every other block tiny
    c.vs[int(c.table[1, 0]), 2, 0] = 1               # head 2 of request 1: one block tiny
    c.vs[int(c.table[2, 9]), 3, :] -= 40             # head 3 of request 2: a page small
    c.vs[int(c.table[2, 3]), 5, 1] = 255             # head 5 of request 2: a NaN block and a tiny one
    c.vs[int(c.table[2, 4]), 5, 1] = 1
    want, wl = c.ref()
    out, lse = c.run(ctx)
    assert ((lse.double() - wl).abs() <= 5e-4).all()
    for a, b, r in ((0, 600, 0), (600, 800, 1), (800, 877, 2)):
        for h in range(8):
            g, w = out[a:b, 4 * h:4 * h + 4].double(), want[a:b, 4 * h:4 * h + 4]
            if (r, h) == (2, 5):
                assert torch.isnan(g).all()
                continue
            assert float((g - w).norm() / w.norm()) <= TOL[dtype], (h, a)
            by_row = (g - w).flatten(0, 1).norm(dim=1) / w.flatten(0, 1).norm(dim=1)
            assert float(by_row.max()) <= 4 * TOL[dtype], (h, a)


def test_prompts_among_thousands_of_requests(ctx):
    g = synth.rng(58)
    spans = [(int(c), 1) for c in g.integers(1, 40, 8192)]
    for r, s in ((0, (300, 290)), (4096, (700, 257)), (8191, (500, 40))):
        spans[r] = s
    c = Case(spans, 8, 2, 64, 32, torch.float16, seed=58)
    out, lse = c.run(ctx)
    few = [0, 1, 2, 4095, 4096, 4097, 8190, 8191]
    rows = [i for r in few for i in range(int(c.cu[r]), int(c.cu[r + 1]))]
    d = Case.__new__(Case)
    d.__dict__.update(c.__dict__)
    d.ctx, d.new = [c.ctx[r] for r in few], [c.new[r] for r in few]
    d.table, d.q = c.table[few], c.q[rows]
    d.cu = torch.tensor([0] + list(np.cumsum(d.new)), dtype=torch.int32)
    want, wl = d.ref()
    assert float((out[rows].double() - want).norm() / want.norm()) <= TOL[torch.float16]
    assert ((lse[rows].double() - wl).abs() <= 5e-4).all() and torch.isfinite(out).all()
