"""The paged 8-bit K/V cache on the GPU: block tables and slot maps from
request lengths (kv_plan, kv_release) against a plain loop, new rows quantised
into their blocks (kv_append) bit for bit against numpy, and read back
(kv_read).  Whole numbers and 8-bit values are compared exactly."""
import numpy as np
import pytest
import torch

from cpu_model_b200 import mx, synth

pytestmark = pytest.mark.gpu


def cuda(a, dtype=None):
    return torch.as_tensor(np.ascontiguousarray(a), dtype=dtype, device="cuda")


# ------------------------------------------------------------------- plan ---
def plan_ref(past, add, P, table, stack, n_tokens):
    """The definition, page by page and row by row."""
    table, stack = table.copy(), list(stack)
    width = table.shape[1]
    short = 0
    ctx, cu, slots, pos, req = [], [0], [], [], []
    for r, (p, n) in enumerate(zip(past, add)):
        p, n = max(p, 0), max(n, 0)
        for j in range(-(-p // P), -(-(p + n) // P)):
            if j >= width:
                short += 1
            elif stack:
                table[r, j] = stack.pop()
            else:
                table[r, j] = -1
                short += 1
        ctx.append(p + n)
        cu.append(cu[-1] + n)
        for t in range(p, p + n):
            page = table[r, t // P] if t // P < width else -1
            slots.append(page * P + t % P if page >= 0 else -1)
            pos.append(t)
            req.append(r)
    fill = lambda v: np.array((v + [-1] * n_tokens)[:n_tokens], np.int32)
    return table, ctx, cu, fill(slots), fill(pos), fill(req), len(stack), short


def plan_case(R, past_hi, new_hi, P, seed, spare=5, narrow=0, negative=False):
    g = synth.rng(seed)
    past = g.integers(0, past_hi + 1, R)
    add = g.integers(0, new_hi + 1, R)
    if negative:
        past[::3] = -4
        add[1::4] = -7
    width = max(1, int(-(-(past + add).max() // P)) - narrow)
    have = [min(-(-max(int(p), 0) // P), width) for p in past]
    want = int(sum(max(0, min(-(-(max(int(p), 0) + max(int(n), 0)) // P), width) - h) for p, n, h in zip(past, add, have)))
    n_pages = max(1, sum(have) + want + max(spare, 0))
    ids = g.permutation(n_pages).astype(np.int32)
    table = np.full((R, width), -1, np.int32)
    at = 0
    for r, h in enumerate(have):
        table[r, :h] = ids[at:at + h]
        at += h
    stack = ids[at:] if spare >= 0 else ids[at:at + max(0, want + spare)]
    return past.astype(np.int32), add.astype(np.int32), table, stack, n_pages


@pytest.mark.parametrize("R,past_hi,new_hi,P,kw", [
    (1, 0, 1, 32, {}), (1, 700, 1, 64, {}), (7, 90, 40, 32, {}), (33, 2303, 1, 64, {}), (300, 500, 3, 128, {}),
    (257, 100, 97, 32, {}), (5000, 60, 9, 32, {}), (8192, 40, 1, 64, {}), (40, 300, 70, 32, {"negative": True}),
    (30, 200, 50, 32, {"spare": -6}), (30, 200, 50, 32, {"spare": -10 ** 6}), (25, 400, 90, 32, {"narrow": 5}),
    (12, 0, 0, 64, {}), (3, 5000, 4000, 1024, {})])
@pytest.mark.parametrize("in_place", [False, True])
def test_plan(ctx, R, past_hi, new_hi, P, kw, in_place):
    past, add, table, stack, n_pages = plan_case(R, past_hi, new_hi, P, R + past_hi, **kw)
    n = int(np.maximum(add, 0).sum()) + 3
    ref = plan_ref(past, add, P, table, stack, n)
    free = np.full(n_pages, -9, np.int32)
    free[:len(stack)] = stack
    d_past, d_table, d_count = cuda(past), cuda(table), cuda([len(stack)], torch.int32)
    p = mx.kv_plan(d_past, cuda(add), P, d_table, cuda(free), d_count, n, in_place=in_place, ctx=ctx)
    ctx.synchronize()
    for name, got, want in (("table", d_table, ref[0]), ("ctx", p.ctx_len, ref[1]), ("cu", p.cu, ref[2]),
                            ("slots", p.slots, ref[3]), ("positions", p.positions, ref[4]),
                            ("requests", p.requests, ref[5]), ("free", p.free_count, [ref[6]]), ("short", p.short, [ref[7]])):
        np.testing.assert_array_equal(got.cpu().numpy(), np.asarray(want, np.int32), err_msg=name)
    if in_place:
        assert p.ctx_len is d_past and p.free_count is d_count
    else:
        np.testing.assert_array_equal(d_past.cpu().numpy(), past)
        assert int(d_count) == len(stack)


def test_plan_fewer_map_rows_than_tokens(ctx):
    """Only n_tokens rows of the maps are written."""
    past, add = np.array([3, 70], np.int32), np.array([40, 5], np.int32)
    table = np.array([[4, -1], [7, 2]], np.int32)
    table = np.concatenate([table, np.full((2, 1), -1, np.int32)], 1)
    p = mx.kv_plan(cuda(past), cuda(add), 32, cuda(table), cuda([1, 3, 0, 5, 6, 8], torch.int32), cuda([3], torch.int32), 10,
                   ctx=ctx)
    ctx.synchronize()
    assert p.slots.tolist() == [4 * 32 + 3 + i for i in range(10)] and p.cu.tolist() == [0, 40, 45]


def test_release(ctx):
    g = synth.rng(5)
    P, R, width, n_pages = 64, 50, 9, 600
    lens = g.integers(0, width * P + 1, R).astype(np.int32)
    ids = g.permutation(n_pages).astype(np.int32)
    table = np.full((R, width), -1, np.int32)
    at = 0
    for r in range(R):
        h = -(-int(lens[r]) // P)
        table[r, :h] = ids[at:at + h]
        at += h
    table[3, 0] = -1                       # a page that was never there
    done = g.integers(0, 2, R).astype(np.uint8)
    free = np.full(n_pages, -1, np.int32)
    left = n_pages - at
    free[:left] = ids[at:]
    stack, t2, l2 = list(free[:left]), table.copy(), lens.copy()
    for r in range(R):
        if done[r]:
            for j in range(-(-int(lens[r]) // P)):
                if t2[r, j] >= 0:
                    stack.append(t2[r, j])
                t2[r, j] = -1
            l2[r] = 0
    dl, dt, df, dc = cuda(lens), cuda(table), cuda(free), cuda([left], torch.int32)
    mx.kv_release(cuda(done), dl, P, dt, df, dc, ctx=ctx)
    ctx.synchronize()
    np.testing.assert_array_equal(dt.cpu().numpy(), t2)
    np.testing.assert_array_equal(dl.cpu().numpy(), l2)
    assert int(dc) == len(stack) and df[:len(stack)].tolist() == stack


def test_plan_and_release_keep_every_page(ctx):
    """Steps of growth and release: no page is lost or owned twice."""
    g = synth.rng(9)
    P, R, width, n_pages = 32, 24, 12, 200
    lens, table = cuda(np.zeros(R, np.int32)), cuda(np.full((R, width), -1, np.int32))
    free, count = cuda(g.permutation(n_pages), torch.int32), cuda([n_pages], torch.int32)
    for step in range(12):
        add = g.integers(0, 60, R).astype(np.int32)
        add = np.minimum(add, width * P - lens.cpu().numpy()).astype(np.int32)
        p = mx.kv_plan(lens, cuda(add), P, table, free, count, int(add.sum()), in_place=True, ctx=ctx)
        assert int(p.short) == 0
        mx.kv_release(cuda((g.random(R) < 0.3).astype(np.uint8)), lens, P, table, free, count, ctx=ctx)
        owned = table[table >= 0].tolist() + free[:int(count)].tolist()
        assert sorted(owned) == list(range(n_pages))
        held = (table >= 0).sum(1).cpu().numpy()
        np.testing.assert_array_equal(held, -(-lens.cpu().numpy() // P))


# ----------------------------------------------------------------- append ---
def exponent_byte(top):
    """Smallest e >= -127 with top <= 127 * 2^e, as a byte."""
    if not np.isfinite(top):
        return 255
    if top == 0:
        return 0
    m, x = np.frexp(np.float64(top) / 127.0)
    return int(max(x - 1 if m == 0.5 else x, -127) + 127)


def v_place(t, d):
    return ((d >> 1) * 4 + (t >> 1) % 4) * 16 + (d & 1) * 8 + (t >> 3) * 2 + (t & 1)


def append_ref(q, sc, rows, slots, P, layout_v):
    """q int8 [pages][H][nb][32*D], sc uint8 [pages][H][nb], rows float64
    [n][H][D]: run by run, in place."""
    n, H, D = rows.shape
    total = q.shape[0] * P
    nb = P // 32
    place = np.array([[v_place(t, d) if layout_v else t * D + d for d in range(D)] for t in range(32)])
    i = 0
    while i < n:
        s = int(slots[i])
        if not 0 <= s < total:
            i += 1
            continue
        j = i
        while j < n and 0 <= slots[j] < total and slots[j] // 32 == s // 32:
            j += 1
        page, b = s // P, s % P // 32
        offs = [int(x) % 32 for x in slots[i:j]]
        for h in range(H):
            x = rows[i:j, h]
            byte = exponent_byte(np.abs(x).max() if np.isfinite(x).all() else np.inf)
            blk = q[page, h, b]
            if offs[0]:
                was = int(sc[page, h, b])
                byte = max(byte, was)
                if byte > was and byte != 255:
                    blk[:] = np.rint(blk.astype(np.float64) * 2.0 ** (was - byte)).astype(np.int8)
            if byte == 255:
                v = np.zeros_like(x)
            else:
                v = np.rint(x * 2.0 ** (127 - byte))
            for o, row in zip(offs, v):
                blk[place[o]] = row.astype(np.int8)
            sc[page, h, b] = byte
        i = j
    return q, sc


def make_cache(n_pages, P, H, D, seed):
    g = synth.rng(seed)
    nb = P // 32
    k = g.integers(-127, 128, (n_pages, H, nb, 32, D)).astype(np.int8)
    v = g.integers(-127, 128, (n_pages, H, nb, D // 2, 4, 2, 8)).astype(np.int8)
    ks = g.integers(118, 126, (n_pages, H, nb)).astype(np.uint8)
    vs = g.integers(118, 126, (n_pages, H, nb)).astype(np.uint8)
    return k, v, ks, vs


def check_append(ctx, P, H, D, dtype, slots, rows_k, rows_v, n_pages, seed, stride=0):
    k, v, ks, vs = make_cache(n_pages, P, H, D, seed)
    cache = mx.KVCache(cuda(k), cuda(v), cuda(ks), cuda(vs))
    n = len(slots)
    if stride:
        buf = torch.zeros((n, stride), dtype=dtype, device="cuda")
        dk = buf[:, 8:8 + H * D].unflatten(1, (H, D))
        dv = buf[:, stride - H * D:].unflatten(1, (H, D))
        dk.copy_(cuda(rows_k).to(dtype))
        dv.copy_(cuda(rows_v).to(dtype))
    else:
        dk, dv = cuda(rows_k).to(dtype), cuda(rows_v).to(dtype)
    mx.kv_append(cache, dk, dv, cuda(slots, torch.int32), ctx=ctx)
    ctx.synchronize()
    touched = {}
    for i, s in enumerate(slots):
        if 0 <= s < n_pages * P:
            touched.setdefault(int(s) // 32, []).append((i, int(s) % 32))
    for name, q, sc, src, lay in (("k", k, ks, dk, False), ("v", v, vs, dv, True)):
        before = q.reshape(n_pages, H, P // 32, 32 * D)
        q0, sc0 = before.copy(), sc.copy()
        ref, rsc = append_ref(before, sc, src.float().double().cpu().numpy(), slots, P, lay)
        got = getattr(cache, name).cpu().numpy().reshape(ref.shape)
        gsc = getattr(cache, name + "_scale").cpu().numpy()
        np.testing.assert_array_equal(gsc, rsc, err_msg=name + " scales")
        place = np.array([[v_place(t, d) if lay else t * D + d for d in range(D)] for t in range(32)])
        for blk in range(n_pages * P // 32):
            pg, b = blk // (P // 32), blk % (P // 32)
            if blk not in touched:
                np.testing.assert_array_equal(got[pg, :, b], q0[pg, :, b], err_msg="%s block %d was not to be touched" % (name, blk))
                continue
            first = touched[blk][0][1]
            # a block that the run started is defined where rows went; one that it extended, everywhere
            offs = [o for _, o in touched[blk]] if first == 0 else list(range(32))
            for h in range(H):
                sel = place[offs].reshape(-1)
                np.testing.assert_array_equal(got[pg, h, b][sel], ref[pg, h, b][sel], err_msg="%s block %d head %d" % (name, blk, h))
    return cache


def request_slots(g, P, n_pages, spans):
    """Slots of (past, new) spans over shuffled pages."""
    ids = list(g.permutation(n_pages))
    out = []
    for p, n in spans:
        pages = [ids.pop() for _ in range(-(-(p + n) // P))]
        out += [pages[t // P] * P + t % P for t in range(p, p + n)]
    return np.array(out, np.int32), None


SPANS = {
    "one": [(0, 1)], "one_inside": [(37, 1)], "block": [(0, 32)], "prompt": [(0, 100)], "continue": [(29, 70), (64, 40)],
    "steps": [(i * 7 % 95, 1) for i in range(21)], "few": [(30, 5), (3, 9), (0, 7), (31, 2), (16, 8)],
    "mixed": [(0, 33), (5, 1), (40, 64), (31, 1), (0, 2), (63, 3)]}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("P,H,D", [(32, 1, 64), (64, 3, 128), (128, 2, 64), (1024, 1, 128)])
@pytest.mark.parametrize("span", sorted(SPANS))
def test_append(ctx, P, H, D, dtype, span):
    g = synth.rng(P + H + D)
    spans = SPANS[span]
    n_pages = sum(-(-(p + n) // P) for p, n in spans) + 2
    slots, _ = request_slots(g, P, n_pages, spans)
    n = len(slots)
    mag = np.exp(g.normal(0, 2, (n, H, 1)))
    check_append(ctx, P, H, D, dtype, slots, g.normal(0, 1, (n, H, D)) * mag * 0.05, g.normal(0, 1, (n, H, D)) * mag, n_pages,
                 7, stride=2 * H * D + 24)


def test_append_many_rows(ctx):
    """Enough rows that a CTA takes 32 of them, runs that end everywhere in it."""
    g = synth.rng(3)
    P, H, D = 64, 2, 128
    spans = [(int(g.integers(0, 90)), int(g.integers(1, 300))) for _ in range(40)] + [(int(g.integers(0, 90)), 1) for _ in range(200)]
    n_pages = sum(-(-(p + n) // P) for p, n in spans) + 1
    slots, _ = request_slots(g, P, n_pages, spans)
    n = len(slots)
    assert n * H > 8 * 148 * 8
    check_append(ctx, P, H, D, torch.bfloat16, slots, g.normal(0, 1, (n, H, D)), g.normal(0, 1, (n, H, D)), n_pages, 5)


def test_append_values_at_the_edges(ctx):
    """Zeros, denormals, the largest finite values, exponent boundaries, NaN
    and infinities, skipped slots, slots outside the pool."""
    P, H, D, n_pages = 32, 1, 64, 14
    rows = np.zeros((12, H, D))
    rows[1, 0, 3] = 2.0 ** -140
    rows[2, 0, :] = 3.3e38
    rows[3, 0, 5] = 127.0 * 2.0 ** 3
    rows[4, 0, 5] = np.float32(np.nextafter(np.float32(127.0 * 2.0 ** 3), np.float32(2e3)))
    rows[5, 0, 0] = np.nan
    rows[6, 0, 63] = np.inf
    rows[7, 0, 1] = -np.inf
    rows[8, 0, :] = np.linspace(-1, 1, D)
    rows[9, 0, :] = 0.5
    rows[10, 0, :] = 1.0
    rows[11, 0, :] = 1.0
    slots = np.array([p * 32 for p in range(9)] + [9 * 32 + 4, -1, n_pages * 32], np.int32)
    check_append(ctx, P, H, D, torch.float32, slots, rows, rows[:, :, ::-1].copy(), n_pages, 11)
    # rounding halfway goes to the even integer, before and after a re-rounding
    halves = np.zeros((2, H, D))
    halves[0, 0, :8] = [127, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 3]
    halves[1, 0, 0] = 254.0
    cache = check_append(ctx, P, H, D, torch.float32, np.array([0], np.int32), halves[:1], halves[:1], 2, 12)
    mx.kv_append(cache, cuda(halves[1:], torch.float32), cuda(halves[1:], torch.float32), cuda([1], torch.int32), ctx=ctx)
    k, v = mx.kv_read(cache, cuda([0, 1], torch.int32), ctx=ctx)
    # 127 0 2 2 0 -2 -2 3 at step 1, halved: 63.5 -> 64 and 1.5 -> 2
    assert k[0, 0, :8].tolist() == v[0, 0, :8].tolist() == [128, 0, 2, 2, 0, -2, -2, 4]
    assert k[1, 0, 0] == 254


def test_append_nan_stays_in_its_block(ctx):
    """A NaN marks its block and head only, for as long as the block is
    extended; starting the block again clears it."""
    P, H, D = 64, 2, 64
    cache = mx.KVCache.empty(2, P, H, D)
    rows = torch.ones((3, H, D), device="cuda")
    rows[1, 0, 7] = float("nan")
    slots = cuda([0, 1, 32], torch.int32)
    mx.kv_append(cache, rows, torch.ones_like(rows), slots, ctx=ctx)
    one = torch.ones((1, H, D), device="cuda")
    mx.kv_append(cache, one, one, cuda([2], torch.int32), ctx=ctx)
    k, v = mx.kv_read(cache, cuda([0, 1, 2, 32], torch.int32), ctx=ctx)
    assert torch.isnan(k[:3, 0]).all() and (k[:3, 1] == 1).all() and (k[3] == 1).all() and (v == 1).all()
    mx.kv_append(cache, one, one, cuda([0], torch.int32), ctx=ctx)
    assert (mx.kv_read(cache, cuda([0], torch.int32), ctx=ctx)[0] == 1).all()


@pytest.mark.parametrize("P,H,D", [(32, 2, 64), (128, 3, 128)])
def test_read_values(ctx, P, H, D):
    n_pages = 5
    k, v, ks, vs = make_cache(n_pages, P, H, D, 21)
    ks[1, 0, 0], vs[2, 1, 0] = 0, 255
    cache = mx.KVCache(cuda(k), cuda(v), cuda(ks), cuda(vs))
    g = synth.rng(2)
    for slots in (g.permutation(n_pages * P)[:77], np.arange(40, 40 + 64), [-1, 0, n_pages * P, 5], [n_pages * P - 1]):
        slots = np.asarray(slots, np.int32)
        want_k = np.zeros((len(slots), H, D))
        want_v = np.zeros((len(slots), H, D))
        for i, s in enumerate(slots):
            if 0 <= s < n_pages * P:
                pg, b, t = s // P, s % P // 32, s % 32
                f = np.where(ks[pg, :, b] == 255, np.nan, np.exp2(ks[pg, :, b].astype(np.float64) - 127))
                want_k[i] = k[pg, :, b, t].astype(np.float64) * f[:, None]
                f = np.where(vs[pg, :, b] == 255, np.nan, np.exp2(vs[pg, :, b].astype(np.float64) - 127))
                flat = v[pg, :, b].reshape(H, -1)
                want_v[i] = flat[:, [v_place(t, d) for d in range(D)]].astype(np.float64) * f[:, None]
        for dt in (torch.float32, torch.bfloat16):
            gk, gv = mx.kv_read(cache, cuda(slots), dt, ctx=ctx)
            np.testing.assert_array_equal(gk.double().cpu().numpy(), want_k)
            np.testing.assert_array_equal(gv.double().cpu().numpy(), want_v)


def test_offsets_beyond_32_bits(ctx):
    """Blocks whose bytes lie past 2^31 in the pool."""
    P, H, D, n_pages = 64, 8, 128, 40000
    nb = P // 32
    assert n_pages * H * P * D > 2 ** 31
    cache = mx.KVCache(torch.empty((n_pages, H, nb, 32, D), dtype=torch.int8, device="cuda"),
                       torch.empty((n_pages, H, nb, D // 2, 4, 2, 8), dtype=torch.int8, device="cuda"),
                       torch.zeros((n_pages, H, nb), dtype=torch.uint8, device="cuda"),
                       torch.zeros((n_pages, H, nb), dtype=torch.uint8, device="cuda"))
    x = torch.randn((96, H, D), device="cuda")
    y = torch.randn((96, H, D), device="cuda")
    slots = torch.cat([torch.arange(48) + (n_pages - 1) * P, torch.arange(48) + 20000 * P]).to("cuda", torch.int32)
    mx.kv_append(cache, x, y, slots, ctx=ctx)
    k, v = mx.kv_read(cache, slots, ctx=ctx)
    for got, want in ((k, x), (v, y)):      # half a step of a block whose maximum is below 8: 8/127 < 2^-3
        assert (got - want).abs().max() <= 2.0 ** -5
    del cache
    torch.cuda.empty_cache()


def test_refusals(ctx):
    P, H, D = 64, 2, 64
    cache = mx.KVCache.empty(3, P, H, D)
    x = torch.zeros((4, H, D), device="cuda")
    s = torch.zeros(4, dtype=torch.int32, device="cuda")
    i32 = lambda n: torch.zeros(n, dtype=torch.int32, device="cuda")
    bad = [
        lambda: mx.kv_append(cache, x.double(), x.double(), s),
        lambda: mx.kv_append(cache, x, x.bfloat16(), s),
        lambda: mx.kv_append(cache, x[:, :1], x[:, :1], s),
        lambda: mx.kv_append(cache, x, x, s[:3]),
        lambda: mx.kv_append(cache, x, x, s.long()),
        lambda: mx.kv_append(cache, x.cpu(), x.cpu(), s),
        lambda: mx.kv_append(cache, x.transpose(1, 2).contiguous().transpose(1, 2), x, s),
        lambda: mx.kv_append(cache, torch.zeros(4 * H * D + 1, device="cuda")[1:].view(4, H, D), x, s),
        lambda: mx.kv_read(cache, s, torch.float64),
        lambda: mx.kv_read(cache, s.float()),
        lambda: mx.KVCache.empty(3, 48, H, D),
        lambda: mx.KVCache(cache.k, cache.k, cache.k_scale, cache.v_scale),
        lambda: mx.KVCache(cache.k, cache.v, cache.k_scale[:2], cache.v_scale),
        lambda: mx.kv_append(mx.KVCache.empty(3, P, H, 96), x, x, s),
        lambda: mx.kv_append(mx.KVCache.empty(3, P, H, 96), torch.zeros((4, H, 96), device="cuda"),
                             torch.zeros((4, H, 96), device="cuda"), s),
        lambda: mx.kv_append(mx.KVCache.empty(1, 2048, H, D), x, x, s),
        lambda: mx.kv_plan(i32(3), i32(2), P, i32((3, 4)), i32(9), i32(1), 4),
        lambda: mx.kv_plan(i32(3), i32(3), 33, i32((3, 4)), i32(9), i32(1), 4),
        lambda: mx.kv_plan(i32(3), i32(3), P, i32((2, 4)), i32(9), i32(1), 4),
        lambda: mx.kv_plan(i32(3), i32(3), P, i32((3, 4)), i32(9), i32(1), -1),
        lambda: mx.kv_plan(i32(3).long(), i32(3), P, i32((3, 4)), i32(9), i32(1), 4),
        lambda: mx.kv_plan(i32(8193), i32(8193), P, i32((8193, 1)), i32(9), i32(1), 4),
        lambda: mx.kv_release(i32(3), i32(3), P, i32((3, 4)), i32(9), i32(1)),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail("case %d was not refused" % i)
    mx.kv_append(cache, x[:0], x[:0], s[:0])         # nothing to do is not an error
    assert mx.kv_read(cache, s[:0])[0].shape == (0, H, D)


def test_two_streams_share_no_workspace(ctx):
    """Plans of many CTAs (they count themselves in a workspace) queued on two streams at once."""
    past, add, table, stack, n_pages = plan_case(5000, 200, 20, 32, 77)
    n = int(add.sum())
    ref = plan_ref(past, add, 32, table, stack, n)
    free = cuda(np.concatenate([stack, np.full(n_pages - len(stack), -1)]), torch.int32)
    args = [cuda(past), cuda(add), cuda([len(stack)], torch.int32)]
    tables = [cuda(table) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    out = []
    for i in range(20):
        with torch.cuda.stream(streams[i % 2]):
            out.append(mx.kv_plan(args[0], args[1], 32, tables[i % 2], free, args[2], n, ctx=ctx))
    torch.cuda.synchronize()
    for p in out:
        np.testing.assert_array_equal(p.slots.cpu().numpy(), ref[3])
        assert int(p.free_count) == ref[6] and p.ctx_len.tolist() == ref[1]


def test_plans_captured_on_one_stream_run_on_two(ctx):
    """Plans of many CTAs, captured on one stream, replayed on two at once."""
    cases = [plan_case(5000, 200, 20, 32, 77 + i) for i in range(2)]
    s = [torch.cuda.Stream() for _ in range(3)]
    graphs = []
    for past, add, table, stack, n_pages in cases:
        n = int(add.sum())
        free = cuda(np.concatenate([stack, np.full(n_pages - len(stack), -1)]), torch.int32)
        args = [cuda(past), cuda(add), 32, cuda(table), free, cuda([len(stack)], torch.int32), n]
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s[0]):
            p = mx.kv_plan(*args, ctx=ctx)
        graphs.append((g, p, args, plan_ref(past, add, 32, table, stack, n)))
    torch.cuda.synchronize()
    for _ in range(30):
        for i, (g, p, args, ref) in enumerate(graphs):
            with torch.cuda.stream(s[1 + i]):
                p.slots.zero_()
                p.ctx_len.zero_()
                g.replay()
    torch.cuda.synchronize()
    for g, p, args, ref in graphs:
        np.testing.assert_array_equal(p.slots.cpu().numpy(), ref[3])
        np.testing.assert_array_equal(args[3].cpu().numpy(), ref[0])
        assert int(p.free_count) == ref[6] and p.ctx_len.tolist() == ref[1]


@pytest.mark.parametrize("P", [32, 1024])
def test_lengths_near_the_end_of_int32(ctx, P):
    """Lengths whose next page's end is no int32: pages and slots as page by page, and their pages come back."""
    top = 2 ** 31 - 1
    past, add = np.array([5, top - 40, 0, top, 33], np.int32), np.array([3, 40, 40, 0, 7], np.int32)
    table = np.full((5, 3), -1, np.int32)
    held = iter(range(20))
    for r in range(5):
        for j in range(min(3, -(-int(past[r]) // P))):
            table[r, j] = next(held)
    stack = np.arange(20, 27, dtype=np.int32)
    free = np.concatenate([stack, np.full(23, -1, np.int32)])
    n = 92
    ref = plan_ref([int(x) for x in past], [int(x) for x in add], P, table, stack, n)
    d = [cuda(past), cuda(table), cuda(free), cuda([7], torch.int32)]
    p = mx.kv_plan(d[0], cuda(add), P, d[1], d[2], d[3], n, in_place=True, ctx=ctx)
    ctx.synchronize()
    for got, want in ((d[1], ref[0]), (p.ctx_len, ref[1]), (p.cu, ref[2]), (p.slots, ref[3]), (p.positions, ref[4]), (p.requests, ref[5]),
                      (p.free_count, [ref[6]]), (p.short, [ref[7]])):
        np.testing.assert_array_equal(got.cpu().numpy(), np.asarray(want, np.int32))
    mx.kv_release(cuda(np.ones(5, np.uint8)), d[0], P, d[1], d[2], d[3], ctx=ctx)
    assert (d[1] == -1).all() and (d[0] == 0).all()
    owned = int((ref[0] >= 0).sum())
    assert int(d[3]) == ref[6] + owned
    assert d[2][ref[6]:ref[6] + owned].tolist() == [int(x) for x in ref[0].flatten() if x >= 0]


@pytest.mark.parametrize("n,h,nb,d", [(2, 0, 1, 64), (0, 2, 1, 64), (2, 2, 0, 64), (2, 2, 1, 0)])
def test_caches_of_nothing_are_refused(n, h, nb, d):
    i8 = lambda *s: torch.zeros(s, dtype=torch.int8, device="cuda")
    u8 = lambda: torch.zeros((n, h, nb), dtype=torch.uint8, device="cuda")
    with pytest.raises(ValueError):
        mx.KVCache(i8(n, h, nb, 32, d), i8(n, h, nb, d // 2, 4, 2, 8), u8(), u8())


def test_versions_of_what_is_written(ctx):
    """Every tensor that a call writes into says so to autograd."""
    P, H, D = 32, 1, 64
    cache = mx.KVCache.empty(4, P, H, D)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    lens, table, free, count = i32(0, 0), i32([-1, -1], [-1, -1]), i32(0, 1, 2, 3), i32(4)

    def raised(tensors, f):
        before = [t._version for t in tensors]
        r = f()
        assert all(t._version > b for t, b in zip(tensors, before))
        return r
    p = raised([table], lambda: mx.kv_plan(lens, i32(3, 1), P, table, free, count, 4, ctx=ctx))
    raised([table, lens, count], lambda: mx.kv_plan(lens, i32(3, 1), P, table, free, count, 4, in_place=True, ctx=ctx))
    x = torch.randn((4, H, D), device="cuda")
    raised([cache.k, cache.v, cache.k_scale, cache.v_scale], lambda: mx.kv_append(cache, x, x, p.slots, ctx=ctx))
    raised([lens, table, free, count], lambda: mx.kv_release(i32(1, 1).bool(), lens, P, table, free, count, ctx=ctx))
    with torch.inference_mode():
        y = torch.zeros((2, 5), device="cuda")
        r = mx.token_logprobs(y, i32(0, 1), ctx=ctx)
        mx.token_logprobs_grad(y, i32(0, 1), r.lse, r.entropy, torch.ones(2, device="cuda"), out=y, ctx=ctx)


@pytest.mark.parametrize("n", [1, 12])
def test_append_to_a_block_with_the_largest_scale(ctx, n):
    """A block whose scale is 2^127 already: new rows are rounded to that step, not lost."""
    P, H, D = 32, 1, 64
    cache = mx.KVCache.empty(1, P, H, D)
    cache.k_scale.fill_(254)
    cache.v_scale.fill_(254)
    x = torch.zeros((n, H, D), device="cuda")
    x[:, 0, 0], x[:, 0, 1], x[:, 0, 2], x[:, 0, 3] = 3e38, -2e38, 1e38, 8e37
    mx.kv_append(cache, x, x, cuda(np.arange(1, n + 1), torch.int32), ctx=ctx)
    want = torch.round(x.double() * 2.0 ** -127)
    assert want[0, 0, :4].tolist() == [2, -1, 1, 0]
    assert torch.equal(cache.k[0, 0, 0, 1:n + 1].double(), want[:, 0])
    for i in range(n):
        for d in range(4):
            assert int(cache.v.flatten()[v_place(i + 1, d)]) == int(want[i, 0, d])


def test_a_cache_follows_its_tensors(ctx):
    """The cache's tensors are the caller's: other memory given to one is what the next call uses, another shape is refused."""
    P, H, D = 32, 2, 64
    cache = mx.KVCache.empty(2, P, H, D)
    x = torch.randn((3, H, D), device="cuda")
    slots = cuda([0, 1, 2], torch.int32)
    mx.kv_append(cache, x, x, slots, ctx=ctx)
    want = mx.kv_read(cache, slots, ctx=ctx)
    old = cache.k.clone(), cache.k_scale.clone()
    cache.k.set_(torch.zeros_like(cache.k))
    cache.k_scale.set_(torch.zeros_like(cache.k_scale))
    assert (mx.kv_read(cache, slots, ctx=ctx)[0] == 0).all()
    mx.kv_append(cache, x, x, slots, ctx=ctx)
    assert all(torch.equal(a, b) for a, b in zip(mx.kv_read(cache, slots, ctx=ctx), want))
    assert torch.equal(cache.k, old[0]) and torch.equal(cache.k_scale, old[1])
    cache.v_scale.set_(torch.zeros(1, dtype=torch.uint8, device="cuda"))
    for f in (lambda: mx.kv_append(cache, x, x, slots), lambda: mx.kv_read(cache, slots),
              lambda: mx.kv_attention(x, cache, slots[None, :1].contiguous(), slots[:1], slots[:2])):
        with pytest.raises(ValueError):
            f()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 3, 40])
def test_append_k_of_its_own_and_v_as_a_slice(ctx, n, dtype):
    """What a rotary embedding leaves: K rows of their own beside V rows inside the fused ones, and the other way round."""
    P, H, D = 32, 2, 64
    fused = torch.randn((n, 6 * H * D), device="cuda").to(dtype)
    v = fused[:, 5 * H * D:].unflatten(1, (H, D))
    k = torch.randn((n, H, D), device="cuda").to(dtype)
    slots = torch.arange(5, 5 + n, dtype=torch.int32, device="cuda")
    for a, b in ((k, v), (v, k)):
        caches = [mx.KVCache.empty(2, P, H, D) for _ in range(2)]
        mx.kv_append(caches[0], a, b, slots, ctx=ctx)
        mx.kv_append(caches[1], a.contiguous(), b.contiguous(), slots, ctx=ctx)
        for name in ("k", "v", "k_scale", "v_scale"):
            assert torch.equal(getattr(caches[0], name), getattr(caches[1], name))
    odd = torch.zeros((n, 6 * H * D + 1), device="cuda").to(dtype)[:, :H * D].unflatten(1, (H, D))
    if n > 1:
        for a, b in ((k, odd), (odd, k), (k, k[:1].expand(n, H, D))):
            with pytest.raises(ValueError):
                mx.kv_append(caches[0], a, b, slots, ctx=ctx)
