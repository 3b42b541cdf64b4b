"""Token log probabilities, entropy, top alternatives and their gradient
against the formulas in 64 bits.

Tolerances: sums of exp in fp32 over partial sums of a few dozen terms, ex2 to 2^-22:
1e-6 relative in s, so 2e-6 absolute in lse, logp and entropy for results of
order 1, plus fp32's 2^-24 of the logits' size (|x - M| below 64: 4e-6); an
entropy's terms add p |log p| errors of the same size: 1e-5 absolute bounds all three.
Gradients: 3e-6 relative 2-norm in fp32 (p carries exp's error at |log p| <= 20);
16-bit gradients are the fp32 ones rounded once, bit for bit."""
import numpy as np
import pytest
import torch

from cpu_model_b200 import mx, synth

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
ABS = 1e-5


def rows_of(n, v, dtype, seed, pad=0, peak=True, banned=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    buf = (torch.randn((n, v + pad), device="cuda", generator=gen) * 2).to(dtype)
    x = buf[:, :v]
    t = torch.randint(0, v, (n,), device="cuda", generator=gen).to(torch.int32)
    if peak:
        r = torch.arange(0, n, 2, device="cuda")
        x[r, t[r].long()] += 8
    if banned:
        x[:, :min(banned, v - 1)] = -float("inf")
    return x, t


def ref(x, t):
    x = x.double()
    m = x.amax(1, keepdim=True)                       # log p apart from lse: a row of the type's lowest value keeps log 1/V
    logs = torch.log(torch.exp(x - m).sum(1, keepdim=True))
    lse = (m + logs)[:, 0]
    lp = (x - m) - logs
    p = lp.exp()
    ent = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(1)
    tt = t.long().clamp(0, x.shape[1] - 1)
    logp = lp.gather(1, tt[:, None])[:, 0]
    inside = (t >= 0) & (t < x.shape[1])
    return torch.where(inside, logp, torch.zeros_like(logp)), ent, lse, lp, p


def close(a, b, tol=ABS):
    a, b = a.double(), b.double()
    same = (a == b) | (torch.isnan(a) & torch.isnan(b))
    ok = same | ((a - b).abs() <= tol)
    assert ok.all(), float((a - b)[~ok].abs().max())


def top_ref(x, k):
    """Stable descending order: ties to the lower id, NaN first."""
    y = x.float() + 0.0
    v, i = torch.sort(torch.where(torch.isnan(y), torch.full_like(y, float("inf")), y), dim=1, descending=True, stable=True)
    if torch.isnan(y).any():
        key = torch.where(torch.isnan(y), 2, torch.where(y == float("inf"), 1, 0))
        order = []
        for r in range(y.shape[0]):
            vals = y[r].cpu().numpy()
            nan = np.isnan(vals)
            order.append(np.lexsort((np.arange(len(vals)), -np.where(nan, 0, vals), ~nan)))
        i = torch.as_tensor(np.stack(order), device=y.device)
    return i[:, :k]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,v,k,pad", [
    (1, 1, 1, 0), (3, 2, 2, 0), (5, 3, 1, 1), (4, 80, 20, 1), (9, 127, 32, 3), (7, 1000, 5, 0), (6, 2047, 7, 5),
    (5, 4096, 32, 0), (3, 8193, 20, 1), (1, 32000, 20, 0), (2, 32001, 1, 0), (200, 32000, 5, 1), (33, 50257, 3, 0),
    (1, 131072, 32, 0), (150, 5003, 0, 2)])
def test_forward(ctx, n, v, k, pad, dtype):
    x, t = rows_of(n, v, dtype, n + v, pad, banned=3 if v > 50 else 0)
    t[n // 2] = max(3, v - 1) if v > 50 else 0
    r = mx.token_logprobs(x, t, k, ctx=ctx)
    ctx.synchronize()
    logp, ent, lse, lp, _ = ref(x, t)
    close(r.logp, logp)
    close(r.entropy, ent)
    close(r.lse, lse)
    if k == 0:
        assert r.top_ids is None
        return
    ids = top_ref(x, k)
    assert torch.equal(r.top_ids.long(), ids)
    close(r.top_logp, lp.gather(1, ids))


@pytest.mark.parametrize("v", [50, 700, 5000, 40000])
def test_ties_go_to_the_lower_id(ctx, v):
    """Equal logits everywhere, a few values, and -0 beside 0."""
    for x in (torch.zeros((4, v), device="cuda"), torch.randint(0, 3, (4, v), device="cuda").float(),
              torch.where(torch.rand((4, v), device="cuda") < 0.5, -0.0, 0.0)):
        t = torch.zeros(4, dtype=torch.int32, device="cuda")
        r = mx.token_logprobs(x, t, 32, ctx=ctx)
        assert torch.equal(r.top_ids.long(), top_ref(x, 32))
        _, ent, lse, lp, _ = ref(x, t)
        close(r.lse, lse)
        close(r.entropy, ent)
        close(r.top_logp, lp.gather(1, r.top_ids.long()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [75, 2051, 32001])
def test_alternatives_at_a_row_s_ends(ctx, v, dtype):
    """The largest logits are the first and the last ones, in rows that start
    on every alignment."""
    x, t = rows_of(17, v, dtype, v, pad=2, peak=False)
    x[:, :9] += 30
    x[:, -9:] += 30
    r = mx.token_logprobs(x, t, 18, ctx=ctx)
    assert torch.equal(r.top_ids.long(), top_ref(x, 18))
    close(r.top_logp, ref(x, t)[3].gather(1, r.top_ids.long()))


@pytest.mark.parametrize("v", [40, 3000, 40000])
def test_empty_infinite_and_nan_rows(ctx, v):
    inf = float("inf")
    x, t = rows_of(7, v, torch.float32, v)
    x[0] = -inf                                       # nothing left
    x[1] = -inf
    x[1, 17] = 3.0                                    # one token left
    t[1] = 17
    x[2, 5] = inf
    x[3, 9] = float("nan")
    x[4, 11] = -float("nan")
    x[5] = torch.finfo(torch.float32).min             # the type's lowest value, everywhere
    x[6, :20] = torch.finfo(torch.float32).min        # and as a mask
    t[6] = 25
    r = mx.token_logprobs(x, t, 4, ctx=ctx)
    assert r.lse[0] == -inf and r.logp[0] == -inf and r.entropy[0] == 0 and (r.top_logp[0] == -inf).all()
    assert r.top_ids[0].tolist() == [0, 1, 2, 3]
    assert r.lse[1] == 3.0 and r.logp[1] == 0 and r.entropy[1] == 0 and r.top_ids[1].tolist() == [17, 0, 1, 2]
    assert torch.isnan(r.logp[2:5]).all() and torch.isnan(r.entropy[2:5]).all() and torch.isnan(r.lse[3:5]).all()
    for row in (2, 3, 4):
        assert r.top_ids[row].tolist() == top_ref(x[row:row + 1], 4)[0].tolist()
    assert r.top_ids[5].tolist() == [0, 1, 2, 3]
    close(r.logp[5:], ref(x[5:], t[5:])[0])
    close(r.entropy[5:], ref(x[5:], t[5:])[1], 2e-5)
    g = mx.token_logprobs_grad(x, t, r.lse, r.entropy, torch.ones(7, device="cuda"), torch.ones(7, device="cuda"), ctx=ctx)
    assert (g[0] == 0).all() and (g[1] == 0).all() and torch.isnan(g[2:5]).any(1).all()
    assert torch.isfinite(g[5:]).all() and (g[5] == 0).all() and (g[6, :20] == 0).all()


def test_targets_outside_the_vocabulary(ctx):
    x, t = rows_of(5, 100, torch.float32, 1)
    t[0], t[1], t[2] = -1, 100, 2 ** 30
    r = mx.token_logprobs(x, t, ctx=ctx)
    assert (r.logp[:3] == 0).all()
    close(r.logp, ref(x, t)[0])
    g = mx.token_logprobs_grad(x, t, r.lse, r.entropy, torch.ones(5, device="cuda"), ctx=ctx)
    assert (g[:3] == 0).all() and (g[3:] != 0).any()


def test_outputs_are_optional_through_the_c_entry(ctx):
    import ctypes
    x, t = rows_of(3, 500, torch.float32, 2)
    p = lambda a: ctypes.c_void_p(a.data_ptr() if a is not None else 0)
    lse = torch.empty(3, device="cuda")
    ctx._bind()
    assert ctx.lib.mxq_token_logprobs(ctx.h, 0, p(x), 500, 3, 500, p(t), 0, None, None, p(lse), None, None) == 0
    close(lse, ref(x, t)[2])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,v,pad,gpad", [(1, 1, 0, 0), (4, 3, 1, 0), (5, 80, 0, 1), (3, 1001, 2, 0), (6, 8192, 0, 0),
                                          (2, 32000, 1, 0), (3, 50257, 0, 0)])
def test_gradient_against_the_formula(ctx, n, v, pad, gpad, dtype):
    x, t = rows_of(n, v, dtype, n + v, pad, banned=2 if v > 50 else 0)
    r = mx.token_logprobs(x, t, ctx=ctx)
    gen = torch.Generator(device="cuda").manual_seed(5)
    dl, de = torch.randn(n, device="cuda", generator=gen), torch.randn(n, device="cuda", generator=gen)
    logp, ent, lse, lp, p = ref(x, t)
    hit = torch.zeros_like(p)
    hit.scatter_(1, t.long()[:, None], 1.0)
    lpf = torch.where(p > 0, lp, torch.zeros_like(lp))
    for a, b in ((dl, de), (dl, None), (None, de)):
        want = 0
        if a is not None:
            want = want + a.double()[:, None] * (hit - p)
        if b is not None:
            want = want - b.double()[:, None] * p * (lpf + ent[:, None])
        out = torch.full((n, v + gpad), 7.0, dtype=dtype, device="cuda")
        g = mx.token_logprobs_grad(x, t, r.lse, r.entropy, a, b, out=out[:, :v], ctx=ctx)
        assert (out[:, v:] == 7).all()
        f = mx.token_logprobs_grad(x.float(), t, r.lse, r.entropy, a, b, ctx=ctx)
        err = float((f.double() - want).norm())
        assert err <= 3e-6 * float(want.norm()) + 1e-7 * (n * v) ** 0.5, (err, float(want.norm()))
        assert torch.equal(g, f.to(dtype))
    again = x.clone()
    mx.token_logprobs_grad(again, t, r.lse, r.entropy, dl, de, out=again, ctx=ctx)          # in place
    fresh = mx.token_logprobs_grad(x, t, r.lse, r.entropy, dl, de, ctx=ctx)
    assert torch.equal(again, fresh)


def test_gradient_against_differences(ctx):
    """Central differences of the forward pass, h = 2^-6: their error is h^2/6
    of a third derivative below 1 (4e-5) plus 2 * 1e-5 / 2h of rounding (6.4e-4)."""
    n, v, h = 3, 40, 2.0 ** -6
    x, t = rows_of(n, v, torch.float32, 3, peak=False)
    x.requires_grad_(True)
    logp, ent = mx.token_logp(x, t)
    w, u = torch.tensor([1.0, -0.5, 2.0], device="cuda"), torch.tensor([0.3, 1.0, -1.0], device="cuda")
    ((logp * w).sum() + (ent * u).sum()).backward()
    base = x.detach()
    for j in range(v):
        up, down = base.clone(), base.clone()
        up[:, j] += h
        down[:, j] -= h
        a, b = mx.token_logprobs(up, t, ctx=ctx), mx.token_logprobs(down, t, ctx=ctx)
        diff = (w * (a.logp - b.logp) + u * (a.entropy - b.entropy)) / (2 * h)
        assert ((diff - x.grad[:, j]).abs() <= (w.abs() + u.abs()) * 7e-4).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_autograd_matches_torch(ctx, dtype):
    x, t = rows_of(6, 300, dtype, 4)
    a = x.clone().requires_grad_(True)
    b = x.double().clone().requires_grad_(True)
    logp, ent = mx.token_logp(a, t)
    (logp.sum() - 0.1 * ent.sum()).backward()
    lp = torch.log_softmax(b, 1)
    (lp.gather(1, t.long()[:, None]).sum() + 0.1 * (lp.exp() * lp).sum()).backward()
    assert a.grad.dtype == dtype
    if dtype == torch.float32:
        assert float((a.grad.double() - b.grad).norm()) <= 3e-6 * float(b.grad.norm())
    else:                                             # rounded once: half a unit of the last of 8 or 11 bits, each element
        unit = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
        assert ((a.grad.double() - b.grad).abs() <= b.grad.abs() * (unit + 1e-5) + 2.0 ** -24).all()


def test_elements_beyond_32_bits(ctx):
    """Rows that start past 2^31 elements."""
    n, v = 67200, 32000
    assert (n - 1) * v > 2 ** 31
    x = torch.zeros((n, v), dtype=torch.bfloat16, device="cuda")
    last, t = rows_of(3, v, torch.bfloat16, 6)
    x[-3:] = last
    tt = torch.zeros(n, dtype=torch.int32, device="cuda")
    tt[-3:] = t
    r = mx.token_logprobs(x, tt, 2, ctx=ctx)
    close(r.logp[-3:], ref(last, t)[0])
    assert torch.equal(r.top_ids[-3:].long(), top_ref(last, 2))
    g = mx.token_logprobs_grad(x, tt, r.lse, r.entropy, torch.ones(n, device="cuda"), out=x, ctx=ctx)
    small = mx.token_logprobs_grad(last, t, r.lse[-3:].clone(), r.entropy[-3:].clone(), torch.ones(3, device="cuda"), ctx=ctx)
    assert torch.equal(g[-3:], small)
    del x, g
    torch.cuda.empty_cache()


def test_refusals(ctx):
    x, t = rows_of(4, 100, torch.float32, 1)
    r = mx.token_logprobs(x, t, ctx=ctx)
    for f in (lambda: mx.token_logprobs(x, t, 33), lambda: mx.token_logprobs(x, t, -1), lambda: mx.token_logprobs(x[:, :3], t, 4),
              lambda: mx.token_logprobs(x.double(), t), lambda: mx.token_logprobs(x, t.long()), lambda: mx.token_logprobs(x, t[:3]),
              lambda: mx.token_logprobs(x.t(), torch.zeros(100, dtype=torch.int32, device="cuda")), lambda: mx.token_logprobs(x.cpu(), t),
              lambda: mx.token_logprobs(x[0], t), lambda: mx.token_logprobs_grad(x, t, r.lse[:2], r.entropy, r.logp),
              lambda: mx.token_logprobs_grad(x, t, r.lse, None, r.logp, r.logp),
              lambda: mx.token_logprobs_grad(x, t, r.lse, r.entropy, r.logp, out=torch.empty_like(x, dtype=torch.bfloat16))):
        with pytest.raises(ValueError):
            f()
    assert mx.token_logprobs(x[:0], t[:0], 2).top_ids.shape == (0, 2)


def test_gradient_into_the_logits_raises_their_version(ctx):
    """A graph that has saved the logits does not go on with what was written over them."""
    x, t = rows_of(4, 300, torch.float32, 9)
    r = mx.token_logprobs(x, t, ctx=ctx)
    w = torch.ones(4, 300, device="cuda", requires_grad=True)
    y = (x * w).sum()                                 # saves x
    mx.token_logprobs_grad(x, t, r.lse, r.entropy, torch.ones(4, device="cuda"), out=x, ctx=ctx)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    out = torch.empty_like(x)
    before = out._version
    assert mx.token_logprobs_grad(x, t, r.lse, r.entropy, torch.ones(4, device="cuda"), out=out, ctx=ctx) is out
    assert out._version > before
