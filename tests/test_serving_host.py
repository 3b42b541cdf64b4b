"""The serving calls' host side, without a GPU: what autograd is told."""
import pytest
import torch

from cpu_model_b200 import mx


@pytest.fixture
def on_cpu(monkeypatch):
    """token_logprobs and its gradient in torch operations."""
    def forward(logits, targets, top_k=0, ctx=None):
        lp = torch.log_softmax(logits.detach().float(), 1)
        return mx.TokenLogprobs(lp.gather(1, targets.long()[:, None])[:, 0], -(lp.exp() * lp).sum(1), torch.logsumexp(logits.detach().float(), 1))

    def grad(logits, targets, lse, entropy, dlogp=None, dentropy=None, out=None, ctx=None):
        with torch.no_grad():
            lp = logits.float() - lse[:, None]
            hit = torch.nn.functional.one_hot(targets.long(), logits.shape[1])
            g = dlogp[:, None] * (hit - lp.exp()) - dentropy[:, None] * lp.exp() * (lp + entropy[:, None])
            return g.to(logits.dtype)
    monkeypatch.setattr(mx, "token_logprobs", forward)
    monkeypatch.setattr(mx, "token_logprobs_grad", grad)


def test_second_derivatives_are_refused(on_cpu):
    """The gradient is not differentiable; it does not pass for a constant."""
    x = torch.randn(3, 7, requires_grad=True)
    t = torch.tensor([1, 0, 6], dtype=torch.int32)
    logp, ent = mx.token_logp(x, t)
    (logp.sum() + ent.sum()).backward()
    y = x.detach().double().requires_grad_(True)
    lp = torch.log_softmax(y, 1)
    (lp.gather(1, t.long()[:, None]).sum() - (lp.exp() * lp).sum()).backward()
    assert float((x.grad - y.grad).abs().max()) <= 1e-5
    logp, ent = mx.token_logp(x, t)
    g, = torch.autograd.grad(logp.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        (g.square().sum() + logp.sum()).backward()
    mx.token_logp(x, t)[0].sum().backward()          # the first still goes
