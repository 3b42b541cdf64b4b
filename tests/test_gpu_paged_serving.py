"""The paged serving example end to end: what decoding step by step over the
8-bit cache says of a sequence is what one pass over the whole sequence says,
requests that share the pool do not disturb one another, every page comes back."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def serving():
    spec = importlib.util.spec_from_file_location("paged_serving", os.path.join(ROOT, "examples", "paged_serving.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_steps_agree_with_whole_sequences(serving):
    from cpu_model_b200 import mx
    cfg = serving.Config(layers=2, dim=256, heads=4, kv_heads=2, head_dim=64, ffn=512, vocab=1000, page=32, pages=40, slots=4, max_pages=10)
    model = serving.PagedDecoder(cfg, seed=3)
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, cfg.vocab, (n,), generator=g).tolist() for n in (7, 100, 33, 1, 64, 31)]
    results = serving.generate(model, prompts, 20, top_k=3)
    assert int(model.free_count) == cfg.pages and sorted(model.free.tolist()) == list(range(cfg.pages))
    assert (model.table == -1).all() and (model.lengths == 0).all()
    for ids in ((0, 1, 2, 3), (4, 5)):
        seqs = [prompts[i] + results[i][0] for i in ids]
        logits, targets = serving.score(model, seqs)
        r = mx.token_logprobs(logits, targets)
        at = 0
        for i, s in zip(ids, seqs):
            n = len(prompts[i])
            logp = r.logp[at + n - 1:at + len(s) - 1].cpu()
            ent = r.entropy[at + n - 1:at + len(s) - 1].cpu()
            # the same rows of K and V, but a block that grew a token at a time was
            # re-rounded when its scale rose: up to a step of 2^-7 of its largest value more.
            # Through two layers that moves a logit (of order 1) by a few hundredths.
            assert (logp - torch.tensor(results[i][1])).abs().max() <= 0.15
            assert (ent - torch.tensor(results[i][2])).abs().max() <= 0.15
            at += len(s)
        assert r.logp[at - 1] == 0          # a target of -1


def test_requests_do_not_disturb_one_another(serving):
    cfg = serving.Config(layers=1, dim=256, heads=2, kv_heads=1, head_dim=128, ffn=256, vocab=500, page=32, pages=30, slots=3, max_pages=8)
    g = torch.Generator().manual_seed(5)
    prompts = [torch.randint(0, cfg.vocab, (n,), generator=g).tolist() for n in (40, 3, 77, 12)]
    model = serving.PagedDecoder(cfg, seed=4)
    together = serving.generate(model, prompts, 10)
    for i, p in enumerate(prompts):
        alone = serving.generate(serving.PagedDecoder(cfg, seed=4), [p], 10)[0]
        assert alone[0] == together[i][0]
        assert max(abs(a - b) for a, b in zip(alone[1], together[i][1])) <= 1e-3


def test_gradient_of_the_generated_tokens(serving):
    from cpu_model_b200 import mx
    cfg = serving.Config(layers=1, dim=256, heads=2, kv_heads=1, head_dim=64, ffn=256, vocab=300, page=32, pages=20, slots=2, max_pages=8)
    model = serving.PagedDecoder(cfg, seed=6)
    logits, targets = serving.score(model, [[1, 2, 3, 4, 5], [9, 8, 7]])
    logits.requires_grad_(True)
    logp, entropy = mx.token_logp(logits, targets)
    logp.sum().backward()
    assert (logits.grad[4] == 0).all() and (logits.grad[7] == 0).all()      # rows without a target
    want = -torch.softmax(logits.detach().double(), 1)
    rows = [0, 1, 2, 3, 5, 6]
    want[rows, targets[rows].long()] += 1
    assert float((logits.grad[rows].double() - want[rows]).norm() / want[rows].norm()) <= 3e-6
