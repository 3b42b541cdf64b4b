"""The serving calls' host side, without a GPU: what autograd is told, the
binding's build and what goes on without it."""
import ctypes
import os
import shutil
import subprocess
import sys

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


def a_package(tmp_path, serve):
    """The package's files with another _serve.so."""
    here = os.path.dirname(os.path.abspath(mx.__file__))
    pkg = tmp_path / "cpu_model_b200"
    pkg.mkdir()
    for f in os.listdir(here):
        if f.endswith(".py"):
            shutil.copy(os.path.join(here, f), pkg / f)
    os.symlink(os.path.join(here, "libmxq.so"), pkg / "libmxq.so")
    if serve is not None:
        (pkg / "_serve.so").write_bytes(serve)
    return tmp_path


@pytest.mark.parametrize("serve", [None, b"built against another torch"])
def test_without_the_binding_the_rest_works(tmp_path, serve):
    """A binding that is not there or does not load is missed by its own calls, with the reason, and by nobody else."""
    code = """
import torch
from cpu_model_b200 import mx
mx.MXContext, mx.mx_linear, mx.MXWeight
calls = [lambda: mx.kv_plan(*[torch.zeros(1)] * 3, None, None, None, 1), lambda: mx.token_logprobs(torch.zeros(1, 1), None),
         lambda: mx.KVCache(None, None, None, None), lambda: mx.KVCache.empty(1, 32, 1, 64)]
for f in calls:
    try:
        f()
    except ImportError as e:
        assert "_serve.so" in str(e) and "cpu_model_b200.build" in str(e), e
    else:
        raise AssertionError("did not say that the binding is missing")
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=a_package(tmp_path, serve), capture_output=True, text=True)
    assert r.returncode == 0, r.stderr


def test_library_builds_without_torch(monkeypatch, capfd):
    """nvcc is enough for the library; the binding is left out, with a word."""
    from cpu_model_b200 import build
    done = []
    monkeypatch.setattr(build, "build_library", lambda *a, **k: done.append("library"))
    monkeypatch.setattr(build.subprocess, "check_call", lambda cmd: done.append(cmd[0]))
    monkeypatch.setitem(sys.modules, "torch", None)
    assert build.build(force=True) == build.LIB
    assert done == ["library"] and "_serve.so" in capfd.readouterr().err


def test_binding_of_another_torch_is_built_again(monkeypatch, tmp_path):
    from cpu_model_b200 import build
    so = tmp_path / "_serve.so"
    monkeypatch.setattr(build, "BINDING", str(so))
    done = []
    monkeypatch.setattr(build, "build_library", lambda *a, **k: done.append("library"))
    monkeypatch.setattr(build, "needs_build", lambda: False)
    monkeypatch.setattr(build.subprocess, "check_call", lambda cmd: (done.append("binding"), open(cmd[cmd.index("-o") + 1], "w").close()))
    build.build()
    assert done == ["binding"] and os.path.exists(so)
    build.build()
    assert done == ["binding"]
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    build.build()
    assert done == ["binding"] * 2


def test_calls_in_the_documents_have_the_library_s_arguments(tmp_path):
    """The documented serving step, compiled with every device array a pointer: an address of one would not do."""
    import glob
    import re
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    calls = []
    for doc in glob.glob(os.path.join(root, "*.md")):
        for block in re.findall(r"```c\n(.*?)```", open(doc).read(), re.S):
            calls += re.findall(r"mxq_(?:kv|token)_\w+\([^;]*\);", block)
    assert len(calls) >= 5
    ints = "past add len table free_pages free_count free_count_dev cu slot position request short_dev chosen top_ids".split()
    src = '#include "mxq.h"\nvoid f(mxq_ctx ctx, mxq_kv_cache* cache, int l, size_t R, size_t page, size_t max_pages, size_t n_pages, size_t n_tokens,\n' \
          '  size_t row_stride, size_t n_heads, size_t max_new, size_t rows, size_t vocab, size_t top_k, float scale, const uint8_t* done,\n' \
          '  const float* q, const float* k, const float* v, const float* logits, float* out, float* lse, float* logp, float* entropy,\n' \
          '  float* top_logp, %s) {\n%s\n}\n' % (", ".join("int32_t* " + n for n in ints), "\n".join(calls))
    (tmp_path / "doc.cpp").write_text(src)
    r = subprocess.run(["g++", "-fsyntax-only", "-I" + os.path.join(root, "include"), str(tmp_path / "doc.cpp")], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr


def test_a_context_of_another_device_is_refused(monkeypatch):
    """Its kernels would run there, on a stream of the tensors' device."""
    class Context:
        device = 1
        h = ctypes.c_void_p(1)

    class OnDevice0:
        def get_device(self):
            return 0
    with pytest.raises(ValueError, match="device"):
        mx._address(Context(), OnDevice0())
    Context.device = 0
    assert mx._address(Context(), OnDevice0()) == 1
