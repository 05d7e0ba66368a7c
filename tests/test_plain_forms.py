"""The plain forms of perf/more_operators.py are yardsticks that run many times over one state: a pass leaves its
inputs as they are, and the next one gives the same."""
import importlib.util
import os

import numpy as np
import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def operators(monkeypatch):
    """The module, its index arrays on the CPU."""
    spec = importlib.util.spec_from_file_location("more_operators_plain", os.path.join(ROOT, "perf", "more_operators.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    arange = torch.arange
    monkeypatch.setattr(torch, "arange", lambda *a, device=None, **k: arange(*a, **k))
    assert not module.own
    return module


@pytest.mark.parametrize("k", [0, 1, 32])
@pytest.mark.parametrize("f32", [False, True])
def test_log_probabilities(operators, f32, k):
    rows, V = 300, 517  # more than one slice of rows
    c = {"kind": "logprobs", "rows": rows, "vocab": V, "pad": 3, "k": k, "f32": f32}
    g = torch.Generator()
    g.manual_seed(k)
    logits = (torch.randn(rows, V + 3, generator=g) * 2).to(torch.float32 if f32 else torch.bfloat16)
    s = {"case": c, "logits": logits, "targets": torch.randint(0, V, (rows,), generator=g, dtype=torch.int32),
         "lp": torch.zeros(rows), "ent": torch.zeros(rows), "ids": torch.zeros(rows, k, dtype=torch.int32),
         "top": torch.zeros(rows, k)}
    before = logits.clone()
    first = [x.clone() for x in operators.run(s)]
    assert torch.equal(logits, before)
    for a, b in zip(first, operators.run(s)):
        assert torch.equal(a, b)

    # ... and it is right.  Differences from the largest are under 32, so an exponential is 3 x 32 + 2 steps of 2^-24 off at
    # most and a sum of V another V of them: under V 2^-22 in all.  The entropy's weighted sum has factors of up to 32, of
    # which the mean is under 10.
    logp = torch.log_softmax(before[:, :V].double(), -1)
    order = np.argsort(-before[:, :V].double().numpy(), 1, kind="stable")[:, :k]
    np.testing.assert_array_equal(first[2].numpy(), order)
    tol = V * 2.0 ** -22
    np.testing.assert_allclose(first[0].double(), logp.gather(1, s["targets"].long()[:, None])[:, 0], atol=tol, rtol=1e-6)
    np.testing.assert_allclose(first[1].double(), -(logp.exp() * logp).sum(-1), atol=tol * 10, rtol=1e-6)
    np.testing.assert_allclose(first[3].double(), logp.gather(1, torch.from_numpy(order.copy())), atol=tol, rtol=1e-6)
