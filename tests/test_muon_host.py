"""What Muon does on the host, over tensors without memory: no GPU needed."""

from __future__ import annotations

import copy
import pickle

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import scao_amd


def _params(n=2):
    return [torch.nn.Parameter(torch.randn(3, 5)) for _ in range(n)]


@pytest.mark.parametrize("ns_dtype", [None, torch.bfloat16])
def test_a_state_of_the_optimizer_whose_arguments_these_are(ns_dtype):
    """torch.optim.Muon's groups know no ns_dtype: it stays as it was given here."""
    if not hasattr(torch.optim, "Muon"):
        pytest.skip("a torch without Muon")
    theirs = torch.optim.Muon(_params(), lr=0.3, weight_decay=0.2)
    for p in theirs.param_groups[0]["params"]:
        theirs.state[p]["momentum_buffer"] = torch.randn(3, 5)
    ours = scao_amd.Muon(_params(), ns_dtype=ns_dtype)
    ours.load_state_dict(theirs.state_dict())
    group = ours.param_groups[0]
    assert (group["lr"], group["weight_decay"], group["ns_dtype"]) == (0.3, 0.2, ns_dtype)
    assert len(ours._check(group)) == 3 * 5
    for p, q in zip(group["params"], theirs.param_groups[0]["params"]):
        assert torch.equal(ours.state[p]["momentum_buffer"], theirs.state[q]["momentum_buffer"])
    # and what is copied or pickled has it too
    for twin in (copy.deepcopy(ours), pickle.loads(pickle.dumps(ours))):
        assert twin.param_groups[0]["ns_dtype"] is ns_dtype


def test_a_first_step_is_not_captured(monkeypatch):
    """Replays of a graph that holds the momentum's zeroing would all start from zero."""
    with FakeTensorMode():
        p = torch.nn.Parameter(torch.empty(8, 16, device="cuda"))
        p.grad = torch.empty(8, 16, device="cuda")
        opt = scao_amd.Muon([p])
        monkeypatch.setattr(torch.cuda, "is_initialized", lambda: True)
        monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        with pytest.raises(RuntimeError, match="captured"):
            opt.step()
        assert "momentum_buffer" not in opt.state[p]
        # one of another type would be converted at every replay, from where it was
        opt.state[p]["momentum_buffer"] = torch.empty(8, 16, device="cuda", dtype=torch.bfloat16)
        with pytest.raises(RuntimeError, match="captured"):
            opt.step()
        opt.state[p]["momentum_buffer"] = torch.empty(8, 16, device="cuda")
        opt.step()


def test_a_refused_step_steps_no_group(monkeypatch):
    steps = []
    monkeypatch.setattr(scao_amd._lib.torch_host(), "muon_step", lambda *a: steps.append(a))
    with FakeTensorMode():
        good, bad = (torch.nn.Parameter(torch.empty(s, device="cuda")) for s in ((8, 16), (4, 4)))
        good.grad, bad.grad = torch.empty(8, 16, device="cuda"), torch.empty(4, 4, device="cuda")
        opt = scao_amd.Muon([dict(params=[good]), dict(params=[bad])])
        opt.step()
        assert len(steps) == 2
        turned = torch.nn.Parameter(torch.empty(4, 6, device="cuda").t())
        turned.grad = torch.empty(6, 4, device="cuda")
        opt.add_param_group(dict(params=[turned]))
        with pytest.raises(ValueError, match="contiguous"):
            opt.step()
        turned.grad = None
        opt.param_groups[1]["lr"] = float("nan")
        with pytest.raises(ValueError, match="lr"):
            opt.step()
        assert len(steps) == 2
