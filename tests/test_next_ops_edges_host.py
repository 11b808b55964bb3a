"""Refusals of the operators from hidden states to ids that need no GPU: they come before anything is looked for on one."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad


@pytest.fixture(scope="module")
def ops(built):
    from graphtok_b200 import next_ops
    return next_ops


def calls_with(ops):
    """Each call that could pass a gradient on to what it is given, by the argument's name."""
    logits, u, ids, offsets = torch.zeros(2, 5), torch.zeros(2), torch.zeros(4, dtype=torch.int32), torch.tensor([0, 2, 4], dtype=torch.int32)
    for name in ("repetition", "presence", "frequency"):
        yield name, lambda t, name=name: ops.adjust_logits(logits, ids, offsets, **{name: t})
    for name in ("temperature", "top_p", "min_p"):
        yield name, lambda t, name=name: ops.sample(logits, u, **{name: t})
    yield "u", lambda t: ops.sample(logits, t)


def test_gradients_of_penalties_and_wishes_are_refused(ops):
    """A learned penalty or temperature would be trained with nothing, and nobody told."""
    for name, call in calls_with(ops):
        leaf = torch.ones(2, requires_grad=True)
        with pytest.raises(NotImplementedError, match="no gradient"):
            call(leaf)
        with pytest.raises(NotImplementedError, match="no gradient"):
            call(leaf * 0.5)
        for fine in (leaf.detach(), torch.ones(2)):
            with pytest.raises(ValueError, match="must be on the GPU"):
                call(fine)
        with torch.no_grad(), pytest.raises(ValueError, match="must be on the GPU"):
            call(leaf)
        with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
            call(forward_ad.make_dual(torch.ones(2), torch.ones(2)))


def test_penalties_without_a_history_are_refused(ops, monkeypatch):
    """They would change nothing, whatever they say.  (The checks behind the GPU's are reached as on one.)"""
    monkeypatch.setattr(ops, "_on_gpu", lambda first, **others: 0)
    monkeypatch.setattr(ops, "_there", lambda index, f, *args: args[-1])
    logits = torch.zeros(2, 5)
    for name, none in (("repetition", 1.0), ("presence", 0.0), ("frequency", 0.0)):
        for value in (1.2, -1.0, float("nan"), float("inf"), torch.ones(2), torch.ones(3)):
            with pytest.raises(ValueError, match=name + " without ids"):
                ops.adjust_logits(logits, **{name: value})
        assert ops.adjust_logits(logits, **{name: none}) and ops.adjust_logits(logits, **{name: int(none)})
    with pytest.raises(ValueError, match="prompt_lengths without ids"):
        ops.adjust_logits(logits, prompt_lengths=torch.zeros(2, dtype=torch.int32))
