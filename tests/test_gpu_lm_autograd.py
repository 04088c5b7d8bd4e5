"""What torch's differentiation modes get of the language-model operators besides
the gradients."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


def calls():
    """Each operator as a function of one float32 tensor [4, 2, 8] or [4, 8]."""
    import prlstm_b200 as P

    z, h = torch.randn(4, 2, 8, device=DEV), torch.randn(2, 8, device=DEV)
    tok = torch.tensor([1, 3, 0, 2], device=DEV)
    return {
        "gated z": (lambda t: P.gated_recurrence(t, z, h), (4, 2, 8)),
        "gated x": (lambda t: P.gated_recurrence(z, t), (4, 2, 8)),
        "linear b": (lambda t: P.linear_recurrence(z, t, h), (4, 2, 8)),
        "state": (lambda t: P.linear_recurrence(z, z, t), (2, 8)),
        "gated step": (lambda t: P.gated_recurrence_step(t, h, h), (2, 8)),
        "linear step": (lambda t: P.linear_recurrence_step(h, h, t), (2, 8)),
        "embedding": (lambda t: P.embedding(tok, t), (4, 8)),
        "logits": (lambda t: P.token_logprobs(t, tok, top=2), (4, 8)),
    }


@pytest.mark.parametrize("name", ["gated z", "gated x", "linear b", "state", "gated step", "linear step", "embedding", "logits"])
def test_forward_mode_is_refused(name):
    """A tangent is refused, with or without a graph; a tensor without one is not."""
    call, shape = calls()[name]
    t = torch.randn(*shape, device=DEV)
    want = call(t)
    with fwd.dual_level():
        dual = fwd.make_dual(t, torch.ones_like(t))
        with pytest.raises(NotImplementedError):
            call(dual)
        with torch.no_grad(), pytest.raises(NotImplementedError):
            call(dual)
        got = call(t)
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.jvp(call, (t,), (torch.ones_like(t),))
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.vmap(call)(t[None])
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.grad(lambda t: (out := call(t), out if isinstance(out, torch.Tensor) else out[0])[1].sum())(t)
    leaves = [got, want] if isinstance(got, torch.Tensor) else list(zip(got, want))
    for pair in ([leaves] if isinstance(got, torch.Tensor) else leaves):
        assert pair[0] is pair[1] or torch.equal(pair[0], pair[1])
