"""GPU: what autograd has to know of the sequence operators: writes in place, tangents, traces."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from test_gpu_sequence import DEV, _case, _dev, _seq

pytestmark = pytest.mark.gpu


def _step(d, state, **kw):
    return _seq().linear_attention_step(d["q"][0], d["k"][0], d["v"][0], d["log_decay"], state, **kw)


@pytest.mark.parametrize("out", [False, True])
def test_a_step_on_a_saved_state_is_seen(out):
    """The backward pass reads the initial state again: after a step has written into it, the pass is refused."""
    d = _dev(_case(6, 2, 2, 16, 16, torch.float32))
    q, state = d["q"].requires_grad_(), d["state"]
    y, _ = _seq().linear_attention(q, d["k"], d["v"], d["log_decay"], state)
    version = state._version
    with torch.no_grad():
        if out:
            _step(d, torch.zeros_like(state), state_out=state)
        else:
            _step(d, state)
    assert state._version > version
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(y, q, d["dout"])
    # a state that is only read stays as it is
    y, _ = _seq().linear_attention(q, d["k"], d["v"], d["log_decay"], state)
    with torch.no_grad():
        _step(d, state, state_out=torch.empty_like(state))
    torch.autograd.grad(y, q, d["dout"])


def test_a_state_out_that_requires_a_gradient_is_refused():
    """What autograd knows of such a tensor would not be what it holds."""
    d = _dev(_case(1, 2, 2, 16, 16, torch.float32))
    leaf = torch.zeros_like(d["state"]).requires_grad_()
    for out in (leaf, leaf * 2):
        with pytest.raises(ValueError, match="no gradient"):
            _step(d, d["state"], state_out=out)
    with torch.no_grad():
        _step(d, d["state"], state_out=leaf)
    assert bool(leaf.detach().any())


def test_steps_in_inference_mode():
    d = _dev(_case(1, 2, 2, 16, 16, torch.float32))
    want = _step(d, d["state"].clone())
    with torch.inference_mode():
        got = _step(d, d["state"].clone())  # a state without a version
        again = _step(d, d["state"])        # one with
    assert torch.equal(got, want) and torch.equal(again, want)


@pytest.mark.parametrize("graph", [False, True])
def test_a_collection_on_a_saved_memory_is_seen(graph):
    from test_gpu_retention import _setup
    env, policy, buf, col = _setup(16, 8)
    col.collect()
    values, log_probs, _ = policy.evaluate_actions(buf.observations.clone(), buf.actions.clone(), buf.dones.clone(), col.memory)
    col.collect(graph=graph)
    with pytest.raises(RuntimeError, match="inplace"):
        (values.sum() + log_probs.sum()).backward()
    env.close()


def test_tangents_are_refused():
    """The operators have no forward-mode derivative; without one their results would be constants."""
    d = _dev(_case(6, 2, 2, 16, 16, torch.float32))
    s = _seq()
    with fwd.dual_level():
        for n in ("q", "k", "v", "state"):
            a = dict(d, **{n: fwd.make_dual(d[n], torch.ones_like(d[n]))})
            for grad in (False, True):
                with torch.set_grad_enabled(grad):
                    with pytest.raises(ValueError, match="forward-mode"):
                        s.linear_attention(a["q"], a["k"], a["v"], a["log_decay"], a["state"])
            with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):
                _step(a, a["state"])
            with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):
                _step(d, d["state"], state_out=fwd.make_dual(torch.zeros_like(d["state"]), torch.ones_like(d["state"])))
        ld = fwd.make_dual(d["log_decay"], torch.ones_like(d["log_decay"]))
        with pytest.raises(ValueError, match="forward-mode"):
            s.linear_attention(d["q"], d["k"], d["v"], ld, d["state"])
        x, w = torch.randn(4, 8, device=DEV), torch.ones(8, device=DEV)
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))
        for a in ((dual(x), w, w), (x, dual(w), w), (x, w, dual(w))):
            with pytest.raises(ValueError, match="forward-mode"):
                s.group_norm_act(a[0], 2, a[1], a[2])
        s.linear_attention(d["q"], d["k"], d["v"], d["log_decay"], d["state"])  # without a tangent: as ever
        s.group_norm_act(x, 2, w, w)
        # a gradient that carries one
        q = d["q"].detach().requires_grad_()
        out, _ = s.linear_attention(q, d["k"], d["v"], d["log_decay"], d["state"])
        with pytest.raises(ValueError, match="forward-mode"):
            torch.autograd.grad(out, q, dual(torch.ones_like(out)))
        x.requires_grad_()
        y = s.group_norm_act(x, 2, w, w)
        with pytest.raises(ValueError, match="forward-mode"):
            torch.autograd.grad(y, x, dual(torch.ones_like(y)))


def test_traces_are_refused():
    """A trace would hold the allocation of the results and no operator."""
    d = _dev(_case(6, 2, 2, 16, 16, torch.float32))
    s = _seq()
    calls = [(lambda q: s.linear_attention(q, d["k"], d["v"], d["log_decay"])[0], d["q"]),
             (lambda q: s.linear_attention_step(q, d["k"][0], d["v"][0], d["log_decay"], d["state"]), d["q"][0]),
             (lambda x: s.group_norm_act(x, 4), torch.randn(4, 8, device=DEV))]
    for f, x in calls:
        with pytest.raises(RuntimeError, match="trac"):
            torch.jit.trace(f, (x,), check_trace=False)
    x = torch.randn(4, 8, device=DEV, requires_grad=True)
    with pytest.raises(RuntimeError, match="trac"):
        torch.jit.trace(lambda x: s.group_norm_act(x, 4), (x,), check_trace=False)
