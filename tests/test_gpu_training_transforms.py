"""``torch.ops.rwkv_tl.embed``, ``.layer_norm`` and ``.token_logprobs`` under autograd's batching, vmap, checkpointing, saved-
tensor hooks and graph capture: the same bits as the kernels called one by one; and the transforms that are refused."""

from __future__ import annotations

import pytest
import torch
import torch.utils.checkpoint

import rwkv_tl_amd  # noqa: F401
from rwkv_tl_amd import kernels as K

pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore:There is a performance drop")]
ops = torch.ops.rwkv_tl
N, C, V = 6, 72, 305


@pytest.fixture
def data(cuda):
    g = torch.Generator().manual_seed(11)
    r = lambda *s: torch.randn(*s, generator=g).to(cuda)  # noqa: E731
    t = torch.randint(0, V, (N,), generator=g)
    t[2] = -1
    return {"table": r(V, C), "t": t.to(cuda), "x": r(N, C), "w": r(C), "b": r(C), "z": 3 * r(N, V), "dy": r(N, C), "s": r(N), "h": r(N),
            "many": r(3, N, C), "ups": r(3, N)}


def _lp_grad(d, s, h):
    return K.token_logprobs_backward(s, h, d["z"], d["t"], 0.7)


def test_batched_gradients(data):
    d = data
    w = d["table"].clone().requires_grad_()
    (got,) = torch.autograd.grad(ops.embed(w, d["t"], 2.0), w, d["many"], is_grads_batched=True)
    assert torch.equal(got, torch.stack([K.embed_backward(g, d["t"], V, scale=2.0) for g in d["many"]]))
    leaves = [d[k].clone().requires_grad_() for k in ("x", "w", "b")]
    got = torch.autograd.grad(ops.layer_norm(*leaves), leaves, d["many"], is_grads_batched=True)
    _, m, r = K.layer_norm_forward(d["x"], d["w"], d["b"])
    want = [K.layer_norm_backward(g, d["x"], d["w"], m, r) for g in d["many"]]
    assert all(torch.equal(a, torch.stack(b)) for a, b in zip(got, zip(*want)))
    z = d["z"].clone().requires_grad_()
    lp, ent = ops.token_logprobs(z, d["t"], 0.7)
    (got,) = torch.autograd.grad((lp, ent), z, (d["ups"], d["ups"].flip(0)), is_grads_batched=True)
    assert torch.equal(got, torch.stack([_lp_grad(d, a, b) for a, b in zip(d["ups"], d["ups"].flip(0))]))


@pytest.mark.parametrize("which", ["logprob", "entropy"])
def test_one_gradient_of_two_batched(data, which):
    """The other one the same for the whole batch."""
    d = data
    z = d["z"].clone().requires_grad_()
    out = ops.token_logprobs(z, d["t"], 0.7)
    pair = (lambda u: (u, d["h"])) if which == "logprob" else (lambda u: (d["s"], u))
    got = torch.vmap(lambda u: torch.autograd.grad(out, z, pair(u), retain_graph=True)[0])(d["ups"])
    assert torch.equal(got, torch.stack([_lp_grad(d, *pair(u)) for u in d["ups"]]))
    got = torch.vmap(lambda u: torch.autograd.grad(out[which == "entropy"], z, u, retain_graph=True)[0])(d["ups"])
    assert torch.equal(got, torch.stack([_lp_grad(d, *((u, None) if which == "logprob" else (None, u))) for u in d["ups"]]))


def test_vectorized_jacobian(data):
    d = data
    got = torch.autograd.functional.jacobian(lambda z: ops.token_logprobs(z, d["t"], 0.7)[0], d["z"], vectorize=True)
    want = torch.zeros(N, N, V, device=got.device)
    want[range(N), range(N)] = _lp_grad(d, torch.ones(N, device=got.device), None)
    assert torch.equal(got, want)
    got = torch.autograd.functional.jacobian(lambda b: ops.layer_norm(d["x"], d["w"], b), d["b"], vectorize=True)
    assert torch.equal(got, torch.eye(C, device=got.device).expand(N, C, C))


def test_vmap(data):
    d = data
    assert torch.equal(torch.vmap(lambda t: ops.embed(d["table"], t))(d["t"]), K.embed(d["table"], d["t"]))
    tables = torch.stack([d["table"], -d["table"]])
    assert torch.equal(torch.vmap(lambda w: ops.embed(w, d["t"], 0.5))(tables), torch.stack([K.embed(w, d["t"], scale=0.5) for w in tables]))
    norm = lambda x, w, b: K.layer_norm_forward(x, w, b)[0]  # noqa: E731
    got = torch.vmap(lambda x: ops.layer_norm(x, d["w"], d["b"]))(d["many"])
    assert torch.equal(got, norm(d["many"], d["w"], d["b"]))
    got = torch.vmap(lambda w: ops.layer_norm(d["x"], w, d["b"]))(torch.stack([d["w"], d["b"]]))  # x is the same for all
    assert torch.equal(got, torch.stack([norm(d["x"], w, d["b"]) for w in (d["w"], d["b"])]))
    got = torch.vmap(lambda b: ops.layer_norm(d["x"], d["w"], b))(torch.stack([d["w"], d["b"]]))
    assert torch.equal(got, torch.stack([norm(d["x"], d["w"], b) for b in (d["w"], d["b"])]))
    got = torch.vmap(lambda z, t: ops.token_logprobs(z, t, 0.7))(d["z"], d["t"])
    assert all(torch.equal(a, b) for a, b in zip(got, K.token_logprobs(d["z"], d["t"], temperature=0.7)))
    got = torch.vmap(lambda t: ops.token_logprobs(d["z"][0], t, 0.7))(d["t"])  # many tokens of one row
    want = K.token_logprobs(d["z"][:1].expand(N, V), d["t"], temperature=0.7)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_gradients_through_vmap(data):
    """Leaves outside, the operators inside: gradients of the batch."""
    d = data
    x, w, b = (d[k].clone().requires_grad_() for k in ("many", "w", "b"))
    y = torch.vmap(lambda u: ops.layer_norm(u, w, b))(x)
    up = d["many"].flip(0)
    got = torch.autograd.grad(y, (x, w, b), up)
    _, m, r = K.layer_norm_forward(d["many"], d["w"], d["b"])
    want = [K.layer_norm_backward(g, u, d["w"], p, q) for g, u, p, q in zip(up, d["many"], m, r)]
    assert torch.equal(got[0], torch.stack([v[0] for v in want]))
    for i in (1, 2):  # (three slices' sums, in either order)
        assert torch.allclose(got[i], sum(v[i] for v in want), rtol=1e-5, atol=1e-5)
    z = d["z"].clone().requires_grad_()
    lp, ent = torch.vmap(lambda u, t: ops.token_logprobs(u, t, 0.7))(z, d["t"])
    assert torch.equal(torch.autograd.grad((lp, ent), z, (d["s"], d["h"]))[0], _lp_grad(d, d["s"], d["h"]))


def _step(d, table, w, b):
    y = ops.layer_norm(ops.embed(table, d["t"], 1.5), w, b)
    lp, ent = ops.token_logprobs(y @ table.t(), d["t"], 0.7)
    return lp.sum() + 0.1 * ent.sum()


def _leaves(d):
    return [d[k].clone().requires_grad_() for k in ("table", "w", "b")]


def test_checkpointing_and_saved_tensor_hooks(data):
    d = data
    leaves = _leaves(d)
    want = torch.autograd.grad(_step(d, *leaves), leaves)
    for reentrant in (False, True):
        loss = torch.utils.checkpoint.checkpoint(lambda *a: _step(d, *a), *leaves, use_reentrant=reentrant)
        for v in leaves:
            v.grad = None
        loss.backward()
        assert all(torch.equal(v.grad, u) for v, u in zip(leaves, want))
    with torch.autograd.graph.save_on_cpu():
        loss = _step(d, *leaves)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(loss, leaves), want))


def test_saved_tensors_changed_in_place_are_refused(data):
    d = data
    x, z, t = d["x"].clone(), d["z"].clone(), d["t"].clone()
    w = d["w"].clone().requires_grad_()
    y = ops.layer_norm(x, w, d["b"])
    lp, _ = ops.token_logprobs(z * w.sum(), t)
    e = ops.embed(d["table"].clone().requires_grad_(), t)
    x.add_(1)
    t.add_(1)
    for out in (y, lp, e):
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.sum().backward()


def test_captured_steps(data):
    """A step through autograd captured once and replayed on other inputs, eager work between the replays."""
    d = data
    leaves = _leaves(d)

    def step():
        loss = _step(d, *leaves)
        return loss.detach(), *torch.autograd.grad(loss, leaves)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        with torch.no_grad():
            leaves[0].mul_(1.25)
            d["t"].copy_(torch.randint(-1, V, (N,), generator=torch.Generator().manual_seed(i)))
        graph.replay()
        torch.cuda.synchronize()
        got = [v.clone() for v in out]
        want = step()
        assert all(torch.allclose(a, b, rtol=1e-6, atol=1e-6) for a, b in zip(got, want))  # (the table's gradients: in either order)


def test_transforms_without_a_rule_are_refused(data):
    d = data
    calls = {"table": lambda v: ops.embed(v, d["t"]).sum(), "x": lambda v: ops.layer_norm(v, d["w"], d["b"]).sum(),
             "z": lambda v: ops.token_logprobs(v, d["t"])[0].sum()}
    for k, f in calls.items():
        with pytest.raises(RuntimeError, match="setup_context"):  # torch's own refusal, as of its registered operators
            torch.func.grad(f)(d[k])
        with pytest.raises(NotImplementedError, match="jvp"), torch.autograd.forward_ad.dual_level():
            f(torch.autograd.forward_ad.make_dual(d[k], d[k]))
