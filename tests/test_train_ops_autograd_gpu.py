"""What the training-side operators tell autograd: tensors that they write count
a new version, forward-mode tangents are refused instead of dropped, and nothing
that they do becomes part of a graph behind the caller's back."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import grad_clip
import group_norm_act as gna
import scaled_embedding as emb

pytestmark = pytest.mark.gpu


def saved_gradient(device, shape=(6, 8)):
    """A gradient that a graph has saved, and a loss over it."""
    x = torch.randn(shape, generator=torch.Generator(device).manual_seed(0), device=device)
    x.requires_grad_()
    gx, = torch.autograd.grad((x ** 3).sum(), x, create_graph=True)
    return x, gx, (gx * gx).sum()


@pytest.mark.parametrize("limit", [0.1, 1e9], ids=["scaled", "within the limit"])
def test_clipping_counts_versions(cuda, limit):
    wide = torch.ones(8, 12, device=cuda)
    tensors = [torch.ones(5, device=cuda), torch.ones(3, 4, 5, device=cuda).permute(2, 0, 1),
               wide[:, 3:7]]
    before = [t._version for t in tensors]
    grad_clip.grad_norm(tensors)
    assert [t._version for t in tensors] == before               # only read
    grad_clip.clip_grads(tensors, limit)
    after = [t._version for t in tensors]
    assert all(a > b for a, b in zip(after, before))
    out = [torch.zeros_like(t) for t in tensors]
    at = [o._version for o in out]
    grad_clip.clip_grads(tensors, limit, out=out)
    assert all(o._version > v for o, v in zip(out, at))
    assert [t._version for t in tensors] == after                # read again
    p = torch.nn.Parameter(torch.ones(4, device=cuda))
    p.grad = torch.ones(4, device=cuda)
    v = p.grad._version
    grad_clip.clip_grad_norm_([p], limit)
    assert p.grad._version > v and p._version == 0


def test_a_graph_refuses_a_gradient_that_was_clipped_since(cuda):
    x, gx, loss = saved_gradient(cuda)
    grad_clip.clip_grads([gx], 0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_an_added_embedding_gradient_counts_versions(cuda):
    ids = torch.tensor([0, 2, 2], device=cuda)
    _, gx, loss = saved_gradient(cuda)
    v = gx._version
    emb.scaled_embedding_backward(torch.ones(3, 8, device=cuda), ids, 6, grad_weight=gx)
    assert gx._version > v
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_inference_tensors_are_written_as_before(cuda):
    """They have no versions; torch's own operators refuse them outside of
    inference mode, these never have."""
    with torch.inference_mode():
        g = torch.full((4,), 2.0, device=cuda)
    assert float(grad_clip.clip_grads([g], 1.0)) == 4.0
    assert float(g.double().norm()) == pytest.approx(1.0, rel=1e-5)


def test_embedding_gradients_added_to_inference_tensors(cuda):
    with torch.inference_mode():
        main = torch.zeros(6, 8, device=cuda)
    emb.scaled_embedding_backward(torch.ones(1, 8, device=cuda), torch.tensor([5], device=cuda), 6,
                                  grad_weight=main)
    assert float(main[5].sum()) == 8.0


def test_copies_for_gradients_with_holes_stay_out_of_the_graph(cuda):
    """A clipped view of a gradient that is itself part of a graph: its values
    change, its derivative is not replaced by that of the copies."""
    x, gx, _ = saved_gradient(cuda)
    view = gx[:, 2:5]
    grad_clip.clip_grads([view], 0.1)
    assert float(view.detach().double().norm()) == pytest.approx(0.1, rel=1e-5)
    assert gx.grad_fn.name() != "CopySlices"
    leaf = torch.ones(4, 6, device=cuda, requires_grad=True)     # a leaf, dense or through a copy
    grad_clip.clip_grads([leaf], 1.0)
    with torch.no_grad():
        part = leaf[:, 1:3]
    grad_clip.clip_grads([part], 0.5)
    assert float(part.detach().double().norm()) == pytest.approx(0.5, rel=1e-5)


@pytest.mark.parametrize("grad_mode", [True, False], ids=["grad", "no_grad"])
@pytest.mark.parametrize("which", [0, 1, 2], ids=["input", "weight", "bias"])
def test_group_norm_refuses_tangents(cuda, grad_mode, which):
    args = [torch.randn(2, 8, 3, 3, device=cuda), torch.ones(8, device=cuda),
            torch.zeros(8, device=cuda)]
    plain = gna.group_norm_act(args[0], 2, args[1], args[2], act="silu")
    with forward_ad.dual_level(), torch.set_grad_enabled(grad_mode):
        # without tangents the call is what it is outside
        assert torch.equal(gna.group_norm_act(args[0], 2, args[1], args[2], act="silu"), plain)
        dual = list(args)
        dual[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(NotImplementedError):
            gna.group_norm_act(dual[0], 2, dual[1], dual[2], act="silu")
        with pytest.raises(NotImplementedError):
            gna.group_norm_act_forward(dual[0], 2, dual[1], dual[2], act="silu")
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.jvp(lambda t: gna.group_norm_act(t, 2), (args[0],), (torch.ones_like(args[0]),))


def test_the_other_operators_refuse_tangents(cuda):
    x, w = torch.randn(2, 8, 3, 3, device=cuda), torch.randn(5, 8, device=cuda)
    ids, gy = torch.tensor([1, 4], device=cuda), torch.randn(2, 8, device=cuda)
    _, mean, rstd = gna.group_norm_act_forward(x, 2)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        for call in (lambda: gna.group_norm_act_backward(dual(x), x, mean, rstd, 2),
                     lambda: gna.group_norm_act_backward(x, dual(x), mean, rstd, 2),
                     lambda: emb.scaled_embedding(ids, dual(w)),
                     lambda: emb.scaled_embedding_forward(dual(w), ids),
                     lambda: emb.scaled_embedding_backward(dual(gy), ids, 5),
                     lambda: emb.scaled_embedding_backward(gy, ids, 5, grad_weight=dual(w)),
                     lambda: grad_clip.grad_norm([gy, dual(w)]),
                     lambda: grad_clip.clip_grads([gy, dual(w)], 1.0),
                     lambda: grad_clip.clip_grads([gy], 1.0, out=[dual(gy)])):
            with pytest.raises(NotImplementedError):
                call()


def test_a_function_with_a_derivative_of_its_own_may_call_them(cuda):
    """Inside a custom Function, where torch takes care of the tangents itself."""
    class Twice(torch.autograd.Function):
        @staticmethod
        def forward(ctx, w, ids):
            ctx.ids = ids
            return emb.scaled_embedding_forward(w, ids, 2.0)

        @staticmethod
        def jvp(ctx, dw, _):
            return emb.scaled_embedding_forward(dw, ctx.ids, 2.0)

    w, dw = torch.randn(2, 5, 8, device=cuda)
    ids = torch.tensor([1, 4, 1], device=cuda)
    with forward_ad.dual_level():
        y, dy = forward_ad.unpack_dual(Twice.apply(forward_ad.make_dual(w, dw), ids))
    assert torch.equal(y, 2 * w[ids]) and torch.equal(dy, 2 * dw[ids])
