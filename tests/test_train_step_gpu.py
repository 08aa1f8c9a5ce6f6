"""The example training step: every operator in one graph, forward and backward."""
import math
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_the_example_learns(cuda, dtype):
    import bev_train_step
    losses, norms = bev_train_step.train(30, dtype)
    assert all(math.isfinite(v) for v in losses + norms) and all(n > 0 for n in norms)
    # a fixed map of four classes (log 4 = 1.386 at chance) is being fitted
    assert losses[-1] < 0.8 * losses[0]


def test_every_parameter_gets_the_gradient_of_the_plain_operators(cuda):
    """The example's model with the three operators replaced by torch's: same
    gradients (fp32; the deformable operators are the same on both sides)."""
    import bev_train_step
    from torch import nn

    class Norm(nn.Module):
        def __init__(self, m):
            super().__init__()
            self.weight, self.bias, self.m = m.weight, m.bias, [m]

        def forward(self, x):
            y = nn.functional.group_norm(x, self.m[0].num_groups, self.weight, self.bias, self.m[0].eps)
            return nn.functional.silu(y) if self.m[0].act == "silu" else y.relu()

    class Lookup(nn.Module):
        def __init__(self, m):
            super().__init__()
            self.weight = m.weight

        def forward(self, ids):
            return self.weight[ids]

    torch.manual_seed(1)
    model = bev_train_step.BevHead(64, 12, 10, 3).to(cuda)
    feats = torch.randn(2, 64, 9, 11, device=cuda).contiguous(memory_format=torch.channels_last)
    g = torch.randn(3, 12, 10, device=cuda)

    def grads():
        model.zero_grad()
        # the 1x1 convolution in fp32 too: cuDNN's default is TF32
        with torch.backends.cudnn.flags(enabled=True, allow_tf32=False):
            model(feats).backward(g)
        return {n: p.grad.clone() for n, p in model.named_parameters()}

    own = grads()
    for name in ("norm", "out_norm"):
        setattr(model, name, Norm(getattr(model, name)))
    for name in ("row_pos", "col_pos"):
        setattr(model, name, Lookup(getattr(model, name)))
    plain = grads()
    assert set(own) == set(plain)
    for n in own:
        # chains of a few hundred fp32 roundings through two norms and the attention
        assert float((own[n] - plain[n]).norm()) <= 1e-4 * float(plain[n].norm()) + 1e-6, n


def test_the_step_does_not_wait_for_the_device(cuda):
    """Forward, backward, clipping and the weights' step are only queued."""
    import bev_train_step
    from torch import nn
    model = bev_train_step.BevHead(64, 12, 10, 3).to(cuda)
    feats = torch.randn(2, 64, 9, 11, device=cuda).contiguous(memory_format=torch.channels_last)
    target = torch.randint(0, 3, (1, 12, 10), device=cuda)
    opt = torch.optim.SGD(model.parameters(), lr=0.05, momentum=0.9)

    def step():
        loss = nn.functional.cross_entropy(model(feats).float()[None], target)
        opt.zero_grad(set_to_none=True)
        loss.backward()
        bev_train_step.clip_grad_norm_(model.parameters(), 1.0)
        opt.step()

    step()                                                       # what is set up once
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        step()
    finally:
        torch.cuda.set_sync_debug_mode("default")


def test_meetings_of_two_streams_do_not_mix(cuda):
    """Launches whose CTAs meet, on two streams at once: each starts when all of
    its CTAs fit, and results are those of the calls one after the other."""
    import grad_clip
    import group_norm_act as gna
    g = torch.Generator(cuda).manual_seed(2)
    x = torch.randn(4, 60, 50, 128, generator=g, device=cuda).half().permute(0, 3, 1, 2)
    _, mean, rstd = gna.group_norm_act_forward(x, 8, act="silu")
    grads = [torch.randn(k, generator=g, device=cuda) for k in (5, 300_000, 77, 1_000_000)]
    out = [torch.empty_like(t) for t in grads]
    want = gna.group_norm_act_backward(x, x, mean, rstd, 8, act="silu")[0]
    norm = grad_clip.clip_grads(grads, 1.0, out=out).clone()
    clipped = [o.clone() for o in out]
    torch.cuda.synchronize()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(20):
        with torch.cuda.stream(one):
            got = gna.group_norm_act_backward(x, x, mean, rstd, 8, act="silu")[0]
        with torch.cuda.stream(two):
            again = grad_clip.clip_grads(grads, 1.0, out=out)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(again, norm)
    assert all(torch.equal(a, b) for a, b in zip(out, clipped))
