"""Group norm with activation against its formulas in 64 bits, forward and backward.

Tolerances.  A result is rounded once to its type (u = 2^-24, 2^-11, 2^-8 for
fp32, fp16, bf16).  Before that the kernel works in fp32: x - mean carries the
rounding of the mean, |mean| / sd units of relative error, and the chain after
it a handful of roundings, so the relative L2 error of y and dx is taken as
u_type + 16 u32 (1 + max |mean| / sd).  Channel sums may be off by 64 u32 of the sum of
their terms' magnitudes (short chains per thread, then a tree), plus the type's
rounding.
"""
import pytest
import torch

import group_norm_act as gna
from helpers import rel_l2

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
IDS = ["f32", "f16", "bf16"]
EPS = 1e-5


def reference(x, gy, weight, bias, groups, act, eps=EPS):
    """The formulas in fp64 -> dict of outputs, gradients and error scales."""
    n, c = x.shape[:2]
    xd = x.detach().double().reshape(n, groups, c // groups, -1)
    w = torch.ones(c, dtype=torch.float64, device=x.device) if weight is None else weight.double()
    b = torch.zeros(c, dtype=torch.float64, device=x.device) if bias is None else bias.double()
    w, b = (t.detach().view(1, groups, c // groups, 1) for t in (w, b))
    mean = xd.mean((2, 3), keepdim=True)
    var = (xd - mean).square().mean((2, 3), keepdim=True)
    rstd = 1 / (var + eps).sqrt()
    xhat = (xd - mean) * rstd
    z = xhat * w + b
    sig = torch.sigmoid(z)
    y = {"none": z, "relu": z.clamp_min(0), "silu": z * sig}[act]
    out = {"y": y.reshape(x.shape), "mean": mean.view(n, groups), "rstd": rstd.view(n, groups),
           "ratio": float((mean.abs() * rstd).max())}
    if gy is None:
        return out
    slope = {"none": torch.ones_like(z), "relu": (z > 0).double(),
             "silu": sig * (1 + z * (1 - sig))}[act]
    dz = gy.double().reshape(xd.shape) * slope
    dxh = dz * w
    dx = rstd * (dxh - dxh.mean((2, 3), keepdim=True) - xhat * (dxh * xhat).mean((2, 3), keepdim=True))
    out.update(dx=dx.reshape(x.shape), dw=(dz * xhat).sum((0, 3)).view(c), db=dz.sum((0, 3)).view(c),
               dw_abs=(dz * xhat).abs().sum((0, 3)).view(c), db_abs=dz.abs().sum((0, 3)).view(c))
    return out


def inputs(seed, shape, dt, pdt, device, mean=0.5):
    g = torch.Generator(device).manual_seed(seed)
    n, c = shape[:2]
    rows = [n, *shape[2:], c]
    x = torch.randn(rows, generator=g, device=device) + mean * torch.randn(c, generator=g, device=device)
    gy = torch.randn(rows, generator=g, device=device)
    w = 1 + 0.3 * torch.randn(c, generator=g, device=device)
    b = 0.3 * torch.randn(c, generator=g, device=device)
    return (x.to(dt).movedim(-1, 1), gy.to(dt).movedim(-1, 1), w.to(pdt), b.to(pdt))


def check_forward(got, ref, dt):
    assert rel_l2(got, ref["y"]) <= UNIT[dt] + 16 * U32 * (1 + ref["ratio"])


def check_backward(got, ref, dt, pdt):
    gi, gw, gb = got
    assert rel_l2(gi, ref["dx"]) <= UNIT[dt] + 16 * U32 * (1 + ref["ratio"])
    for t, k in ((gw, "dw"), (gb, "db")):
        if t is not None:
            lim = (64 * U32 * (1 + ref["ratio"])) * ref[k + "_abs"] + UNIT[pdt] * ref[k].abs()
            assert bool(((t.double() - ref[k]).abs() <= lim + 1e-30).all()), k


SHAPES = [
    ((2, 64, 9, 7), 8),        # whole vectors per group
    ((1, 21, 5, 3), 3),        # no 16-byte rows: one channel at a time
    ((3, 40, 4, 6), 8),        # five channels a group: vectors cross groups
    ((2, 96, 13, 11), 1),      # one group
    ((2, 48, 17, 5), 48),      # instance norm
    ((1, 64, 1, 8), 8),        # a row of pixels
    ((5, 32, 1, 1), 2),        # a single pixel
    ((2, 24, 37), 3),          # one spatial axis
    ((2, 16, 3, 4, 5), 4),     # three
    ((1, 1500, 3, 2), 4),      # fp16: three channel blocks, groups across them
    ((2, 6000, 2, 3), 3),      # several channel blocks of vectors, groups across them
    ((300, 8, 2, 9), 4),       # more images than CTAs
    ((700, 16, 3, 3), 2),
    ((1, 256, 50, 41), 32),    # many slabs of one image
]


@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape,groups", SHAPES, ids=["x".join(map(str, s)) + f"g{g}" for s, g in SHAPES])
def test_matches_formula(cuda, shape, groups, dt):
    x, gy, w, b = inputs(1, shape, dt, torch.float32, cuda)
    # a smooth activation: a ReLU's slope at arguments within rounding of zero
    # is either of two right answers
    ref = reference(x, gy, w, b, groups, "silu")
    y, mean, rstd = gna.group_norm_act_forward(x, groups, w, b, EPS, "silu")
    assert y.dtype == dt and y.shape == x.shape and mean.dtype == torch.float32
    check_forward(y, ref, dt)
    scale = 1 / ref["rstd"]
    assert bool(((mean.double() - ref["mean"]).abs() <= 16 * U32 * (ref["mean"].abs() + scale)).all())
    assert bool(((rstd.double() / ref["rstd"] - 1).abs() <= 16 * U32 * (1 + ref["ratio"])).all())
    got = gna.group_norm_act_backward(gy, x, mean, rstd, groups, w, b, "silu")
    assert got[0].shape == x.shape and got[0].dtype == dt
    assert got[1].dtype == torch.float32 and got[1].shape == (shape[1],)
    check_backward(got, ref, dt, torch.float32)


@pytest.mark.parametrize("act", ["none", "relu", "silu"])
@pytest.mark.parametrize("params", ["both", "weight", "bias", "neither"])
def test_activations_and_parameters(cuda, act, params):
    x, gy, w, b = inputs(2, (2, 64, 11, 6), torch.float16, torch.float16, cuda)
    w = w if params in ("both", "weight") else None
    b = b if params in ("both", "bias") else None
    ref = reference(x, gy, w, b, 8, act)
    y, mean, rstd = gna.group_norm_act_forward(x, 8, w, b, EPS, act)
    check_forward(y, ref, torch.float16)
    if act == "relu":  # arguments within rounding of zero get no gradient in this test
        near = reference(x, None, w, b, 8, "none")["y"].abs() < 1e-5
        gy = gy.masked_fill(near, 0)
        ref = reference(x, gy, w, b, 8, act)
    got = gna.group_norm_act_backward(gy, x, mean, rstd, 8, w, b, act)
    assert (got[1] is None) == (w is None) and (got[2] is None) == (b is None)
    check_backward(got, ref, torch.float16, torch.float16)
    # the module-level call without gradients returns the same bits
    assert torch.equal(gna.group_norm_act(x, 8, w, b, EPS, act), y)


def test_relu_keeps_nan_and_zero_slope_at_zero(cuda):
    x = torch.zeros(1, 8, 2, 2, device=cuda)
    y, mean, rstd = gna.group_norm_act_forward(x, 2, act="relu")
    assert torch.equal(y, x) and float(rstd[0, 0]) == pytest.approx(EPS ** -0.5, rel=1e-6)
    gi, _, _ = gna.group_norm_act_backward(torch.ones_like(x), x, mean, rstd, 2, act="relu")
    assert torch.equal(gi, torch.zeros_like(x))


@pytest.mark.parametrize("offset", [30.0, 3000.0])
def test_mean_far_from_zero(cuda, offset):
    x, gy, w, b = inputs(3, (2, 64, 33, 20), torch.float32, torch.float32, cuda)
    x = x + offset
    ref = reference(x, gy, w, b, 8, "silu")
    y, mean, rstd = gna.group_norm_act_forward(x, 8, w, b, EPS, "silu")
    check_forward(y, ref, torch.float32)
    # the variance does not cancel: its error has no (mean / sd)^2 in it
    assert bool(((rstd.double() / ref["rstd"] - 1).abs() <= 16 * U32 * (1 + ref["ratio"])).all())
    check_backward(gna.group_norm_act_backward(gy, x, mean, rstd, 8, w, b, "silu"), ref,
                   torch.float32, torch.float32)


def test_single_huge_value_and_nonfinite_stay_in_their_group(cuda):
    x, _, w, b = inputs(4, (2, 32, 16, 16), torch.float32, torch.float32, cuda)
    x = x.clone(memory_format=torch.channels_last)
    x[0, 0, 0, 0] = 1e5
    ref = reference(x, None, w, b, 4, "none")
    y, mean, rstd = gna.group_norm_act_forward(x, 4, w, b)
    assert bool(((rstd.double() / ref["rstd"] - 1).abs() <= 32 * U32 * (1 + ref["ratio"])).all())
    x[0, 9, 3, 3] = float("nan")
    x[1, 31, 0, 0] = float("inf")
    y2, mean2, _ = gna.group_norm_act_forward(x, 4, w, b)
    bad = torch.zeros(2, 4, dtype=torch.bool, device=cuda)
    bad[0, 1] = bad[1, 3] = True
    grouped = y2.reshape(2, 4, -1)
    assert bool(grouped[bad].isnan().any(-1).all())
    assert torch.equal(grouped[~bad], y.reshape(2, 4, -1)[~bad])
    assert torch.equal(torch.isfinite(mean2), ~bad)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("c", [32, 21])
def test_squares_past_the_range_of_fp32(cuda, dt, c):
    """Deviations whose squares overflow: an infinite variance, so rstd is 0, the
    output is act(bias) and grad_input 0 -- what the formulas give in fp32."""
    x, gy, w, b = inputs(13, (1, c, 40, 30), dt, torch.float32, cuda)
    x = x * 1e25
    y, mean, rstd = gna.group_norm_act_forward(x, 1, w, b, EPS, "silu")
    assert not rstd.any() and bool(torch.isfinite(mean).all())
    want = torch.nn.functional.silu(b.double()).view(1, c, 1, 1).expand(y.shape)
    assert rel_l2(y, want) <= UNIT[dt] + 16 * U32
    gi, gw, gb = gna.group_norm_act_backward(gy, x, mean, rstd, 1, w, b, "silu")
    assert not gi.any() and not gw.any() and bool(torch.isfinite(gb).all())


@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
def test_layouts(cuda, dt):
    """Channels-last, a channel slice of a wider tensor (aligned or not), a crop,
    NCHW and an expanded gradient give the same result."""
    n, c, h, w_ = 2, 48, 9, 10
    x, gy, w, b = inputs(5, (n, c, h, w_), dt, torch.float32, cuda)
    want = gna.group_norm_act_forward(x, 6, w, b, EPS, "silu")
    gwant = gna.group_norm_act_backward(gy, x, want[1], want[2], 6, w, b, "silu")
    wide = torch.zeros(n, h, w_, 3 * c + 5, device=cuda, dtype=dt)
    big = torch.zeros(n, h + 3, w_ + 2, c, device=cuda, dtype=dt)
    views = []
    for at in (16, 7):
        t = wide.clone()
        t[..., at:at + c] = x.permute(0, 2, 3, 1)
        views.append(t[..., at:at + c].permute(0, 3, 1, 2))
    big[:, 1:1 + h, 2:2 + w_] = x.permute(0, 2, 3, 1)
    views.append(big[:, 1:1 + h, 2:2 + w_].permute(0, 3, 1, 2))
    views.append(x.contiguous())
    ref = reference(x, gy, w, b, 6, "silu")
    for v in views:
        assert torch.equal(v, x)
        got = gna.group_norm_act_forward(v, 6, w, b, EPS, "silu")
        check_forward(got[0], ref, dt)
        check_backward(gna.group_norm_act_backward(gy.contiguous(), v, got[1], got[2], 6, w, b,
                                                   "silu"), ref, dt, torch.float32)
    ones = torch.ones((), device=cuda, dtype=dt).expand(x.shape)
    a = gna.group_norm_act_backward(ones, x, want[1], want[2], 6, w, b, "silu")
    o = gna.group_norm_act_backward(torch.ones_like(x), x, want[1], want[2], 6, w, b, "silu")
    assert all(torch.equal(p, q) for p, q in zip(a, o))
    assert gwant[0].is_contiguous(memory_format=torch.channels_last)


def test_gradients_asked_for_alone(cuda):
    x, gy, w, b = inputs(6, (3, 32, 8, 8), torch.bfloat16, torch.float32, cuda)
    _, mean, rstd = gna.group_norm_act_forward(x, 4, w, b, EPS, "silu")
    full = gna.group_norm_act_backward(gy, x, mean, rstd, 4, w, b, "silu")
    for i in range(3):
        needs = [k == i for k in range(3)]
        part = gna.group_norm_act_backward(gy, x, mean, rstd, 4, w, b, "silu", needs)
        assert [t is not None for t in part] == needs and torch.equal(part[i], full[i])


def test_autograd_module_and_differences(cuda):
    m = gna.GroupNormAct(4, 32, act="silu").to(cuda)
    x, gy, w, b = inputs(7, (2, 32, 6, 5), torch.float32, torch.float32, cuda)
    with torch.no_grad():
        m.weight.copy_(w)
        m.bias.copy_(b)
    x = x.detach().requires_grad_()
    m(x).backward(gy)
    ref = reference(x, gy, w, b, 4, "silu")
    check_backward((x.grad, m.weight.grad, m.bias.grad), ref, torch.float32, torch.float32)
    # directional derivatives by central differences: error h^2 / 6 times a third
    # derivative of order 10 (about 2e-3 at h = 0.03), and fp32 noise u |L| / h
    g = torch.Generator(cuda).manual_seed(8)
    h = 0.03
    for name, t, grad in (("x", x, x.grad), ("w", m.weight, m.weight.grad), ("b", m.bias, m.bias.grad)):
        v = torch.randn(t.shape, generator=g, device=cuda)
        v /= v.square().mean().sqrt()
        with torch.no_grad():
            base = t.clone()
            t.copy_(base + h * v)
            up = (m(x).double() * gy.double()).sum()
            t.copy_(base - h * v)
            down = (m(x).double() * gy.double()).sum()
            t.copy_(base)
        slope = float((up - down) / (2 * h))
        want = float((grad.double() * v.double()).sum())
        assert abs(slope - want) <= 2e-2 * float(gy.norm()), name


def test_launches_that_fill_the_device_follow_each_other(cuda):
    """Each kernel's own limit of resident CTAs decides its launch, whatever ran before it."""
    for dt, c in ((torch.float32, 256), (torch.float32, 250), (torch.bfloat16, 256),
                  (torch.float16, 264), (torch.bfloat16, 255)):
        x, gy, w, b = inputs(12, (2, c, 150, 101), dt, torch.float32, cuda)
        groups = 1 if c % 8 else 8
        ref = reference(x, gy, w, b, groups, "silu")
        y, mean, rstd = gna.group_norm_act_forward(x, groups, w, b, EPS, "silu")
        check_forward(y, ref, dt)
        check_backward(gna.group_norm_act_backward(gy, x, mean, rstd, groups, w, b, "silu"), ref,
                       dt, torch.float32)


def test_waves_of_images(cuda):
    """More data than one wave: every image's statistics come from its own pixels."""
    shape = (14, 256, 70, 80)
    x, gy, w, b = inputs(9, shape, torch.float32, torch.float32, cuda)
    y, mean, rstd = gna.group_norm_act_forward(x, 32, w, b, EPS, "silu")
    ref = reference(x, gy, w, b, 32, "silu")
    check_forward(y, ref, torch.float32)
    check_backward(gna.group_norm_act_backward(gy, x, mean, rstd, 32, w, b, "silu"), ref,
                   torch.float32, torch.float32)


@pytest.mark.parametrize("shape", [(0, 16, 4, 4), (2, 16, 0, 4)])
def test_empty(cuda, shape):
    x = torch.zeros(shape, device=cuda)
    w = torch.ones(16, device=cuda)
    y, mean, rstd = gna.group_norm_act_forward(x, 4, w, w)
    assert y.shape == shape and mean.shape == (shape[0], 4)
    assert torch.equal(mean, torch.zeros_like(mean))
    gi, gw, gb = gna.group_norm_act_backward(x, x, mean, rstd, 4, w, w)
    assert gi.shape == shape and not gw.any() and not gb.any()


def test_repeats_bit_for_bit_and_on_another_stream(cuda):
    x, gy, w, b = inputs(10, (3, 64, 40, 30), torch.float16, torch.float16, cuda)
    one = gna.group_norm_act_forward(x, 8, w, b, EPS, "silu")
    g1 = gna.group_norm_act_backward(gy, x, one[1], one[2], 8, w, b, "silu")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        two = gna.group_norm_act_forward(x, 8, w, b, EPS, "silu")
        g2 = gna.group_norm_act_backward(gy, x, two[1], two[2], 8, w, b, "silu")
    s.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(one + tuple(g1), two + tuple(g2)))


def test_graph_capture(cuda):
    x, gy, w, b = inputs(11, (2, 64, 20, 30), torch.float16, torch.float16, cuda)
    want = gna.group_norm_act_forward(x, 8, w, b, EPS, "silu")
    gwant = gna.group_norm_act_backward(gy, x, want[1], want[2], 8, w, b, "silu")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = gna.group_norm_act_forward(x, 8, w, b, EPS, "silu")
        ggot = gna.group_norm_act_backward(gy, x, got[1], got[2], 8, w, b, "silu")
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want + tuple(gwant), got + tuple(ggot)))


def test_refusals(cuda):
    x = torch.randn(1, 8, 4, 4, device=cuda)
    w = torch.ones(8, device=cuda)
    with pytest.raises(RuntimeError, match="must divide"):
        gna.group_norm_act(x, 3)
    with pytest.raises(RuntimeError, match="dtype"):
        gna.group_norm_act(x.double(), 2)
    with pytest.raises(RuntimeError, match="parameter dtype"):
        gna.group_norm_act(x, 2, w.half(), w.half())
    with pytest.raises(RuntimeError, match="share a dtype"):
        gna.group_norm_act(x.half(), 2, w.half(), w)
    with pytest.raises(RuntimeError, match=r"\[C\]"):
        gna.group_norm_act(x, 2, torch.ones(7, device=cuda))
    with pytest.raises(RuntimeError, match="eps"):
        gna.group_norm_act(x, 2, eps=-1.0)
    with pytest.raises(ValueError, match="act"):
        gna.group_norm_act(x, 2, act="gelu")
    with pytest.raises(RuntimeError, match="is on cpu"):
        gna.group_norm_act(x, 2, w.cpu())
    y, mean, rstd = gna.group_norm_act_forward(x, 2)
    with pytest.raises(RuntimeError, match="grad_output"):
        gna.group_norm_act_backward(x[:, :4], x, mean, rstd, 2)
    with pytest.raises(RuntimeError, match="mean and rstd"):
        gna.group_norm_act_backward(x, x, mean.half(), rstd, 2)


SILU_Z = [-float("inf"), -3.3e38, -1e36, -1e20, -1000.0, -200.0, -100.0, -89.0, -88.1, -87.8, -87.5,
          -87.0, -80.0, -40.0, -20.0, -16.5, -10.0, -5.0, -2.5, -1.3, -0.7, -0.1, -1e-3, 0.0]
SILU_Z = SILU_Z + [-z for z in reversed(SILU_Z[2:])] + [0.5, 3.0]  # 48


@pytest.mark.parametrize("c", [48, 47], ids=["vectors", "elements"])
@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
def test_silu_at_every_argument(cuda, dt, c):
    """The activation's argument is the bias alone (weight 0).

    SiLU and its slope have their limits at minus infinity.  The sigmoid s is
    zero where it would be subnormal, and |z s| is below 88 * 2^-126 there: 2^-119.
    Else its relative error is that of e^-z (2^-22 of the exponential, |z| units
    of its rounded argument), which counts 1 - s times, and 6 units of the
    reciprocal and its step; the slope s (1 + z (1 - s)) has it 1 + |z| times at most.
    """
    z = torch.tensor(SILU_Z[:c], device=cuda)
    g = torch.Generator(cuda).manual_seed(21)
    x = torch.randn(2, 3, 5, c, generator=g, device=cuda).to(dt).permute(0, 3, 1, 2)
    gy = torch.randn(2, 3, 5, c, generator=g, device=cuda).to(dt).permute(0, 3, 1, 2)
    zero = torch.zeros(c, device=cuda)
    y, mean, rstd = gna.group_norm_act_forward(x, 1, zero, z, EPS, "silu")
    zd = z.double()
    s = torch.sigmoid(zd)
    want = torch.where(zd == -float("inf"), 0.0, zd * s)
    slope = torch.where(zd.isinf(), (zd > 0).double(), s * (1 + zd * (1 - s)))
    units = 6 + (4 + zd.abs().clamp_max(200)) * (1 - s)
    over = want.to(dt).isinf()                                   # +inf, or past the type's range
    row = y[0, :, 0, 0]
    assert torch.equal(y, row.view(1, c, 1, 1).expand(y.shape))
    assert bool((row[over] == float("inf")).all())
    lim = (units * U32 + UNIT[dt]) * want.abs() + 2.0 ** -119 + (2.0 ** -25 if dt == torch.float16 else 0)
    assert bool(((row.double() - want).abs() <= lim)[~over].all())
    gi, gw, gb = gna.group_norm_act_backward(gy, x, mean, rstd, 1, zero, z, "silu")
    assert not gi.any()
    total, mag = gy.double().sum((0, 2, 3)), gy.double().abs().sum((0, 2, 3))
    lim = (units * (1 + zd.abs().clamp_max(200)) * s + 64 * slope.abs()) * U32 * mag + 2.0 ** -119 * mag
    assert bool(((gb.double() - slope * total).abs() <= lim).all())
    assert bool(torch.isfinite(gw).all())


def test_silu_keeps_nan(cuda):
    for dt in DTYPES:
        x = torch.randn(1, 8, 4, 4, device=cuda).to(dt)
        b = torch.zeros(8, device=cuda)
        b[3] = float("nan")
        y, mean, rstd = gna.group_norm_act_forward(x, 8, None, b, EPS, "silu")
        assert bool(y[:, 3].isnan().all()) and int(y.isnan().sum()) == 16
        gi, _, gb = gna.group_norm_act_backward(torch.ones_like(x), x, mean, rstd, 8, None, b, "silu")
        assert bool(gi[:, 3].isnan().all()) and int(gi.isnan().sum()) == 16
        assert bool(gb[3].isnan()) and int(gb.isnan().sum()) == 1


@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
def test_silu_at_its_upper_end(cuda, dt):
    """Arguments whose product with log2(e) overflows, and infinity: the argument
    itself, with slope one where it is finite."""
    c = 8
    z = torch.tensor([2.3e38, 2.5e38, 3.3e38, float("inf"), 88.0, 1e30, 0.0, 1e5], device=cuda)
    g = torch.Generator(cuda).manual_seed(24)
    x = torch.randn(2, 3, 5, c, generator=g, device=cuda).to(dt).permute(0, 3, 1, 2)
    gy = torch.randn(2, 3, 5, c, generator=g, device=cuda).to(dt).permute(0, 3, 1, 2)
    zero = torch.zeros(c, device=cuda)
    y, mean, rstd = gna.group_norm_act_forward(x, 1, zero, z, EPS, "silu")
    assert torch.equal(y, z.to(dt).view(1, c, 1, 1).expand(y.shape))
    z[3] = 1e38
    gi, gw, gb = gna.group_norm_act_backward(gy, x, mean, rstd, 1, zero, z, "silu")
    assert not gi.any() and bool(torch.isfinite(gw).all())
    slope = torch.ones(c, dtype=torch.float64, device=cuda)
    slope[6] = 0.5
    lim = 64 * U32 * gy.double().abs().sum((0, 2, 3))
    assert bool(((gb.double() - slope * gy.double().sum((0, 2, 3))).abs() <= lim).all())


def test_the_16_bit_sigmoid_is_good_to_a_few_units(cuda):
    """grad_bias is an fp32 sum also for 16-bit tensors; with one nonzero
    gradient a channel it is the slope itself.  Error of the slope as in
    test_silu_at_every_argument; near zero that is 9 units of 2^-24."""
    c = 4096
    z = torch.linspace(-30, 30, c, device=cuda)
    for dt in (torch.float16, torch.bfloat16):
        x = torch.randn(1, c, 1, 2, generator=torch.Generator(cuda).manual_seed(22), device=cuda).to(dt)
        gy = torch.zeros_like(x)
        gy[..., 0] = 1
        zero = torch.zeros(c, device=cuda)
        _, mean, rstd = gna.group_norm_act_forward(x, 1, zero, z, EPS, "silu")
        _, _, gb = gna.group_norm_act_backward(gy, x, mean, rstd, 1, zero, z, "silu")
        zd = z.double()
        s = torch.sigmoid(zd)
        slope = s * (1 + zd * (1 - s))
        units = 6 + (4 + zd.abs()) * (1 - s)
        lim = (units * (1 + zd.abs()) * s + 3 * slope.abs()) * U32
        assert bool(((gb.double() - slope).abs() <= lim).all())


def test_offsets_past_31_bits(cuda):
    """2.2e9 elements in two images of a repeated block, whose statistics are the
    block's.  A thread's fp32 chains are some 15000 terms long here; rounding
    errors add up like a random walk, to about sqrt(15000) units: 512 allowed."""
    n, c, hw, part = 2, 64, 17_000_000, 1000
    g = torch.Generator(cuda).manual_seed(23)
    block = torch.randn(n, part, c, generator=g, device=cuda)
    block = (block + torch.tensor([0.0, 2.0], device=cuda).view(n, 1, 1)).bfloat16()
    x = torch.empty(n, hw, c, dtype=torch.bfloat16, device=cuda)
    x.view(n, hw // part, part, c).copy_(block[:, None].expand(n, hw // part, part, c))
    x, small = x.permute(0, 2, 1), block.permute(0, 2, 1)
    y, mean, rstd = gna.group_norm_act_forward(x, 8, act="silu")
    ref = reference(small, small, None, None, 8, "silu")
    assert bool(((mean.double() - ref["mean"]).abs() <= 512 * U32 * (1 + ref["mean"].abs())).all())
    assert bool(((rstd.double() / ref["rstd"] - 1).abs() <= 512 * U32).all())
    limit = UNIT[torch.bfloat16] + 512 * U32 * (1 + ref["ratio"])
    gi, _, _ = gna.group_norm_act_backward(x, x, mean, rstd, 8, act="silu")
    for t, want in ((y, ref["y"]), (gi, ref["dx"])):
        assert rel_l2(t[:, :, -part:], want) <= limit
        parts = t.permute(0, 2, 1).reshape(n, hw // part, part, c)
        assert bool((parts == parts[:, :1]).all())               # every repetition alike
