"""Global gradient norm and clipping against 64-bit arithmetic.

Tolerances.  The squares are summed in fp32 in chains of at most 64 / 4 terms,
then in fp64: the norm's relative error is at most about 16 u32 (u32 = 2^-24).
c = max_norm / (norm + eps) carries that and two roundings, and an output one
more of its own type: 32 u32 + u_type of the value, and half a subnormal step.
"""
import math

import pytest
import torch

import grad_clip
from bevk import cabi

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
STEP = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def make(seed, sizes, dtypes, device, std=0.02):
    g = torch.Generator(device).manual_seed(seed)
    return [(torch.randn(s, generator=g, device=device) * std).to(dtypes[i % len(dtypes)])
            for i, s in enumerate(sizes)]


def want_norm(grads, inf=False):
    flat = torch.cat([g.detach().double().reshape(-1) for g in grads])
    return float(flat.abs().max()) if inf else float(flat.square().sum().sqrt())


def check(norm, outs, grads, max_norm, inf=False):
    ref = want_norm(grads, inf)
    assert norm.dtype == torch.float32 and norm.dim() == 0
    assert abs(float(norm) - ref) <= 16 * U32 * ref
    c = min(1.0, max_norm / (ref + grad_clip.CLIP_EPS))
    for o, g in zip(outs, grads):
        e = g.double() * c
        lim = (32 * U32 + UNIT[o.dtype]) * e.abs() + STEP[o.dtype]
        assert o.shape == g.shape and bool(((o.double() - e).abs() <= lim).all())


SIZES = {
    "one": [1],
    "few": [3, 1000, 17, 64 * 64, 1, 5, 100_003],
    "matrices": [(64, 33), (7,), (128, 3, 3, 3), (1,), (2048, 511)],
    "empty among": [0, 12, 0, 2050, 0],
    "hundreds": [1 + 37 * i % 5000 for i in range(350)],
    "thousands": [1 + 31 * i % 400 for i in range(2300)],
    "tiles": [2048, 2047, 2049, 4096, 8 * 2048 + 1],
}


@pytest.mark.parametrize("inf", [False, True], ids=["l2", "inf"])
@pytest.mark.parametrize("name", SIZES)
def test_norm_and_scaling(cuda, name, inf):
    grads = make(1, SIZES[name], DTYPES, cuda)
    kind = math.inf if inf else 2.0
    ref = want_norm(grads, inf)
    assert abs(float(grad_clip.grad_norm(grads, kind)) - ref) <= 16 * U32 * ref
    before = [g.clone() for g in grads]
    out = [torch.empty_like(g, dtype=torch.float32) for g in grads]
    norm = grad_clip.clip_grads(grads, 0.4 * ref, kind, out=out)
    check(norm, out, grads, 0.4 * ref, inf)
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    norm = grad_clip.clip_grads(grads, 0.4 * ref, kind)          # in place
    check(norm, grads, before, 0.4 * ref, inf)


@pytest.mark.parametrize("odt", DTYPES, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("gdt", DTYPES, ids=["f32", "f16", "bf16"])
def test_types_and_alignment(cuda, gdt, odt):
    """Every pair of types, with gradients and outputs at any element offset."""
    sizes = [1, 7, 8, 9, 513, 4100, 65537]
    for gat in (0, 1, 3, 8):
        for oat in (0, 1, 6):
            gbuf = make(2, [sum(sizes) + gat], [gdt], cuda)[0]
            obuf = torch.full((sum(sizes) + oat,), 7.0, dtype=odt, device=cuda)
            grads, out, a = [], [], 0
            for s in sizes:
                grads.append(gbuf[gat + a:gat + a + s])
                out.append(obuf[oat + a:oat + a + s])
                a += s
            ref = want_norm(grads)
            check(grad_clip.clip_grads(grads, 0.25 * ref, out=out), out, grads, 0.25 * ref)
            assert bool((obuf[:oat] == 7.0).all())


@pytest.mark.parametrize("dt", DTYPES, ids=["f32", "f16", "bf16"])
def test_within_the_limit_nothing_changes(cuda, dt):
    grads = make(3, [1001, 64, 5], [dt], cuda)
    before = [g.clone() for g in grads]
    ref = want_norm(grads)
    norm = grad_clip.clip_grads(grads, 2 * ref)
    check(norm, grads, before, 2 * ref)
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    out = [torch.zeros_like(g) for g in grads]
    grad_clip.clip_grads(grads, 2 * ref, out=out)
    assert all(torch.equal(a, b) for a, b in zip(out, before))
    grad_clip.clip_grads(grads, 0.0)                             # a limit of zero
    assert not any(g.any() for g in grads)


@pytest.mark.parametrize("inf", [False, True], ids=["l2", "inf"])
def test_nan_and_infinity(cuda, inf):
    kind = math.inf if inf else 2.0
    for tensor, at in ((0, 0), (1, 4999), (2, 0)):
        grads = make(4, [40_000, 5000, 1], [torch.float32, torch.float16], cuda)
        grads[tensor][at] = float("nan")
        assert math.isnan(float(grad_clip.clip_grads(grads, 1.0, kind)))
        assert all(bool(g.isnan().all()) for g in grads)
        grads = make(4, [40_000, 5000, 1], [torch.float32, torch.float16], cuda)
        grads[tensor][at] = -float("inf")
        assert float(grad_clip.clip_grads(grads, 1.0, kind)) == math.inf
        bad = grads[tensor].isnan()
        assert int(bad.sum()) == 1 and bool(bad[at])
        assert sum(int(g.count_nonzero()) for g in grads) == 1    # the NaN; the rest is zero
    zeros = [torch.zeros(100, device=cuda)]
    assert float(grad_clip.clip_grads(zeros, 1.0, kind)) == 0.0 and not zeros[0].any()


def test_layouts(cuda):
    """Dense permuted tensors in place; tensors with holes through a copy."""
    g = torch.Generator(cuda).manual_seed(5)
    wide = torch.randn(64, 50, generator=g, device=cuda)
    nhwc = torch.randn(16, 3, 3, 8, generator=g, device=cuda).permute(0, 3, 1, 2)
    grads = [wide[:, 3:20], nhwc, wide.t()[30:33].contiguous().t(), wide[5, 40:]]
    rest = wide.clone()
    before = [t.clone() for t in grads]
    ref = want_norm(before)
    check(grad_clip.clip_grads(grads, 0.3 * ref), grads, before, 0.3 * ref)
    keep = torch.ones_like(wide, dtype=torch.bool)
    keep[:, 3:20] = False
    keep[5, 40:] = False
    assert torch.equal(wide[keep], rest[keep])                   # what lies between is not written
    grads = [b.clone(memory_format=torch.preserve_format) for b in before]
    out = [torch.zeros_like(t, memory_format=torch.contiguous_format) for t in grads]
    check(grad_clip.clip_grads(grads, 0.3 * ref, out=out), out, before, 0.3 * ref)


def test_offsets_past_31_bits(cuda):
    n = (1 << 31) + 4099
    g = torch.zeros(n, dtype=torch.bfloat16, device=cuda)
    g[0] = 3.0
    g[-1] = 4.0
    assert float(grad_clip.clip_grads([g], 2.5)) == 5.0
    assert float(g[0]) == 1.5 and float(g[-1]) == 2.0 and float(g.double().sum()) == 3.5


def test_large_values(cuda):
    g = torch.full((1000,), 1e18, device=cuda)
    ref = 1e18 * math.sqrt(1000)
    assert abs(float(grad_clip.grad_norm([g])) - ref) <= 1e-6 * ref
    assert float(grad_clip.grad_norm([g], math.inf)) == pytest.approx(1e18, rel=1e-6)


def test_parameters_and_streams(cuda):
    torch.manual_seed(6)
    m = torch.nn.Sequential(torch.nn.Linear(64, 128), torch.nn.GELU(), torch.nn.Linear(128, 3))
    m = m.to(cuda)
    m.register_parameter("unused", torch.nn.Parameter(torch.zeros(3, device=cuda)))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        m(torch.randn(32, 64, device=cuda)).square().sum().backward()
        grads = [p.grad for p in m.parameters() if p.grad is not None]
        before = [g.clone() for g in grads]
        norm = grad_clip.clip_grad_norm_(m.parameters(), 0.5)
        check(norm, grads, before, 0.5)
        one = grad_clip.clip_grad_norm_(m[0].weight, 1e9)
        assert float(one) == pytest.approx(float(m[0].weight.grad.norm()), rel=1e-5)
    s.synchronize()
    assert m.unused.grad is None
    m[0].weight.grad[0, 0] = float("nan")
    kept = m[2].weight.grad.clone()
    with pytest.raises(RuntimeError, match="not finite"):
        grad_clip.clip_grad_norm_(m.parameters(), 0.5, error_if_nonfinite=True)
    assert torch.equal(m[2].weight.grad, kept)


def test_repeats_bit_for_bit_and_graph_capture(cuda):
    grads = make(7, SIZES["hundreds"], [torch.bfloat16], cuda)
    out = [torch.empty_like(g, dtype=torch.float32) for g in grads]
    norm = grad_clip.clip_grads(grads, 1.0, out=out)
    want = [o.clone() for o in out]
    for o in out:
        o.zero_()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = grad_clip.clip_grads(grads, 1.0, out=out)
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(norm, again) and all(torch.equal(a, b) for a, b in zip(out, want))


def test_refusals(cuda):
    g = torch.randn(100, device=cuda)
    with pytest.raises(RuntimeError, match="overlaps"):
        grad_clip.clip_grads([g, g], 1.0)
    with pytest.raises(RuntimeError, match="overlaps"):
        grad_clip.clip_grads([g[:60], g[50:]], 1.0)
    with pytest.raises(RuntimeError, match="overlaps"):
        grad_clip.clip_grads([g[:50], g[50:]], 1.0, out=[g[50:], torch.empty(50, device=cuda)])
    with pytest.raises(RuntimeError, match="overlaps"):
        o = torch.empty(60, device=cuda)
        grad_clip.clip_grads([g[:50], g[50:]], 1.0, out=[o[:50], o[10:]])
    assert float(grad_clip.grad_norm([g, g])) == pytest.approx(math.sqrt(2) * float(g.norm()), rel=1e-5)
    with pytest.raises(RuntimeError, match="expanded"):
        grad_clip.clip_grads([torch.ones((), device=cuda).expand(5)], 1.0)
    with pytest.raises(RuntimeError, match="shape"):
        grad_clip.clip_grads([g], 1.0, out=[g[:50]])
    with pytest.raises(RuntimeError, match="one output"):
        grad_clip.clip_grads([g], 1.0, out=[])
    with pytest.raises(RuntimeError, match="max_norm"):
        grad_clip.clip_grads([g], -1.0)
    with pytest.raises(RuntimeError, match="max_norm"):
        grad_clip.clip_grads([g], float("nan"))
    with pytest.raises(RuntimeError, match="dtype"):
        grad_clip.clip_grads([g.double()], 1.0)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        grad_clip.clip_grads([g, g.cpu()], 1.0)
    with pytest.raises(ValueError, match="norm_type"):
        grad_clip.grad_norm([g], 1.0)
    with pytest.raises(RuntimeError, match="no gradients"):
        grad_clip.grad_norm([])


def test_c_abi_checks_before_any_launch(cuda):
    L = cabi.lib()
    t = (cabi.GradTensor * 1)()
    t[0].grad, t[0].out, t[0].numel = 6, 6, 4                    # not aligned to fp32
    assert L.bevk_grad_clip(t, 1, 0, 1.0, 1e-6, 1, 16, 16, 1 << 20, None) == cabi.ERR_MISALIGNED


@pytest.mark.parametrize("n", [37, 5000, 10_000_000])
@pytest.mark.parametrize("size", [1e37, 5e18, 1e10, 1e-10, 1e-19, 1e-24, 1e-30, 1e-38])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_norms_over_the_range_of_fp32(cuda, dt, size, n):
    """Only the norm itself has to fit fp32, not the squares or their sums."""
    if size * n ** 0.5 > 1e38:
        n = 50
    g = torch.Generator(cuda).manual_seed(8)
    # the same magnitudes in every thread's share, within a factor of two
    flat = ((0.5 + torch.rand(n, generator=g, device=cuda)) * size).to(dt)
    flat *= torch.where(torch.rand(n, generator=g, device=cuda) < 0.5, -1.0, 1.0).to(dt)
    grads = [flat[:1], flat[1:4], flat[4:]]
    before = [t.clone() for t in grads]
    ref = want_norm(grads)
    assert abs(float(grad_clip.grad_norm(grads)) - ref) <= 16 * U32 * ref + 2.0 ** -149
    check(grad_clip.clip_grads(grads, 0.5 * ref), grads, before, 0.5 * ref)


def test_small_and_large_among_others(cuda):
    g = torch.full((10_000_000,), 1e-30, device=cuda)
    zeros = torch.zeros(1_000_000, device=cuda)
    zeros[::2] = -0.0
    for at, v in ((5, 1e-3), (9_999_999, -1e25), (4_000_001, 1e-20)):
        t = g.clone()
        t[at] = v
        ref = want_norm([t])
        assert abs(float(grad_clip.grad_norm([zeros, t])) - ref) <= 16 * U32 * ref
    assert float(grad_clip.grad_norm([zeros])) == 0.0
    # a norm past fp32's range is infinite and scales by zero
    t = torch.full((2,), 3e38, device=cuda)
    assert float(grad_clip.clip_grads([t], 1.0)) == math.inf and not t.any()
