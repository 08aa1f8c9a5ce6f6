"""Embedding lookup with scaling and its gradient against 64-bit sums.

Tolerances.  A looked-up value is one fp32 product rounded to its type, so it
equals the same expression in torch.  A gradient row is an fp32 sum of its k
terms: first in order over at most 32, then over pieces in eight stretches, so
chains are at most 32 + k / 256 + 8 long (and never more than k): its error is
at most (32 + k / 256 + 10) u32 of the sum of magnitudes, plus the output
type's rounding of the value (u32 = 2^-24).
"""
import pytest
import torch

import scaled_embedding as emb

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
STEP = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
IDS = ["f32", "f16", "bf16"]


def expected(gy, ids, rows, scale, padding=None, old=None):
    """-> (gradient, sum of magnitudes, terms per row) in fp64."""
    ids, gy = ids.reshape(-1).long(), gy.double().reshape(-1, gy.shape[-1]) * scale
    ok = (ids >= 0) & (ids < rows)
    if padding is not None:
        ok &= ids != padding
    ids, gy = ids[ok], gy[ok]
    zero = torch.zeros(rows, gy.shape[1], dtype=torch.float64, device=gy.device)
    total, mag = zero.index_add(0, ids, gy), zero.index_add(0, ids, gy.abs())
    if old is not None:
        total, mag = total + old.double(), mag + old.double().abs()
    return total, mag, torch.bincount(ids, minlength=rows)


def check(got, want):
    total, mag, k = want
    chain = 42 + k.double()[:, None] / 256
    lim = chain * U32 * mag + UNIT[got.dtype] * total.abs() + STEP[got.dtype]
    assert got.shape == total.shape and bool(((got.double() - total).abs() <= lim).all())
    return got


def ids_of(kind, n, rows, device, seed=0):
    g = torch.Generator(device).manual_seed(seed)
    if kind == "uniform":
        return torch.randint(0, rows, (n,), generator=g, device=device)
    if kind == "skewed":
        u = torch.rand(n, generator=g, device=device)
        return ((rows + 1) ** u - 1).long().clamp_(0, rows - 1)
    if kind == "one":
        return torch.full((n,), rows - 1, device=device)
    if kind == "grid":
        return torch.arange(n, device=device) % rows
    if kind == "blocks":
        return torch.arange(n, device=device) * rows // max(n, 1)
    if kind == "wild":                                     # a third names no row
        return torch.randint(-rows, 2 * rows, (n,), generator=g, device=device)
    raise KeyError(kind)


CASES = [  # n, rows, dim, ids
    (1, 1, 8, "uniform"),
    (1, 70000, 4, "uniform"),
    (31, 5, 16, "uniform"),
    (32, 1, 24, "one"),
    (33, 3, 32, "one"),
    (64, 2, 8, "blocks"),
    (1000, 255, 40, "skewed"),
    (1000, 256, 256, "skewed"),        # the key of what names no row needs another digit
    (4097, 257, 64, "uniform"),        # two CTAs sort
    (5000, 70000, 33, "uniform"),      # rows of no 16-byte multiple; three digits
    (9000, 1000, 72, "wild"),
    (20000, 200, 128, "grid"),
    (40000, 200, 16, "blocks"),
    (33000, 65535, 264, "skewed"),
    (66000, 50000, 8, "skewed"),       # sixteen CTAs, more than 4096 tokens each
    (70000, 17000000, 1, "uniform"),   # four digits, one column
    (30000, 7, 520, "one"),            # one run over all tiles
]


@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
@pytest.mark.parametrize("n,rows,dim,kind", CASES, ids=[f"{a}-{b}-{c}-{d}" for a, b, c, d in CASES])
def test_matches_sums(cuda, n, rows, dim, kind, dt):
    g = torch.Generator(cuda).manual_seed(1)
    ids = ids_of(kind, n, rows, cuda)
    table = torch.randn(rows, dim, generator=g, device=cuda).to(dt)
    gy = torch.randn(n, dim, generator=g, device=cuda).to(dt)
    y = emb.scaled_embedding_forward(table, ids, 1.7)
    ok = (ids >= 0) & (ids < rows)
    scale = torch.tensor(1.7, device=cuda)                # fp32, as the kernel has it
    want = (table[ids.clamp(0, rows - 1)].float() * scale).to(dt)
    assert torch.equal(y, torch.where(ok[:, None], want, torch.zeros_like(want)))
    check(emb.scaled_embedding_backward(gy, ids, rows, 1.7), expected(gy, ids, rows, float(scale)))
    # added to an fp32 gradient, with one row left out
    main = torch.randn(rows, dim, generator=g, device=cuda)
    old, pad = main.clone(), int(ids[0].clamp(0, rows - 1))
    got = emb.scaled_embedding_backward(gy, ids.int(), rows, 1.7, padding_idx=pad, grad_weight=main)
    assert got.data_ptr() == main.data_ptr()
    want = expected(gy, ids, rows, float(scale), pad, old)
    check(main, want)
    untouched = want[2] == 0
    assert torch.equal(main[untouched], old[untouched]) and bool(untouched[pad])


def test_more_tokens_than_a_cluster_holds_at_once(cuda):
    n, rows = 300_001, 1000
    g = torch.Generator(cuda).manual_seed(2)
    ids = ids_of("skewed", n, rows, cuda)
    gy = torch.randn(n, 24, generator=g, device=cuda)
    check(emb.scaled_embedding_backward(gy, ids, rows), expected(gy, ids, rows, 1.0))


@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
def test_strides_and_alignment(cuda, dt):
    g = torch.Generator(cuda).manual_seed(3)
    n, rows, dim = 700, 90, 48
    ids = ids_of("skewed", n, rows, cuda).view(7, 100)
    wide = torch.randn(rows, 3 * dim + 1, generator=g, device=cuda).to(dt)
    gwide = torch.randn(n, 2 * dim + 8, generator=g, device=cuda).to(dt)
    for at in (0, 8, 1):
        table, gy = wide[:, at:at + dim], gwide[:, at:at + dim]
        y = emb.scaled_embedding_forward(table, ids)
        assert y.shape == (7, 100, dim) and torch.equal(y, table[ids])
        grad = emb.scaled_embedding_backward(gy, ids.view(-1), rows)
        check(grad, expected(gy, ids, rows, 1.0))
        dest = torch.zeros(rows, dim + 5, device=cuda)
        into = dest[:, :dim] if at == 0 else dest[:, at % 5:at % 5 + dim]
        emb.scaled_embedding_backward(gy, ids.view(-1), rows, grad_weight=into)
        check(into, expected(gy, ids, rows, 1.0))
        assert float(dest.double().sum()) == pytest.approx(float(into.double().sum()), abs=1e-9)
    # gradients of any layout: transposed, expanded (the gradient of a sum)
    t = torch.randn(dim, n, generator=g, device=cuda).to(dt).t()
    check(emb.scaled_embedding_backward(t, ids.view(-1), rows), expected(t, ids, rows, 1.0))
    ones = torch.ones((), device=cuda, dtype=dt).expand(7, 100, dim)
    check(emb.scaled_embedding_backward(ones, ids, rows), expected(ones, ids, rows, 1.0))
    assert torch.equal(emb.scaled_embedding_forward(wide.t()[:dim], ids % dim), wide.t()[:dim][ids % dim])
    noncontiguous = ids.t()
    assert torch.equal(emb.scaled_embedding_forward(wide, noncontiguous), wide[noncontiguous])


@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
def test_nonfinite_values_stay_in_their_rows(cuda, dt):
    ids = ids_of("grid", 500, 10, cuda)
    gy = torch.ones(500, 16, device=cuda, dtype=dt)
    gy[3, 5] = float("nan")
    gy[7, 2] = float("inf")
    grad = emb.scaled_embedding_backward(gy, ids, 12)
    bad = ~torch.isfinite(grad)
    assert int(bad.sum()) == 2 and bool(bad[3, 5]) and bool(bad[7, 2])
    assert not grad[10:].any()
    table = torch.full((3, 8), float("nan"), device=cuda, dtype=dt)
    y = emb.scaled_embedding_forward(table, torch.tensor([-1, 3, 1 << 40], device=cuda))
    assert torch.equal(y, torch.zeros_like(y))            # rows that do not exist are not read


def test_empty(cuda):
    none = torch.zeros(0, dtype=torch.int64, device=cuda)
    table = torch.ones(5, 8, device=cuda)
    assert emb.scaled_embedding_forward(table, none).shape == (0, 8)
    assert emb.scaled_embedding_forward(table, none.view(3, 0)).shape == (3, 0, 8)
    grad = emb.scaled_embedding_backward(torch.zeros(0, 8, device=cuda), none, 5)
    assert grad.shape == (5, 8) and not grad.any()
    main = torch.ones(5, 8, device=cuda)
    emb.scaled_embedding_backward(torch.zeros(0, 8, device=cuda), none, 5, grad_weight=main)
    assert bool((main == 1).all())
    ids = torch.zeros(4, dtype=torch.int64, device=cuda)
    y = emb.scaled_embedding_forward(torch.zeros(0, 8, device=cuda), ids)
    assert y.shape == (4, 8) and not y.any()
    assert emb.scaled_embedding_backward(torch.ones(4, 8, device=cuda), ids, 0).shape == (0, 8)
    grad = emb.scaled_embedding_backward(torch.ones(4, 8, device=cuda), ids - 1, 3)
    assert not grad.any()                                 # no id names a row


def test_offsets_past_31_bits(cuda):
    rows, dim = 1_100_000, 2048                           # 2.25e9 elements of bf16
    ids = torch.tensor([rows - 1, 0, rows - 1, 1_050_000], device=cuda)
    table = torch.zeros(rows, dim, dtype=torch.bfloat16, device=cuda)
    table[rows - 1] = 3.0
    y = emb.scaled_embedding_forward(table, ids, 2.0)
    assert bool((y[0] == 6).all()) and bool((y[2] == 6).all()) and not y[1].any()
    gy = torch.ones(4, dim, dtype=torch.bfloat16, device=cuda)
    emb.scaled_embedding_backward(gy, ids, rows, 0.5, grad_weight=table)
    assert bool((table[rows - 1] == 4).all()) and bool((table[0] == 0.5).all())
    assert bool((table[1_050_000] == 0.5).all()) and float(table[1:1000].double().sum()) == 0.0


def test_module_autograd_and_differences(cuda):
    torch.manual_seed(4)
    m = emb.ScaledEmbedding(50, 24, padding_idx=-50, scale=24 ** 0.5).to(cuda)
    ids = ids_of("skewed", 600, 50, cuda).view(20, 30)
    g = torch.Generator(cuda).manual_seed(5)
    gy = torch.randn(20, 30, 24, generator=g, device=cuda)
    m(ids).backward(gy)
    check(m.weight.grad, expected(gy, ids, 50, m.scale, 0))
    assert not m.weight.grad[0].any()
    # the lookup is linear in the table: a difference of any width is exact but for rounding
    v = torch.randn(50, 24, generator=g, device=cuda)
    v[0] = 0
    with torch.no_grad():
        up = (emb.scaled_embedding(ids, m.weight + v, m.scale).double() * gy.double()).sum()
        down = (emb.scaled_embedding(ids, m.weight - v, m.scale).double() * gy.double()).sum()
    want = (m.weight.grad.double() * v.double()).sum()
    # 14400 products, each with a few roundings of 2^-24 of magnitude 15 or less
    assert abs(float((up - down) / 2 - want)) <= 14400 * 15 * 4 * U32


def test_repeats_bit_for_bit_streams_and_graph(cuda):
    g = torch.Generator(cuda).manual_seed(6)
    ids = ids_of("skewed", 30000, 3000, cuda)
    gy = torch.randn(30000, 136, generator=g, device=cuda).half()
    want = emb.scaled_embedding_backward(gy, ids, 3000)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(3):
            again = emb.scaled_embedding_backward(gy, ids, 3000)
    s.synchronize()
    assert torch.equal(again, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = emb.scaled_embedding_backward(gy, ids, 3000)
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_refusals(cuda):
    w = torch.randn(5, 8, device=cuda)
    ids = torch.zeros(3, dtype=torch.int64, device=cuda)
    gy = torch.zeros(3, 8, device=cuda)
    with pytest.raises(RuntimeError, match="int64 or int32"):
        emb.scaled_embedding_forward(w, ids.float())
    with pytest.raises(RuntimeError, match="dtype"):
        emb.scaled_embedding_forward(w.double(), ids)
    with pytest.raises(RuntimeError, match=r"\[rows, dim\]"):
        emb.scaled_embedding_forward(w.view(-1), ids)
    with pytest.raises(RuntimeError, match="is on cpu"):
        emb.scaled_embedding_forward(w, ids.cpu())
    with pytest.raises(ValueError, match="padding_idx"):
        emb.scaled_embedding_backward(gy, ids, 5, padding_idx=5)
    with pytest.raises(RuntimeError, match="grad_output must be"):
        emb.scaled_embedding_backward(gy[:2], ids, 5)
    with pytest.raises(RuntimeError, match="grad_weight"):
        emb.scaled_embedding_backward(gy, ids, 5, grad_weight=torch.zeros(4, 8, device=cuda))
    with pytest.raises(RuntimeError, match="rows must be"):
        emb.scaled_embedding_backward(gy, ids, 5, grad_weight=torch.zeros(8, 5, device=cuda).t())
    with pytest.raises(RuntimeError, match="dtypes"):
        emb.scaled_embedding_backward(gy, ids, 5, grad_weight=w.half())


@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,dim", [(7, 3), (1000, 5), (12450, 37), (1, 1), (333, 2049)])
def test_zeros_of_odd_tables(cuda, rows, dim, dt):
    """Rows that no id names are zero, whatever the table's size in bytes, and
    nothing is written beside the table."""
    ids = torch.tensor([0], device=cuda)
    gy = torch.ones(1, dim, device=cuda, dtype=dt)
    for _ in range(2):
        torch.full((rows * dim + 4096,), float("nan"), device=cuda, dtype=dt)  # what the memory may hold
        grad = emb.scaled_embedding_backward(gy, ids, rows)
        assert bool((grad[0] == 1).all()) and not grad[1:].any()


def test_dense_gradient_into_a_wider_buffer(cuda):
    """The C ABI's row stride: zeros go to the rows only."""
    import ctypes

    from bevk import cabi
    L = cabi.lib()
    for dim, ld, at in ((24, 40, 0), (24, 25, 0), (23, 40, 1)):
        buf = torch.full((50 * ld + at,), 7.0, device=cuda)
        ids = torch.tensor([3, 3, 49], device=cuda)
        gy = torch.ones(3, dim, device=cuda)
        a = cabi.EmbeddingBackwardArgs()
        a.num_ids, a.num_rows, a.dim, a.ids_are_64bit = 3, 50, dim, 1
        a.grad_output_ld, a.grad_table_ld, a.padding_idx, a.scale = dim, ld, -1, 1.0
        n = L.bevk_embedding_backward_workspace_bytes(ctypes.byref(a))
        ws = torch.empty(n, dtype=torch.uint8, device=cuda)
        cabi.check(L.bevk_embedding_backward(
            ctypes.byref(a), gy.data_ptr(), ids.data_ptr(), buf.data_ptr() + 4 * at, ws.data_ptr(), n,
            torch.cuda.current_stream().cuda_stream), "embedding_backward")
        rows = buf[at:].view(50, ld)
        assert bool((rows[:, dim:] == 7).all()) and bool((buf[:at] == 7).all())
        want = torch.zeros(50, dim, device=cuda)
        want[3], want[49] = 2, 1
        assert torch.equal(rows[:, :dim], want)


def abi_backward(gy, ids, grad_table, rows, dim, ld, accumulate=0, at=0, scale=1.0):
    """The C ABI with grad_table's first element `at` elements into the buffer."""
    import ctypes

    from bevk import cabi
    L, code = cabi.lib(), {torch.float32: cabi.DTYPE_F32, torch.float16: cabi.DTYPE_F16,
                           torch.bfloat16: cabi.DTYPE_BF16}
    a = cabi.EmbeddingBackwardArgs()
    a.num_ids, a.num_rows, a.dim, a.ids_are_64bit = ids.numel(), rows, dim, 1
    a.grad_output_ld, a.grad_table_ld, a.padding_idx, a.scale = dim, ld, -1, scale
    a.grad_output_dtype, a.grad_table_dtype = code[gy.dtype], code[grad_table.dtype]
    a.accumulate = accumulate
    n = L.bevk_embedding_backward_workspace_bytes(ctypes.byref(a))
    ws = torch.empty(n, dtype=torch.uint8, device=gy.device)
    cabi.check(L.bevk_embedding_backward(
        ctypes.byref(a), gy.data_ptr(), ids.data_ptr(),
        grad_table.data_ptr() + at * grad_table.element_size(), ws.data_ptr(), n,
        torch.cuda.current_stream().cuda_stream), "embedding_backward")


@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
def test_adding_keeps_subnormals_and_rounds_alike_at_any_alignment(cuda, dt):
    """old + scale * (the row's sum), rounded once: whichever width the rows are
    taken in, and below the smallest normal number too."""
    g = torch.Generator(cuda).manual_seed(11)
    rows, dim, n = 60, 32, 500
    ids = ids_of("skewed", n, rows, cuda)
    gy = torch.randn(n, dim, generator=g, device=cuda).to(dt)
    old = torch.randn(rows, dim, generator=g, device=cuda)
    got = []
    for ld, at in ((dim, 0), (dim + 1, 0), (dim, 1), (dim + 4, 4)):
        buf = torch.zeros(rows * ld + at, device=cuda)
        view = buf[at:].view(rows, ld)[:, :dim]
        view.copy_(old)
        abi_backward(gy, ids, buf, rows, dim, ld, accumulate=1, at=at, scale=1.7)
        got.append(view.clone())
    assert all(torch.equal(t, got[0]) for t in got[1:])
    # a named row's subnormal elements, and sums that are subnormal or become so
    main = torch.full((4, dim), 3e-40, device=cuda)
    gy = torch.zeros(3, dim, device=cuda)
    gy[1] = 5e-41
    gy[2] = 1.0
    kept = main.clone()
    emb.scaled_embedding_backward(gy, torch.tensor([0, 1, 2], device=cuda), 4, 2.0 ** -130,
                                  grad_weight=main)
    want = kept.double()
    want[1] += 2.0 ** -130 * gy[1].double()
    want[2] += 2.0 ** -130
    assert torch.equal(main, want.float())


@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,dim", [(5, 8), (40, 33), (900, 64), (5000, 136), (60000, 24)])
def test_zeros_stay_inside_the_table(cuda, rows, dim, dt):
    """Tables below and above the size whose zeros get a kernel of their own, at
    any element offset, back to back and with gaps between the rows."""
    gy = torch.ones(2, dim, device=cuda, dtype=dt)
    ids = torch.tensor([rows - 1, 1], device=cuda)
    for ld in (dim, dim + 8, dim + 3):
        for at in (0, 1, 3, 7):
            buf = torch.full((at + rows * ld + 40,), 7.0, device=cuda, dtype=dt)
            abi_backward(gy, ids, buf, rows, dim, ld, at=at)
            table = buf[at:at + rows * ld].view(rows, ld)
            assert bool((buf[:at] == 7).all()) and bool((buf[at + rows * ld:] == 7).all())
            assert bool((table[:, dim:] == 7).all())
            want = torch.zeros(rows, dim, device=cuda, dtype=dt)
            want[rows - 1] = want[1] = 1
            assert torch.equal(table[:, :dim], want)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("n,rows,dim,kind", [(1000, 255, 40, "skewed"), (5000, 3000, 33, "uniform"),
                                             (30000, 7, 520, "one"), (37, 50, 6, "uniform")])
def test_added_to_a_16_bit_gradient(cuda, n, rows, dim, kind, dt):
    g = torch.Generator(cuda).manual_seed(12)
    ids = ids_of(kind, n, rows, cuda)
    gy = torch.randn(n, dim, generator=g, device=cuda).to(dt)
    main = torch.randn(rows, dim, generator=g, device=cuda).to(dt)
    old = main.clone()
    emb.scaled_embedding_backward(gy, ids, rows, 0.5, grad_weight=main)
    want = expected(gy, ids, rows, 0.5, None, old)
    check(main, want)
    assert torch.equal(main[want[2] == 0], old[want[2] == 0])
