"""Token tables on the GPU against their definitions in 64 bits.

Tolerances count roundings.  U is half a step of a type relative to the value; sums in fp32 of terms t are off by at most
(number of additions that a term passes through) * 2^-24 * sum |t|, whatever their order.
"""
import itertools

import numpy as np
import pytest
import torch

import oracle as O
from fbgemm_ascend_b200.types import SparseType, group_row_bytes

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}     # half a step below the normal numbers
CODE = {torch.float32: int(SparseType.FP32), torch.float16: int(SparseType.FP16), torch.bfloat16: int(SparseType.BF16)}
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def ops():
    import fbgemm_ascend_b200  # noqa: F401
    return torch.ops.tbe_b200


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=F32, std=1.0):
    return (torch.randn(*shape, device="cuda", generator=g) * std).to(dtype)


def within(got, want, bound):
    """|got - want| <= bound, element by element; all in 64 bits."""
    got, want = got.double(), want.double()
    assert got.shape == want.shape
    bad = ~((got - want).abs() <= bound)
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} beyond the bound; worst {float(((got - want).abs() / bound).nan_to_num(posinf=1e9).max()):.3g} of it"


def tokens_of(g, n, V, kind, dtype):
    if kind == "uniform":
        t = torch.randint(0, V, (n,), device="cuda", generator=g)
    elif kind == "same":
        t = torch.full((n,), V // 2, device="cuda")
    elif kind == "spread":
        t = torch.arange(n, device="cuda").mul(V // max(n, 1) if n <= V else 1).remainder(V).flip(0)
    elif kind == "hot":
        t = torch.randint(0, V, (n,), device="cuda", generator=g)
        t[torch.rand(n, device="cuda", generator=g) < 0.6] = V - 1
    elif kind == "few":
        t = torch.randint(0, min(V, 3), (n,), device="cuda", generator=g)
    elif kind == "none":
        t = torch.full((n,), -1, device="cuda")
    else:      # "wild": pruned ones and numbers outside the table
        t = torch.randint(-2, V + 2, (n,), device="cuda", generator=g)
        t[::5] = -1
        if n > 3:
            t[3] = torch.iinfo(dtype).max
            t[1] = torch.iinfo(dtype).min
    return t.to(dtype)


# ---- lookup -------------------------------------------------------------------------------------------------------

def lookup64(weight, tokens, scale):
    V = weight.shape[0]
    t = tokens.long().reshape(-1)
    met = (t >= 0) & (t < V)
    out = torch.zeros(t.numel(), weight.shape[1], dtype=torch.float64, device=weight.device)
    out[met] = weight[t[met]].double() * float(np.float32(scale))
    return out.view(*tokens.shape, weight.shape[1])


def lookup_bound(want, dtype):
    """One product rounded to fp32, then to the result's type."""
    return want.abs() * (U[dtype] + 2.0 ** -24 * (1 + U[dtype])) + TINY[dtype] + 2.0 ** -150


@pytest.mark.parametrize("ti,to", list(itertools.product((F32, F16, BF16), repeat=2)))
@pytest.mark.parametrize("D", [1, 4, 7, 8, 20, 64, 100, 1001, 4104])
def test_lookup(ti, to, D):
    g = gen(D)
    for n, V, kind, bits in ((1, 1, "same", torch.int64), (33, 97, "wild", torch.int32), (700, 1000, "wild", torch.int64), (5, 0, "none", torch.int32)):
        w = randn(g, V, D, dtype=ti, std=0.1)
        t = tokens_of(g, n, V, kind, bits)
        for scale in (1.0, 0.37):
            got = ops().token_embedding(w, t, scale=scale, output_dtype=CODE[to])
            assert got.dtype == to
            want = lookup64(w, t, scale)
            within(got, want, lookup_bound(want, to))
            assert bool((got[want.abs().sum(-1) == 0] == 0).all())


def test_lookup_of_many_rows_and_shapes():
    g = gen(5)
    w = randn(g, 5000, 256, dtype=BF16)
    t = tokens_of(g, 300 * 211, 5000, "wild", torch.int64).view(300, 211)
    got = ops().token_embedding(w, t)
    assert got.dtype == BF16 and got.shape == (300, 211, 256)
    assert torch.equal(got.double(), lookup64(w, t, 1.0))         # scale 1 and the same type: the very bytes
    assert ops().token_embedding(w, t[:, :0]).shape == (300, 0, 256)
    assert torch.equal(ops().token_embedding(w, t[0, 0]), got[0, 0])                 # a single number
    assert torch.equal(ops().token_embedding(w, t.t()), got.transpose(0, 1))         # tokens of any stride
    assert ops().token_embedding(w[:, :0], t).shape == (300, 211, 0)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("offset,stride,D", [(0, 80, 64), (1, 67, 64), (8, 72, 72), (4, 68, 68), (2, 64, 30)])
def test_lookup_of_strided_rows(dtype, offset, stride, D):
    g = gen(stride)
    base = randn(g, offset + 40 * stride, dtype=dtype)
    w = base[offset:].view(40, stride)[:, :D]
    t = tokens_of(g, 100, 40, "wild", torch.int32)
    want = lookup64(w, t, 1.0)
    assert torch.equal(ops().token_embedding(w, t).double(), want)
    # a transposed table, one row for all
    assert torch.equal(ops().token_embedding(w.t().contiguous().t(), t).double(), want)
    assert torch.equal(ops().token_embedding(w[:1].expand(40, D), t).double(), lookup64(w[:1].expand(40, D), t, 1.0))


def test_lookup_keeps_special_values():
    w = torch.tensor([[float("inf"), float("-inf"), float("nan"), 0.0, -0.0, 3e38, 1e-40, 65504.0]], device="cuda")
    t = torch.zeros(2, dtype=torch.int64, device="cuda")
    got = ops().token_embedding(w, t)
    assert bool(got[:, 2].isnan().all())          # which NaN a product of one is, IEEE 754 leaves open
    keep = [0, 1, 3, 4, 5, 6, 7]
    assert torch.equal(got[:, keep].view(torch.int32), w.expand(2, 8)[:, keep].contiguous().view(torch.int32))
    half = ops().token_embedding(w, t, output_dtype=CODE[F16])
    assert torch.equal(half[0].nan_to_num(7.0), w[0].half().nan_to_num(7.0))


def test_lookup_reports_tokens_outside_the_table():
    from fbgemm_ascend_b200 import cabi
    g = gen(1)
    w, out = randn(g, 10, 16), torch.full((3, 40), 7.0, device="cuda")
    rows = ops().quantize_to_group_rows(w, 32)
    for call in (lambda t, flag: cabi.token_embedding(w, t, out[:, :16], error_flag=flag),
                 lambda t, flag: cabi.group_row_embedding(rows, 16, 32, t, out[:, :16], error_flag=flag)):
        for last, bit in ((9, 0), (-1, 0), (10, 4), (-2, 4)):
            flag = torch.zeros(1, dtype=torch.int32, device="cuda")
            call(torch.tensor([0, 3, last], device="cuda"), flag)
            assert int(flag) == bit
            assert bool((out[:, 16:] == 7.0).all())               # what lies between the rows stays


# ---- gradient ----------------------------------------------------------------------------------------------------

def grad64(dy, tokens, V, scale, padding=-1):
    """(gradient, sum of magnitudes per element, tokens per row) in 64 bits."""
    t = tokens.long().reshape(-1)
    dy = dy.reshape(t.numel(), -1).double() * float(np.float32(scale))
    met = (t >= 0) & (t < V) & (t != padding)
    z = lambda: torch.zeros(V, dy.shape[1], dtype=torch.float64, device=dy.device)
    total, mass = z().index_put_((t[met],), dy[met], accumulate=True), z().index_put_((t[met],), dy[met].abs(), accumulate=True)
    return total, mass, torch.bincount(t[met], minlength=V).double()[:, None]


def grad_bound(want, mass, count, dtype):
    """A term passes at most `count` additions in fp32, the sum one product; then the rounding to the result's type."""
    off = (count + 2) * 2.0 ** -24 * mass
    return off + (want.abs() + off) * U[dtype] + TINY[dtype] + 2.0 ** -140


GRAD_SIZES = [(1, 1, 8), (1023, 1000, 128), (1025, 40, 264), (2048, 9, 7), (2049, 9, 7), (40, 30, 8193), (1, 5000, 64), (31, 7, 40), (32, 511, 1), (33, 512, 36), (64, 513, 256), (1000, 3, 8), (4095, 1000, 24), (4097, 70_000, 8),
              (9000, 262_143, 16), (20_001, 2, 4), (70_001, 40_000, 12), (140_000, 300, 8), (262_145, 70_000, 4), (300, 50, 1001), (257, 33, 2056)]


@pytest.mark.parametrize("n,V,D", GRAD_SIZES)
@pytest.mark.parametrize("kind", ["uniform", "same", "spread", "hot", "few", "none", "wild"])
def test_grad(n, V, D, kind):
    g = gen(n + D)
    for ti, to, bits, scale, padding in ((F32, F32, torch.int64, 1.0, -1), (BF16, F32, torch.int32, 0.37, V // 2), (F16, F16, torch.int64, 1.0, -1),
                                         (BF16, BF16, torch.int32, 0.5, V - 1)):
        dy, t = randn(g, n, D, dtype=ti, std=0.01), tokens_of(g, n, V, kind, bits)
        got = ops().token_embedding_grad(dy, t, V, scale=scale, padding_idx=None if padding < 0 else padding, output_dtype=CODE[to])
        assert got.dtype == to and got.shape == (V, D)
        want, mass, count = grad64(dy, t, V, scale, padding)
        within(got, want, grad_bound(want, mass, count, to))
        assert bool((got[(count == 0)[:, 0]] == 0).all())
        again = ops().token_embedding_grad(dy, t, V, scale=scale, padding_idx=None if padding < 0 else padding, output_dtype=CODE[to])
        assert torch.equal(got, again)                            # the order of the sums is fixed


@pytest.mark.parametrize("n,V,D,ti,to", [(700, 300_007, 64, F32, F32), (5000, 300_007, 101, BF16, F16), (70_000, 150_000, 128, BF16, F32),
                                         (1, 1_000_033, 32, F16, F32), (200_000, 400_000, 64, F32, BF16)])
@pytest.mark.parametrize("kind", ["uniform", "hot", "wild", "none"])
def test_grad_of_a_large_table(n, V, D, ti, to, kind):
    """Tables whose rows are cleared partly beside the sums, where no token names them."""
    g = gen(n)
    dy, t = randn(g, n, D, dtype=ti, std=0.01), tokens_of(g, n, V, kind, torch.int64)
    junk = torch.full((V, D), float("nan"), device="cuda", dtype=to)          # what the allocator hands out next
    del junk
    got = ops().token_embedding_grad(dy, t, V, padding_idx=7, output_dtype=CODE[to])
    want, mass, count = grad64(dy, t, V, 1.0, 7)
    within(got, want, grad_bound(want, mass, count, to))
    assert bool((got[(count == 0)[:, 0]] == 0).all())


@pytest.mark.parametrize("n,V,D,stride", [(900, 60_000, 200, 264), (900, 60_000, 199, 201), (40, 77, 8, 9), (9000, 60_000, 200, 264), (9000, 60_000, 199, 201)])
def test_grad_into_rows_that_lie_apart(n, V, D, stride):
    """The C entry point over a wider buffer: every row is written, nothing between the rows."""
    from fbgemm_ascend_b200 import cabi
    g = gen(n)
    lib = cabi.lib()
    dy, t = randn(g, n, D), tokens_of(g, n, V, "hot", torch.int64)
    out = torch.full((V, stride), 7.0, device="cuda")
    need = lib.tbe_b200_token_embedding_grad_scratch_bytes(n, V, D)
    scratch = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    cabi.check(lib.tbe_b200_token_embedding_grad(dy.data_ptr(), 0, D, t.data_ptr(), 64, n, V, D, 2.0, -1, 0, out.data_ptr(), 0, stride, scratch.data_ptr(),
                                                 need, torch.cuda.current_stream().cuda_stream), "grad")
    assert torch.equal(out[:, :D], ops().token_embedding_grad(dy, t, V, scale=2.0)) and bool((out[:, D:] == 7.0).all())


@pytest.mark.parametrize("n,V,D,kind", [(1, 9, 8, "same"), (500, 60, 40, "hot"), (4097, 300, 1001, "wild"), (5000, 100_000, 64, "uniform"),
                                        (300, 40, 33, "same"), (40, 9, 16, "none")])
@pytest.mark.parametrize("ti,to", [(BF16, F32), (F32, F32), (BF16, BF16), (F16, F16)])
def test_grad_into_a_buffer(n, V, D, kind, ti, to):
    g = gen(n)
    dy, t = randn(g, n, D, dtype=ti, std=0.01), tokens_of(g, n, V, kind, torch.int64)
    wide = randn(g, V, D + 8, dtype=to, std=0.01)
    into = wide[:, :D]
    old, beside, version = into.clone(), wide[:, D:].clone(), into._version
    got = ops().token_embedding_grad_(into, dy, t, scale=0.5, padding_idx=-1)        # the last row
    assert got.data_ptr() == into.data_ptr() and into._version > version
    want, mass, count = grad64(dy, t, V, 0.5, V - 1)
    total = want + old.double()
    off = (count + 2) * 2.0 ** -24 * mass + 2.0 ** -24 * total.abs()
    within(into, total, off + (total.abs() + off) * U[to] + TINY[to])
    untouched = (count == 0)[:, 0]
    assert torch.equal(into[untouched], old[untouched]) and torch.equal(wide[:, D:], beside)


@pytest.mark.parametrize("D", [1, 2, 6, 31, 34, 66, 126, 130, 255, 258, 1030])
@pytest.mark.parametrize("ti,to", [(BF16, F32), (F16, F16), (F32, F32), (F32, BF16)])
def test_grad_of_rows_that_begin_anywhere(D, ti, to):
    """More tokens than one launch takes; rows of both matrices 1, 2 or 3 elements behind a border, or alternating."""
    n, V = 2300, 90
    g = gen(D)
    t = tokens_of(g, n, V, "wild", torch.int64)
    for first, gap in ((0, 0), (1, 1), (2, 2), (3, 5), (1, 0)):
        wide = randn(g, n * (D + gap) + first, dtype=ti, std=0.01)
        dy = wide[first:].view(n, D + gap)[:, :D]
        want, mass, count = grad64(dy, t, V, 0.5)
        got = ops().token_embedding_grad(dy, t, V, scale=0.5, output_dtype=CODE[to])
        within(got, want, grad_bound(want, mass, count, to))
        buffer = randn(g, V * (D + gap) + first + 9, dtype=to, std=0.01)
        was = buffer.clone()
        view = lambda b: b[first:first + V * (D + gap)].view(V, D + gap)
        ops().token_embedding_grad_(view(buffer)[:, :D], dy, t, scale=0.5)
        total = want + view(was)[:, :D].double()
        off = (count + 2) * 2.0 ** -24 * mass + 2.0 ** -24 * total.abs()
        within(view(buffer)[:, :D], total, off + (total.abs() + off) * U[to] + TINY[to])
        assert torch.equal(view(buffer)[:, D:], view(was)[:, D:]) and torch.equal(buffer[:first], was[:first]) and torch.equal(buffer[-9:], was[-9:])


def test_grad_of_strided_broadcast_and_empty_rows():
    g = gen(3)
    t = tokens_of(g, 60, 11, "uniform", torch.int64).view(6, 10)
    check = lambda dy: within(ops().token_embedding_grad(dy, t, 11), grad64(dy, t, 11, 1.0)[0], grad_bound(*grad64(dy, t, 11, 1.0), dy.dtype))
    check(randn(g, 6, 10, 40)[:, :, 3:27])
    check(randn(g, 10, 6, 24, dtype=BF16).transpose(0, 1))
    check(randn(g, 24).expand(6, 10, 24))
    check(torch.ones((), device="cuda").expand(6, 10, 24))
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    assert torch.equal(ops().token_embedding_grad(torch.empty(0, 24, device="cuda"), none, 5), torch.zeros(5, 24, device="cuda"))
    for V, D in ((3, 8200), (17_000_000, 4)):                                    # tables that few tokens' own form does not take
        junk = torch.full((V, D), float("nan"), device="cuda")
        del junk
        assert not bool(ops().token_embedding_grad(torch.empty(0, D, device="cuda"), none, V).any())
        dy, one = randn(g, 1, D), torch.tensor([V - 1], device="cuda")
        got = ops().token_embedding_grad(dy, one, V)
        assert torch.equal(got[V - 1:], dy) and not bool(got[:V - 1].any())
    kept = randn(g, 5, 24)
    assert torch.equal(ops().token_embedding_grad_(kept.clone(), torch.empty(0, 24, device="cuda"), none), kept)
    assert ops().token_embedding_grad(randn(g, 60, 24), t.view(-1), 0).shape == (0, 24)
    assert ops().token_embedding_grad(torch.empty(60, 0, device="cuda"), t.view(-1), 7).shape == (7, 0)


def test_grad_of_special_values_stays_in_its_row():
    dy = torch.ones(6, 16, device="cuda")
    dy[1, 3], dy[2, 4], dy[5] = float("nan"), float("inf"), float("nan")
    t = torch.tensor([0, 1, 2, 2, 1, -1], device="cuda")
    got = ops().token_embedding_grad(dy, t, 4)
    assert bool(got[1, 3].isnan()) and float(got[2, 4]) == float("inf")
    assert int(got.isnan().sum()) == 1 and int(got.isinf().sum()) == 1 and torch.equal(got[3], torch.zeros(16, device="cuda"))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_autograd(dtype):
    import fbgemm_ascend_b200 as fa
    g = gen(8)
    emb = fa.TokenEmbedding(300, 72, padding_idx=5, scale=8.0, dtype=dtype)
    t = tokens_of(g, 4 * 33, 300, "wild", torch.int64).view(4, 33)
    t[0, :7] = 5
    out = emb(t)
    dy = randn(g, 4, 33, 72, dtype=dtype)
    out.backward(dy)
    want = grad64(dy, t, 300, 8.0, 5)
    assert emb.weight.grad.dtype == dtype
    within(emb.weight.grad, want[0], grad_bound(*want, dtype))
    # added up by the engine on the second pass, and by the program's own buffer
    emb(t).backward(dy)
    within(emb.weight.grad, 2 * want[0], 3 * grad_bound(2 * want[0], 2 * want[1], want[2], dtype))
    kept = torch.zeros(300, 72, device="cuda")
    emb.add_gradient_(kept, dy, t)
    within(kept, want[0], grad_bound(*want, F32))
    with torch.no_grad():
        assert not emb(t).requires_grad


def test_gradient_against_differences_and_of_the_gradient():
    g = gen(9)
    w, t = randn(g, 20, 12).requires_grad_(), tokens_of(g, 50, 20, "wild", torch.int64)
    e, dy = randn(g, 20, 12), randn(g, 50, 12)
    f = lambda w: (torch.sin(ops().token_embedding(w, t, scale=0.5, padding_idx=3)).double() * dy.double()).sum()
    e[3] = 0      # the padding row has no gradient
    (grad,) = torch.autograd.grad(f(w), w, create_graph=True)
    h = 2.0 ** -6
    with torch.no_grad():
        difference = (f(w + h * e) - f(w - h * e)) / (2 * h)
    # |third derivative| <= (0.5 |e|)^3 |dy| per element; fp32: each of 600 terms is off by a few 2^-24, over 2h = 2^-5
    bound = (h * h / 6) * 0.125 * float((e.abs().max() ** 3) * dy.abs().sum()) + 4 * 2.0 ** -24 / (2 * h) * float(dy.abs().sum())
    assert abs(float((grad.detach().double() * e.double()).sum() - difference)) <= bound
    # second derivative: d/dw <grad, e> = -0.25 sin(.) dy e of the tokens, summed by row
    (second,) = torch.autograd.grad((grad * e).sum(), w)
    rows = lookup64(w.detach(), t, 0.5)
    term = -torch.sin(rows) * dy.double() * lookup64(e, t, 0.5)
    want, mass, count = grad64(term.float(), t, 20, 0.5, 3)
    within(second, want, (count + 40) * 2.0 ** -24 * (mass + 1e-3))


@pytest.mark.parametrize("ti,to", [(F32, F32), (BF16, F32), (F16, BF16)])
@pytest.mark.parametrize("needs_grad", [False, True])
def test_forward_mode(ti, to, needs_grad):
    """The lookup and its gradient are linear: a tangent goes through them as the values do."""
    import torch.autograd.forward_ad as fwd
    g = gen(14)
    V, D = 40, 24
    t = tokens_of(g, 3 * 25, V, "wild", torch.int64).view(3, 25)
    w, dw, dy, ddy = randn(g, V, D, dtype=ti), randn(g, V, D, dtype=ti), randn(g, 3, 25, D, dtype=ti), randn(g, 3, 25, D, dtype=ti)
    look = lambda w: ops().token_embedding(w, t, scale=0.5, padding_idx=3, output_dtype=CODE[to])
    back = lambda dy: ops().token_embedding_grad(dy, t, V, scale=0.5, padding_idx=3, output_dtype=CODE[to])
    for f, x, dx in ((look, w, dw), (back, dy, ddy)):
        value, tangent = f(x), f(dx)
        with fwd.dual_level():
            got = fwd.unpack_dual(f(fwd.make_dual(x.clone().requires_grad_(needs_grad), dx)))
            assert torch.equal(got.primal, value) and got.tangent is not None and torch.equal(got.tangent, tangent)
            assert got.primal.requires_grad == needs_grad
            assert fwd.unpack_dual(f(x)).tangent is None
        value2, tangent2 = torch.func.jvp(f, (x,), (dx,))
        assert torch.equal(value2, value) and torch.equal(tangent2, tangent)


def test_forward_mode_over_reverse():
    """The derivative of a gradient along a direction, which takes both."""
    import torch.autograd.forward_ad as fwd
    g = gen(15)
    w, e, t = randn(g, 20, 12), randn(g, 20, 12), tokens_of(g, 50, 20, "uniform", torch.int64)
    with fwd.dual_level():
        dual = fwd.make_dual(w.clone().requires_grad_(), e)
        (grad,) = torch.autograd.grad((ops().token_embedding(dual, t, scale=0.5) ** 2).sum(), dual, create_graph=True)
        got = fwd.unpack_dual(grad).tangent
    want, mass, count = grad64(2 * lookup64(e, t, 0.5).float(), t, 20, 0.5)
    within(got, want, (count + 8) * 2.0 ** -24 * mass + 2.0 ** -140)


def test_forward_mode_is_refused_where_there_is_no_derivative():
    import torch.autograd.forward_ad as fwd
    w, t, dy = torch.ones(10, 16, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda"), torch.ones(4, 16, device="cuda")
    rows, b = ops().quantize_to_group_rows(w, 32), torch.ones(10, device="cuda")
    calls = [(lambda x: ops().quantize_to_group_rows(x, 32), w), (lambda x: ops().group_row_linear(x, rows, 32), w),
             (lambda x: ops().group_row_linear(w, rows, 32, bias=x), b), (lambda x: ops().token_embedding_grad_(w.clone(), x, t), dy),
             (lambda x: ops().token_embedding_grad_(x, dy, t), w)]
    for f, x in calls:
        with fwd.dual_level():
            dual = fwd.make_dual(x.clone(), torch.ones_like(x))
            with pytest.raises(RuntimeError, match="gradient|graph"):
                f(dual)
            with torch.no_grad(), pytest.raises(RuntimeError, match="gradient|graph"):
                f(dual)
            f(dual.detach())
        with pytest.raises(RuntimeError, match="gradient|graph"):
            torch.func.jvp(f, (x,), (torch.ones_like(x),))
        with pytest.raises(RuntimeError, match="gradient|graph"):
            torch.func.grad(lambda x: f(x).float().sum())(x)


# ---- 4-bit rows with group scales --------------------------------------------------------------------------------

def rows_by_oracle(x, group):
    """The bytes of rows of fp32 x [E, D], group by group by the CPU quantizer of 4-bit rows; and their numbers."""
    E, D = x.shape
    out, back = np.zeros((E, group_row_bytes(D, group)), dtype=np.uint8), np.zeros((E, D), dtype=np.float32)
    for k, lo in enumerate(range(0, D, group)):
        part = O.quantize_nbit_rowwise_sbhalf(np.ascontiguousarray(x[:, lo:lo + group]), 4)
        w = min(group, D - lo) // 2
        out[:, lo // 2:lo // 2 + w] = part[:, :w]
        out[:, D // 2 + 4 * k:D // 2 + 4 * k + 4] = part[:, w:]
        back[:, lo:lo + group] = O.dequantize_nbit_rowwise_sbhalf(part, 4)
    return out, back


@pytest.mark.parametrize("D", [8, 24, 32, 40, 136, 256, 264, 1000, 4096])
@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("kind", ["normal", "const", "tiny", "mixed"])
def test_group_rows_bit_exact(D, group, kind):
    rng = np.random.default_rng(D + group)
    x = rng.normal(0, 0.1, (37, D)).astype(np.float32)
    if kind == "const":
        x[:] = 0.37
    elif kind == "tiny":
        x *= np.float32(1e-9)
    elif kind == "mixed":
        x[::3] *= np.float32(1e-4)
        x[1::3] *= np.float32(300)
        x[:, 0] = 0
    for dtype in (F32, F16, BF16):
        t = torch.from_numpy(x).cuda().to(dtype)
        want, numbers = rows_by_oracle(t.float().cpu().numpy(), group)
        got = ops().quantize_to_group_rows(t, group)
        assert np.array_equal(got.cpu().numpy(), want)
        wide = torch.randn(37, D + 5, device="cuda").to(dtype)
        wide[:, 3:3 + D] = t
        assert torch.equal(ops().quantize_to_group_rows(wide[:, 3:3 + D], group), got)      # rows that are not aligned
        back = ops().group_rows_to_float(got, D, group)
        assert np.array_equal(back.cpu().numpy().view(np.uint32), numbers.view(np.uint32))
        assert torch.equal(ops().group_rows_to_float(got, D, group, output_dtype=CODE[dtype]), back.to(dtype))
    if D <= group and D % 8 == 0:      # one group: the fused rows of the whole package
        fused = torch.ops.fbgemm.FloatToFusedNBitRowwiseQuantizedSBHalf(torch.from_numpy(x).cuda(), 4)
        assert torch.equal(ops().quantize_to_group_rows(torch.from_numpy(x).cuda(), group)[:, :D // 2 + 4], fused)


@pytest.mark.parametrize("D,group", [(8, 32), (200, 64), (256, 32), (1000, 128), (4096, 256), (520, 128)])
@pytest.mark.parametrize("to", [F32, F16, BF16])
def test_group_row_lookup(D, group, to):
    g = gen(D)
    rows = ops().quantize_to_group_rows(randn(g, 90, D, std=0.1), group)
    numbers = ops().group_rows_to_float(rows, D, group)
    for n, kind, bits, scale in ((1, "same", torch.int64, 1.0), (301, "wild", torch.int32, 0.37), (0, "none", torch.int64, 1.0), (5000, "uniform", torch.int64, 2.0)):
        t = tokens_of(g, n, 90, kind, bits)
        got = ops().group_row_embedding(rows, t, D, group, scale=scale, output_dtype=CODE[to])
        want = lookup64(numbers, t, scale)
        within(got, want, lookup_bound(want, to))
    from fbgemm_ascend_b200 import cabi
    out = torch.zeros(5, D + 3, device="cuda", dtype=to)       # rows that are not aligned
    t = torch.tensor([0, 89, -1, 90, 44], device="cuda")
    cabi.group_row_embedding(rows, D, group, t, out[:, 1:1 + D])
    assert torch.equal(out[:, 1:1 + D], ops().group_row_embedding(rows, t, D, group, output_dtype=CODE[to]))
    assert bool((out[:, 0] == 0).all()) and bool((out[:, 1 + D:] == 0).all())


# ---- products with 4-bit rows ------------------------------------------------------------------------------------

def linear_want(x, rows, D, group, bias):
    """(products, bound of the fp32 arithmetic) in 64 bits.

    Codes are whole numbers around their middle: |code - 8| <= 8, so a term is at most |x| * (8 |scale| + |bias + 8 scale|).
    It passes 16-term products of a matrix instruction, up to 16 of them per group (cut off, not rounded: 2^-23), a step
    per group, and the joining of the pieces: 64 + D / group of them at 2^-23 hold for any split.
    """
    numbers = ops().group_rows_to_float(rows, D, group).double()
    G = -(-D // group)
    head = rows[:, D // 2:D // 2 + 4 * G].contiguous().view(torch.float16).double().view(-1, G, 2)
    most = (8 * head[:, :, 0].abs() + (head[:, :, 1] + 8 * head[:, :, 0]).abs()).repeat_interleave(group, 1)[:, :D]
    want, mass = x.double() @ numbers.t(), x.double().abs() @ most.t()
    if bias is not None:
        want, mass = want + bias.double(), mass + bias.double().abs()
    return want, (64 + G) * 2.0 ** -23 * mass


LINEAR_SIZES = [(1, 1, 8, 32), (1, 15, 32, 32), (2, 17, 40, 64), (3, 33, 128, 32), (4, 64, 256, 128), (5, 100, 264, 256), (7, 31, 1000, 32),
                (8, 129, 1024, 64), (9, 50, 2056, 128), (12, 300, 4096, 128), (16, 47, 5000, 32), (17, 20, 512, 64), (35, 70, 776, 128),
                (1, 4099, 2048, 128), (1, 37, 16_400, 256), (8, 10_007, 520, 32), (70_000, 2, 8, 32)]


@pytest.mark.parametrize("m,N,D,group", LINEAR_SIZES)
@pytest.mark.parametrize("ti,to", [(BF16, BF16), (F16, F16), (BF16, F32), (F32, F32), (F16, BF16)])
def test_linear(m, N, D, group, ti, to):
    g = gen(N + D)
    rows = ops().quantize_to_group_rows(randn(g, N, D, std=0.05), group)
    x = randn(g, m, D, dtype=ti)
    for bias in (None, randn(g, N, dtype=to)):
        got = ops().group_row_linear(x, rows, group, bias=bias, output_dtype=CODE[to])
        assert got.dtype == to and got.shape == (m, N)
        want, off = linear_want(x, rows, D, group, bias)
        within(got, want, off + (want.abs() + off) * U[to] + TINY[to])


def test_linear_of_far_apart_magnitudes():
    """Rows of scales from 1e-7 to 1e3 and states from 1e-30 to 1e30: every row and state keeps its own precision."""
    g = gen(4)
    size = 10.0 ** torch.linspace(-3, 4, 64, device="cuda")
    rows = ops().quantize_to_group_rows(randn(g, 64, 512) * size[:, None] / 10, 64)
    for dtype, ends in ((F32, 30), (BF16, 30), (F16, 4)):
        x = (randn(g, 8, 512) * (10.0 ** torch.linspace(-ends, ends, 8, device="cuda"))[:, None]).to(dtype)
        got = ops().group_row_linear(x, rows, 64, output_dtype=CODE[F32])
        want, off = linear_want(x, rows, 512, 64, None)
        within(got, want, off + (want.abs() + off) * U[F32] + 2.0 ** -120)


def test_linear_of_special_values_stays_in_its_state():
    g = gen(6)
    rows = ops().quantize_to_group_rows(randn(g, 40, 320), 64)
    for dtype in (F32, F16, BF16):
        x = randn(g, 5, 320, dtype=dtype)
        clean = ops().group_row_linear(x, rows, 64)
        x[1, 7], x[3, 300], x[3, 2] = float("nan"), float("inf"), float("-inf")
        got = ops().group_row_linear(x, rows, 64)
        assert bool((~got[[1, 3]].isfinite()).all()) and torch.equal(got[[0, 2, 4]], clean[[0, 2, 4]])


def test_linear_of_shapes_and_strides():
    g = gen(7)
    rows = ops().quantize_to_group_rows(randn(g, 50, 136), 64)
    x = randn(g, 2, 3, 136, dtype=BF16)
    got = ops().group_row_linear(x, rows, 64)
    assert got.shape == (2, 3, 50) and got.dtype == BF16
    flat = ops().group_row_linear(x.view(6, 136), rows, 64)
    assert torch.equal(got.view(6, 50), flat)
    assert torch.equal(ops().group_row_linear(x[0, 0], rows, 64), flat[0])
    wide = torch.zeros(6, 150, device="cuda", dtype=BF16)
    for at in (0, 3, 8):
        wide[:, at:at + 136] = x.view(6, 136)
        assert torch.equal(ops().group_row_linear(wide[:, at:at + 136], rows, 64), flat)
    assert torch.equal(ops().group_row_linear(x.view(6, 136).t().contiguous().t(), rows, 64), flat)
    assert ops().group_row_linear(x[:0], rows, 64).shape == (0, 3, 50)
    assert ops().group_row_linear(x, rows[:0], 64).shape == (2, 3, 0)
    assert torch.equal(ops().group_row_linear(x, rows[7:20], 64), got[:, :, 7:20])


def exact_linear(x, rows, D, group, bias=None):
    """(products, bound) in 64 bits, from the codes themselves: a code of 0 leaves nothing but the group's bias.

    An element stands for code * scale + bias, so its terms are |x| * (code |scale| + |bias|).  A term passes up to 32 matrix
    instructions of a group (sums are cut off, 2^-23; 21 additions for the sum of the states), two FMAs a group, 16 shares and the
    bias: 64 + 2 G roundings.  bf16 and fp32 states are held to 2^-23 of an element or 2^-39 of the state's largest one.
    """
    G = -(-D // group)
    code = torch.stack([rows[:, :D // 2] & 15, rows[:, :D // 2] >> 4], 2).view(-1, D).double()
    head = rows[:, D // 2:D // 2 + 4 * G].contiguous().view(torch.float16).double().view(-1, G, 2).repeat_interleave(group, 1)[:, :D]
    number, term = code * head[..., 0] + head[..., 1], code * head[..., 0].abs() + head[..., 1].abs()
    x64 = x.double()
    held = torch.zeros_like(x64) if x.dtype == F16 else torch.maximum(2.0 ** -39 * x64.abs().amax(1, keepdim=True), (2.0 ** -23 if x.dtype == F32 else 0.0) * x64.abs())
    want, mass = x64 @ number.t(), (x64.abs() + held) @ term.t()
    off = held @ number.abs().t()
    if bias is not None:
        want, mass = want + bias.double(), mass + bias.double().abs()
    return want, off + (64 + 2 * G) * 2.0 ** -23 * mass


@pytest.mark.parametrize("m,D,group", [(1, 4096, 128), (3, 1000, 32), (8, 520, 64), (9, 2048, 256), (16, 264, 32), (17, 776, 128), (2, 16_400, 64)])
@pytest.mark.parametrize("ti", [F32, F16, BF16])
def test_linear_of_rows_without_a_span(m, D, group, ti):
    """Groups whose elements are all alike, or nearly: the quantizer gives them scale 1 and codes 0, or a scale far below the bias."""
    g = gen(D + m)
    values = [0.0, -0.0, 1e-3, 1e-4, 1e-5, -1e-6, 1e-7, 0.37, -250.0, 3e-5, 6e-8]
    x = torch.zeros(len(values) + 5, D, device="cuda")
    for r, v in enumerate(values):
        x[r] = v
    few = x[len(values):]
    few[0] = 1e-3 + 3e-7 * torch.rand(D, device="cuda", generator=g)          # a span of a few steps of the scale's smallest number
    few[1] = randn(g, D, std=1e-3)
    few[1, :group] = 0.0                                                      # a group of zeros among small ones
    few[2] = randn(g, D, std=1e-6)
    few[2, -8:] = 1e-6
    few[3] = randn(g, D, std=1e-7)
    few[4] = randn(g, D, std=0.05)
    few[4, group:2 * group] = 2e-6
    rows = ops().quantize_to_group_rows(x, group)
    states = randn(g, m, D, dtype=ti)
    for bias in (None, randn(g, x.shape[0], std=1e-6)):
        got = ops().group_row_linear(states, rows, group, bias=bias, output_dtype=CODE[F32])
        want, off = exact_linear(states, rows, D, group, bias)
        within(got, want, off + (want.abs() + off) * U[F32] + TINY[F32])
        if bias is None:
            assert not bool(got[:, :2].any())                                 # zeros score zero


@pytest.mark.parametrize("dtype,span", [(F32, 60), (BF16, 60), (F16, 20)])
@pytest.mark.parametrize("m", [3, 20])
def test_linear_of_states_with_elements_far_apart(dtype, span, m):
    """Elements of one state over `span` powers of two, and rows from 1e-7 to 1e3."""
    g = gen(span + m)
    for D, group in ((512, 64), (1000, 32), (4096, 128)):
        size = 10.0 ** torch.linspace(-7, 3, 48, device="cuda")
        rows = ops().quantize_to_group_rows(randn(g, 48, D) * size[:, None], group)
        x = (randn(g, m, D) * 2.0 ** (-span * torch.rand(m, D, device="cuda", generator=g))).to(dtype)
        got = ops().group_row_linear(x, rows, group, output_dtype=CODE[F32])
        want, off = exact_linear(x, rows, D, group)
        within(got, want, off + (want.abs() + off) * U[F32] + TINY[F32])


@pytest.mark.parametrize("m,N,D,group,ti", [(1, 40, 512, 128, BF16), (16, 5000, 1000, 32, F32), (8, 70_000, 264, 64, F16), (17, 300, 776, 256, BF16), (3, 20_000, 16_400, 128, F32)])
def test_linear_whose_waits_run_out(m, N, D, group, ti):
    """Rows that do not arrive in time leave NaN and a word for the host, and the next call is as ever."""
    from fbgemm_ascend_b200 import cabi
    lib, g = cabi.lib(), gen(m + D)
    rows, x = ops().quantize_to_group_rows(randn(g, N, D, std=0.05), group), randn(g, m, D, dtype=ti)
    need = lib.tbe_b200_group_row_linear_scratch_bytes(m, D, group, CODE[ti])
    scratch = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")

    def call(polls, to, flag):
        out = torch.zeros(m, N, device="cuda", dtype=to)
        cabi.check(lib.tbe_b200_group_row_linear_bounded(x.data_ptr(), CODE[ti], D, m, rows.data_ptr(), N, rows.shape[1], D, group, None, 0, out.data_ptr(), CODE[to], N,
                                                         None if flag is None else flag.data_ptr(), scratch.data_ptr(), need, polls,
                                                         torch.cuda.current_stream().cuda_stream), "linear")
        return out

    want = ops().group_row_linear(x, rows, group, output_dtype=CODE[F32])
    for to in (F32, BF16):
        flag = torch.zeros(1, dtype=torch.int32, device="cuda")
        assert bool(call(0, to, flag).isnan().all()) and int(flag) == 16
        assert bool(call(0, to, None).isnan().all())
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert torch.equal(call(1 << 20, F32, flag), want) and int(flag) == 0
    assert torch.equal(ops().group_row_linear(x, rows, group, output_dtype=CODE[F32]), want)


# ---- places behind 2^31 -------------------------------------------------------------------------------------------

def test_rows_far_into_a_large_table():
    g = gen(21)
    V, D = 140_000, 16_400
    w = torch.zeros(V, D, device="cuda", dtype=BF16)              # 4.6 GB, 2.3 billion elements
    t = torch.tensor([V - 1, 0, 131_071, 131_072, V - 1, -1], device="cuda")
    w[t[:4]] = randn(g, 4, D, dtype=BF16)
    assert torch.equal(ops().token_embedding(w, t).double(), lookup64(w, t, 1.0))
    dy = randn(g, 6, D, dtype=BF16)
    for again in (1, 500):                                        # a few tokens, and more of them
        rows, tokens = dy.repeat(again, 1), t.repeat(again)
        got = ops().token_embedding_grad(rows, tokens, V)
        for v in (V - 1, 0, 131_071, 131_072):
            want, mass, count = grad64(rows, (tokens == v).long() - 1, 1, 1.0)
            within(got[v:v + 1], want, grad_bound(want, mass, count, BF16))
        got[t[:4]] = 0
        assert not bool(got.any())
        del got, rows


def test_group_rows_far_into_a_large_table():
    import fbgemm_ascend_b200 as fa
    g = gen(22)
    V, D = 2_200_000, 2048
    table = fa.GroupRowTable(V, D, 128)                           # 2.4 GB
    last = randn(g, 5, D, std=0.1)
    table.assign_rows_from_float(last, V - 5)
    t = torch.tensor([V - 1, V - 5, 7, V], device="cuda")
    want = ops().group_rows_to_float(table.rows[V - 5:], D, 128)
    assert torch.equal(table(t).float(), torch.stack([want[4], want[0], torch.zeros_like(want[0]), torch.zeros_like(want[0])]).bfloat16().float())
    x = randn(g, 2, D, dtype=BF16)
    scores = table.linear(x, output_dtype=SparseType.FP32)
    exact, off = linear_want(x, table.rows[V - 5:], D, 128, None)
    within(scores[:, V - 5:], exact, off + (exact.abs() + off) * U[F32])
    assert not bool(scores[:, :V - 5].any())


# ---- together, streams, graphs ------------------------------------------------------------------------------------

def test_train_publish_serve():
    """A table is trained a step, published in 4 bits, and serves tokens and scores; everything on a side stream."""
    import fbgemm_ascend_b200 as fa
    g = gen(11)
    V, D = 515, 264
    emb = fa.TokenEmbedding(V, D, padding_idx=0, scale=16.0)
    t, dy = tokens_of(g, 2000, V, "hot", torch.int64), randn(g, 2000, D)
    before = emb.weight.detach().clone()
    table = fa.GroupRowTable(V, D, 64)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        emb(t).backward(dy)
        with torch.no_grad():
            emb.weight -= 0.01 * emb.weight.grad
        for lo in range(0, V, 200):
            table.assign_rows_from_float(emb.weight[lo:lo + 200], lo)
        hidden = table(t[:9], scale=16.0)
        scores = table.linear(hidden, output_dtype=SparseType.FP32)
    torch.cuda.current_stream().wait_stream(side)
    want, mass, count = grad64(dy, t, V, 16.0, 0)
    after = before.double() - 0.01 * want
    off = 0.01 * grad_bound(want, mass, count, F32) + 3 * 2.0 ** -24 * (before.double().abs() + 0.01 * want.abs())
    within(emb.weight, after, off)
    numbers = table.to_float()
    spans = emb.weight.detach().view(V, -1, 8).double()
    assert np.array_equal(table.rows.cpu().numpy(), rows_by_oracle(emb.weight.detach().cpu().numpy(), 64)[0]) and spans.shape[1] == 33
    looked = lookup64(numbers, t[:9], 16.0)
    within(hidden, looked, lookup_bound(looked, BF16))
    want, off = linear_want(hidden, table.rows, D, 64, None)
    within(scores, want, off + (want.abs() + off) * U[F32])


@pytest.mark.parametrize("n,m,V,D", [(700, 3, 3000, 128), (5000, 20, 3000, 104), (20_000, 16, 200_000, 136), (270_001, 1, 3000, 16)])
def test_graphs_replay_with_new_inputs(n, m, V, D):
    """Two captured graphs of the same calls, replayed in turn with new contents, and an eager call in between."""
    g = gen(12)
    held = []
    for _ in range(2):
        s = {"w": randn(g, V, D, dtype=BF16), "t": tokens_of(g, n, V, "wild", torch.int64), "dy": randn(g, n, D, dtype=BF16), "into": torch.zeros(V, D, device="cuda"),
             "x": randn(g, m, D, dtype=BF16)}

        def step(s=s):
            rows = ops().quantize_to_group_rows(s["w"], 64)
            return [ops().token_embedding(s["w"], s["t"], scale=0.5), ops().token_embedding_grad(s["dy"], s["t"], V, scale=2.0),
                    ops().token_embedding_grad_(s["into"], s["dy"], s["t"]), ops().group_row_embedding(rows, s["t"], D, 64),
                    ops().group_row_linear(s["x"], rows, 64)]

        with torch.no_grad():
            step()
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outs = step()
        held.append((s, step, graph, outs))
    with torch.no_grad():
        for turn in range(3):
            for s, step, graph, outs in held:
                for k in ("w", "dy", "x"):
                    s[k].copy_(randn(g, *s[k].shape, dtype=s[k].dtype))
                s["t"].copy_(tokens_of(g, n, V, ("hot", "uniform", "none")[turn], torch.int64))
                s["into"].zero_()
            for s, step, graph, outs in held:
                graph.replay()
            got = [[o.clone() for o in outs] for _, _, _, outs in held]
            for (s, step, graph, outs), kept in zip(held, got):
                s["into"].zero_()
                for a, b in zip(kept, step()):
                    assert torch.equal(a, b)


def test_capture_of_a_training_step():
    """A step that lookup and backward are captured in, with no eager graph alive; and the refusal where one is, on the default stream."""
    import fbgemm_ascend_b200 as fa
    g = gen(13)
    emb = fa.TokenEmbedding(200, 64)
    t, dy = tokens_of(g, 90, 200, "uniform", torch.int64), randn(g, 90, 64)
    emb(t).backward(dy)
    want = emb.weight.grad.clone()
    emb.weight.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        emb(t).backward(dy)
    emb.weight.grad.zero_()
    graph.replay()
    assert torch.equal(emb.weight.grad, want)
    del graph
    emb.weight.grad = None
    alive = emb(t)                                # an eager graph of the same table, on the default stream
    other = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="before capturing"):
        with torch.cuda.graph(other):
            emb(t)
    torch.cuda.synchronize()
    alive.backward(dy)                            # which goes on as if nothing had been
    assert torch.equal(emb.weight.grad, want)


# ---- refusals -----------------------------------------------------------------------------------------------------

def test_refusals():
    import fbgemm_ascend_b200 as fa
    o = ops()
    w, t = torch.zeros(10, 16, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    dy, rows = torch.zeros(4, 16, device="cuda"), torch.zeros(10, 16, dtype=torch.uint8, device="cuda")
    bad = [
        (lambda: o.token_embedding(w, t.float()), "tokens must be"),
        (lambda: o.token_embedding(w, t.cpu()), "tokens must be a CUDA"),
        (lambda: o.token_embedding(w.long(), t), "float32, float16 or bfloat16"),
        (lambda: o.token_embedding(w.double(), t), "float32, float16 or bfloat16"),
        (lambda: o.token_embedding(w[0], t), "matrix"),
        (lambda: o.token_embedding(w, t, output_dtype=2), "output_dtype"),
        (lambda: o.token_embedding(w, t, padding_idx=10), "padding_idx"),
        (lambda: o.token_embedding(w, t, padding_idx=-11), "padding_idx"),
        (lambda: o.token_embedding_grad(dy[:3], t, 10), "grad must be"),
        (lambda: o.token_embedding_grad(dy, t, -1), "num_embeddings"),
        (lambda: o.token_embedding_grad(dy, t, 1 << 31), "2\\^31"),
        (lambda: o.token_embedding_grad(dy, t, 10, padding_idx=10), "padding_idx"),
        (lambda: o.token_embedding_grad(dy.double(), t, 10), "float32, float16 or bfloat16"),
        (lambda: o.token_embedding_grad_(w, dy[:, :8], t), "rows of 8"),
        (lambda: o.token_embedding_grad_(w.t(), dy, t), "must lie apart"),
        (lambda: o.token_embedding_grad_(w[:1].expand(10, 16), dy, t), "must lie apart"),
        (lambda: o.token_embedding_grad_(w, w[:4], t), "memory"),
        (lambda: o.token_embedding_grad_(w.clone().requires_grad_(), dy, t), "no_grad"),
        (lambda: o.quantize_to_group_rows(w, 48), "group_size"),
        (lambda: o.quantize_to_group_rows(w[:, :12], 32), "multiple of 8"),
        (lambda: o.quantize_to_group_rows(w[0], 32), "matrix"),
        (lambda: o.quantize_to_group_rows(w.clone().requires_grad_(), 32), "no gradient"),
        (lambda: o.group_rows_to_float(rows, 32, 32), "bytes"),
        (lambda: o.group_rows_to_float(rows.float(), 16, 32), "uint8"),
        (lambda: o.group_row_embedding(rows, t.bool(), 16, 32), "tokens must be"),
        (lambda: o.group_row_embedding(rows, t, 16, 32, output_dtype=3), "output_dtype"),
        (lambda: o.group_row_linear(w, rows, 64, bias=w[0]), "bias"),
        (lambda: o.group_row_linear(w[:, :8], rows[:, :15], 64), "bytes"),
        (lambda: o.group_row_linear(w.clone().requires_grad_(), rows, 64), "no gradient"),
        (lambda: o.group_row_linear(w.long(), rows, 64), "float32, float16 or bfloat16"),
        (lambda: o.group_row_linear(w, torch.zeros(161, dtype=torch.uint8, device="cuda")[1:].view(10, 16), 64), "16-byte aligned"),
        (lambda: o.group_row_embedding(torch.zeros(161, dtype=torch.uint8, device="cuda")[1:].view(10, 16), t, 16, 64), "16-byte aligned"),
    ]
    for call, text in bad:
        with pytest.raises(RuntimeError, match=text):
            call()
    table = fa.GroupRowTable(10, 16, 64)
    for call in (lambda: table.assign_rows_from_float(torch.zeros(3, 8, device="cuda")), lambda: table.assign_rows_from_float(w, 1),
                 lambda: fa.GroupRowTable(4, 8, 48), lambda: fa.GroupRowTable(4, 12)):
        with pytest.raises(ValueError):
            call()


def test_group_row_table_keeps_to_the_device_of_its_rows():
    """A device without a number is the one that is current when the table is made, whichever is later."""
    import fbgemm_ascend_b200 as fa
    table = fa.GroupRowTable(10, 16, 64, device="cuda")
    assert table.device == table.rows.device and table.device.index is not None
    table.assign_rows_from_float(torch.ones(10, 16))             # of another device
    assert torch.equal(table.to_float(), torch.ones(10, 16, device="cuda"))


def test_group_row_table_names_what_it_cannot_take():
    import fbgemm_ascend_b200 as fa
    table = fa.GroupRowTable(10, 16, 64)
    for bad, text in ((torch.zeros(3, 16, dtype=torch.float64, device="cuda"), "float32, float16 or bfloat16"), (torch.zeros(3, 16, dtype=torch.int64), "float32, float16 or bfloat16"),
                      (torch.zeros((), device="cuda"), "do not fit"), (torch.zeros(16, device="cuda"), "do not fit"), (torch.zeros(1, 3, 16, device="cuda"), "do not fit")):
        with pytest.raises(ValueError, match=text):
            table.assign_rows_from_float(bad)
    assert not bool(table.rows.any())
