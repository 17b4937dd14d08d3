"""Selection products on the GPU against plain computations in 64 bits.

Tolerance.  A result is a sum of m products in float32 (float64 for float64 values), scaled, with
beta * out added, rounded once to its type.  With u the half step of the type that is summed in and
U that of the result, |got - exact| <= U |exact| + (1 + U) (m + 3) u S, S being the sum of the
absolute values of the terms: m products and additions in any order, alpha, beta and the last
addition (first order, Higham, Accuracy and Stability of Numerical Algorithms, section 3.1).  The
64-bit computation on the CPU has the same bound with u = 2^-53; it is added for float64 results.
Scalars in these tests are exact in float32.  float16 results below 2^-14 have a fixed half step
of 2^-25.
"""

import numpy as np
import pytest
import torch

import flagsparse_b200 as fs
from flagsparse_b200 import selection

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, params=["host module", "python"])
def way(request, monkeypatch):
    """Every test runs with the calls made by the C++ host module and by the Python code."""
    if request.param == "python":
        monkeypatch.setattr(selection, "_host", None)
    else:
        assert selection._host is not None
    return request.param

TYPES = [torch.float16, torch.bfloat16, torch.float32, torch.float64]
HALF_STEP = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24,
             torch.float64: 2.0**-53}
SMALLEST = {torch.float16: 2.0**-25, torch.bfloat16: 2.0**-134, torch.float32: 2.0**-150,
            torch.float64: 0.0}


def ids(v):
    return str(v).replace("torch.", "") if isinstance(v, torch.dtype) else None


def assert_close(got, exact, terms, m, acc=None):
    """`exact`, `terms` (S) float64 on the CPU; m: products per element (a number or a tensor)."""
    t = got.dtype
    u = HALF_STEP[torch.float64 if (acc or t) == torch.float64 else torch.float32]
    big = HALF_STEP[t]
    if t == torch.float64:
        u *= 2
    tol = big * exact.abs() + (1 + big) * (m + 3) * u * terms + SMALLEST[t]
    off = (got.double().cpu() - exact).abs()
    bad = ~(off <= tol)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} outside, worst off "
                           f"{float(off[bad].max())} where {float(tol[bad].max())} is allowed")


def randn(*shape, dtype=torch.float32, seed=0, pad=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    wide = torch.randn(*shape[:-1], shape[-1] + pad, device="cuda", generator=g)
    return wide.to(dtype)[..., :shape[-1]]


def cpu(t):
    return t.detach().double().cpu()


# ------------------------------------------------------------------------------------------------
# embedding lookup
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("n, vocab, dim, pad", [
    (1, 1, 1, 0), (1, 7, 4096, 0), (3, 10, 255, 0), (8, 100, 256, 0), (9, 100, 257, 1),
    (70, 33, 1032, 8), (700, 1000, 1001, 3), (2500, 500, 2048, 0)])
def test_embedding(dtype, n, vocab, dim, pad):
    table = randn(vocab, dim, dtype=dtype, seed=n, pad=pad)
    table[:, ::7] *= 0.0                                                # zeros of both signs
    rng = np.random.default_rng(n)
    tokens = torch.from_numpy(rng.integers(0, vocab, n))
    want = cpu(table)[tokens]
    for index in (torch.int32, torch.int64):
        tok = tokens.to(index).cuda()
        got = fs.flagsparse_embedding(tok, table)
        assert got.dtype == dtype and torch.equal(cpu(got), want)       # a copy, bit for bit
        assert torch.equal(torch.signbit(got).cpu(), torch.signbit(want))
        got = fs.flagsparse_embedding(tok, table, alpha=1.375)
        assert_close(got, 1.375 * want, 1.375 * want.abs(), 0)
    out = randn(n, dim, dtype=dtype, seed=5, pad=pad)
    before = cpu(out)
    got = fs.flagsparse_embedding(tok, table, alpha=-0.75, beta=0.5, out=out)
    assert got is out
    assert_close(out, -0.75 * want + 0.5 * before, 0.75 * want.abs() + 0.5 * before.abs(), 1)
    fs.check_selection_ids()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=ids)
@pytest.mark.parametrize("ignore", [-1, -100, 3, 2**40])
def test_embedding_masked_tokens(dtype, ignore):
    table = randn(11, 40, dtype=dtype)
    table[5] = float("inf")
    tokens = torch.tensor([[0, 3, 10], [1, 5, 2]], device="cuda")
    tokens[1, 2] = ignore
    got = fs.flagsparse_embedding(tokens, table, alpha=2.0, ignore_index=ignore)
    assert got.shape == (2, 3, 40)
    gone = tokens == ignore
    assert torch.equal(got[gone], torch.zeros_like(got[gone]))
    assert torch.equal(got[~gone], table[tokens[~gone]] * 2)
    out = torch.full_like(got, 3.0)
    fs.flagsparse_embedding(tokens, table, alpha=2.0, ignore_index=ignore, out=out, beta=1.0)
    assert torch.equal(out[gone], torch.full_like(out[gone], 3.0))
    all_gone = torch.full((4,), ignore, device="cuda")
    got = fs.flagsparse_embedding(all_gone, table, alpha=float("inf"), ignore_index=ignore)
    assert not got.any()
    fs.check_selection_ids()


def test_embedding_shapes_and_layouts():
    table = randn(50, 24)
    tokens = torch.randint(0, 50, (6, 5), device="cuda")
    want = table[tokens]
    assert torch.equal(fs.flagsparse_embedding(tokens, table), want)
    assert torch.equal(fs.flagsparse_embedding(tokens.t(), table), table[tokens.t()])
    assert torch.equal(fs.flagsparse_embedding(tokens[0, 0], table), want[0, 0])     # 0-d
    assert torch.equal(fs.flagsparse_embedding(tokens, table.t().contiguous().t()), want)
    assert torch.equal(fs.flagsparse_embedding(tokens, table[:, ::2]), want[..., ::2])
    assert torch.equal(fs.flagsparse_embedding(tokens, table[:1].expand(50, 24)),
                       table[:1].expand(50, 24)[tokens])
    assert torch.equal(fs.flagsparse_embedding(tokens, table.flip(0)[:, 1:]),
                       table.flip(0)[tokens][..., 1:])
    for out in (torch.full((6, 5, 24), float("nan"), device="cuda"),
                torch.full((5, 6, 24), float("nan"), device="cuda").transpose(0, 1),
                torch.full((6, 5, 31), float("nan"), device="cuda")[..., :24],
                torch.full((24, 6, 5), float("nan"), device="cuda").permute(1, 2, 0)):
        version = out._version
        assert fs.flagsparse_embedding(tokens, table, out=out) is out
        assert torch.equal(out, want) and out._version > version
    assert fs.flagsparse_embedding(tokens[:0], table).shape == (0, 5, 24)
    assert fs.flagsparse_embedding(tokens, table[:, :0]).shape == (6, 5, 0)
    empty = fs.flagsparse_embedding(torch.full((3,), -1, device="cuda"), table[:0],
                                    ignore_index=-1)
    assert empty.shape == (3, 24) and not empty.any()


def test_embedding_is_the_product_with_the_selection_matrix():
    """The same product by the SpMM of this package with S written out."""
    n, vocab, dim = 300, 90, 64
    for dtype in (torch.bfloat16, torch.float32, torch.float64):
        table, g = randn(vocab, dim, dtype=dtype), randn(n, dim, dtype=dtype, seed=1)
        tokens = torch.randint(0, vocab, (n,), device="cuda")
        ones = torch.ones(n, dtype=dtype, device="cuda")
        ptr = torch.arange(n + 1, device="cuda")
        y = fs.flagsparse_spmm_csr(ones, tokens, ptr, table, (n, vocab), alpha=1.5)
        assert torch.equal(fs.flagsparse_embedding(tokens, table, alpha=1.5), y)
        dense = fs.flagsparse_spmm_csr(ones, tokens, ptr, g, (n, vocab), op="trans")
        mine = fs.flagsparse_embedding_grad(tokens, g, vocab)
        terms = torch.zeros(vocab, dim, dtype=torch.float64).index_add_(0, tokens.cpu(),
                                                                       cpu(g).abs())
        assert_close(mine, cpu(dense), 2 * terms + cpu(dense).abs() * HALF_STEP[dtype] * 2**24, n)


def test_ids_outside_the_table_are_reported():
    table = randn(10, 16)
    tokens = torch.tensor([1, 10, 2, -1, 2**40], device="cuda")
    got = fs.flagsparse_embedding(tokens, table)
    with pytest.raises(IndexError, match="outside its range"):
        fs.check_selection_ids()
    fs.check_selection_ids()                                          # once
    assert torch.equal(got[[0, 2]], table[[1, 2]]) and not got[[1, 3, 4]].any()
    grad = fs.flagsparse_embedding_grad(tokens, torch.ones(5, 16, device="cuda"), 10)
    torch.cuda.synchronize()
    with pytest.raises(IndexError, match="outside its range"):        # by the next call
        fs.flagsparse_embedding(tokens[:1], table)
    assert float(grad.sum()) == 32 and float(grad[[1, 2]].sum()) == 32
    route = fs.prepare_token_route(torch.tensor([[0, 4], [-2, 1]], device="cuda"), 4)
    with pytest.raises(IndexError, match="outside its range"):
        fs.check_selection_ids("cuda")
    assert route.slots.tolist() == [[0, -1], [-1, 1]] and route.indptr.tolist() == [0, 1, 2, 2, 2]


def test_rows_behind_two_to_the_31_elements():
    vocab, dim = (1 << 31) // 4096 + 3, 4096
    table = torch.empty(vocab, dim, dtype=torch.float16, device="cuda")
    table[-3:] = randn(3, dim, dtype=torch.float16)
    keep = table[-3:].clone()
    tokens = torch.tensor([vocab - 1, vocab - 3, vocab - 1], device="cuda")
    assert torch.equal(fs.flagsparse_embedding(tokens, table), table[tokens])
    g = torch.ones(3, dim, dtype=torch.float16, device="cuda")
    fs.flagsparse_embedding_grad(tokens, g, vocab, out=table, beta=1.0)
    count = torch.tensor([1.0, 0.0, 2.0], device="cuda")
    assert torch.equal(table[-3:], (keep.float() + count[:, None]).half())
    fs.flagsparse_embedding_grad(tokens, g, vocab, out=table)
    assert torch.equal(table[-3:], count.half()[:, None].expand(3, dim))
    assert not table[:-3:1000].any() and not table[-4].any()


# ------------------------------------------------------------------------------------------------
# embedding gradient
# ------------------------------------------------------------------------------------------------
def plain_grad(tokens, g, vocab, alpha=1.0, out=None, beta=0.0, ignore=None):
    tokens, g = tokens.reshape(-1).long().cpu(), cpu(g).reshape(tokens.numel(), -1)
    if ignore is not None:
        g, tokens = g[tokens != ignore], tokens[tokens != ignore]
    total = torch.zeros(vocab, g.shape[1], dtype=torch.float64).index_add_(0, tokens, g)
    terms = torch.zeros_like(total).index_add_(0, tokens, g.abs())
    m = torch.bincount(tokens, minlength=vocab)[:, None].double()
    total, terms = alpha * total, abs(alpha) * terms
    if beta:
        total, terms = total + beta * out, terms + abs(beta) * out.abs()
    return total, terms, m


def runs(*lengths):
    """Tokens 0, 1, 2, ... in runs of these lengths, in a mixed order."""
    tokens = torch.repeat_interleave(torch.arange(len(lengths)), torch.tensor(lengths))
    return tokens[torch.from_numpy(np.random.default_rng(0).permutation(tokens.numel()))]


PATTERNS = {
    "one": (torch.zeros(1, dtype=torch.long), 1),
    "one of many": (torch.tensor([40]), 70),
    "same": (torch.zeros(1000, dtype=torch.long) + 2, 5),
    "tiles": (runs(31, 1, 32, 33, 31, 64, 1, 63, 65, 62, 96, 97, 95, 2, 300), 20),
    "whole tiles": (runs(32, 32, 64, 96, 32, 1), 6),
    "short tiles": (runs(7, 1, 8, 9, 7, 15, 16, 17, 1, 24, 23, 25, 2, 40), 20),
    "half tiles": (runs(15, 1, 16, 17, 15, 31, 32, 33, 1, 47, 48, 49, 2, 80), 20),
    "long": (runs(1, 4000, 3, 2500, 33), 7),
    "even": (torch.from_numpy(np.random.default_rng(1).integers(0, 900, 2000)), 900),
    "one chunk": (torch.from_numpy(np.random.default_rng(2).integers(0, 5000, 4096)), 5000),
    "few": (torch.from_numpy(np.random.default_rng(5).zipf(1.2, 256) % 30000), 30000),
    "not few": (torch.from_numpy(np.random.default_rng(5).zipf(1.2, 257) % 3000), 3000),
    "few and same": (torch.full((250,), 3), 4),
    "team of one": (torch.from_numpy(np.random.default_rng(5).zipf(1.3, 1024) % 30000), 30000),
    "team": (torch.from_numpy(np.random.default_rng(5).zipf(1.3, 1025) % 30000), 30000),
    "full team": (torch.from_numpy(np.random.default_rng(6).zipf(1.3, 8192) % 30000), 30000),
    "no team": (torch.from_numpy(np.random.default_rng(7).zipf(1.3, 8193) % 30000), 30000),
    "two passes": (torch.from_numpy(np.random.default_rng(3).zipf(1.2, 9001) % 40000), 40000),
    "many chunks": (torch.from_numpy(np.random.default_rng(4).zipf(1.1, 140001) % 3000), 3000),
}


@pytest.mark.parametrize("pattern", PATTERNS)
@pytest.mark.parametrize("dtype, out_dtype, dim", [
    (torch.float32, torch.float32, 8), (torch.float32, torch.float32, 33),
    (torch.bfloat16, torch.bfloat16, 264), (torch.bfloat16, torch.float32, 40),
    (torch.float16, torch.float16, 7), (torch.float16, torch.float32, 257),
    (torch.bfloat16, torch.bfloat16, 4104), (torch.float32, torch.float32, 2052),
    (torch.float64, torch.float64, 12), (torch.float64, torch.float64, 5)], ids=ids)
def test_embedding_grad(pattern, dtype, out_dtype, dim):
    tokens, vocab = PATTERNS[pattern]
    n = tokens.numel()
    if n * dim > 1 << 24 or vocab * dim > 1 << 24:
        dim = 392                                    # the wide rows: what the CPU sums in a second
    g = randn(n, dim, dtype=dtype, seed=n)
    tok = tokens.cuda()
    got = fs.flagsparse_embedding_grad(tok, g, vocab, out_dtype=out_dtype)
    assert got.dtype == out_dtype and got.shape == (vocab, dim)
    total, terms, m = plain_grad(tokens, g, vocab)
    assert_close(got, total, terms, m, acc=dtype)
    again = fs.flagsparse_embedding_grad(tok.int(), g, vocab, out_dtype=out_dtype)
    assert torch.equal(again, got)                                    # one order of the sums
    # into a strided out: added (other rows untouched), scaled, and written over
    named = torch.bincount(tokens, minlength=vocab) > 0
    for alpha, beta in ((1.5, 1.0), (0.75, 0.5), (1.0, 0.0)):
        out = randn(vocab, dim, dtype=out_dtype, seed=2, pad=3)
        if beta == 0.0:
            out.fill_(float("nan"))
        elif beta == 1.0:
            out[~named.cuda()] = float("nan")
        before = cpu(out)
        assert fs.flagsparse_embedding_grad(tok, g, vocab, alpha=alpha, beta=beta, out=out) is out
        total, terms, m = plain_grad(tokens, g, vocab, alpha, before, beta)
        if beta == 1.0:
            assert torch.isnan(out[~named.cuda()]).all()
            total, terms, m, out = total[named], terms[named], m[named], out[named.cuda()]
        assert_close(out, total, terms, m, acc=dtype)
    fs.check_selection_ids()


@pytest.mark.parametrize("n", [5, 3000, 20000])
@pytest.mark.parametrize("ignore", [-1, 7, 10**12])
def test_embedding_grad_masked_tokens(n, ignore):
    vocab, dim = 400, 48
    tokens = torch.randint(0, vocab, (n,), device="cuda")
    tokens[torch.rand(n, device="cuda") < 0.4] = ignore
    g = randn(n, dim, dtype=torch.bfloat16)
    g[tokens == ignore] = float("nan")
    got = fs.flagsparse_embedding_grad(tokens, g, vocab, ignore_index=ignore)
    total, terms, m = plain_grad(tokens, g, vocab, ignore=ignore)
    assert_close(got, total, terms, m)
    tokens.fill_(ignore)
    got = fs.flagsparse_embedding_grad(tokens, g, vocab, ignore_index=ignore)
    assert not got.any() and not got.isnan().any()
    out = torch.full((vocab, dim), 4.0, device="cuda")
    fs.flagsparse_embedding_grad(tokens, g, vocab, ignore_index=ignore, out=out, beta=0.5)
    assert torch.equal(out, torch.full_like(out, 2.0))
    fs.check_selection_ids()


def test_embedding_grad_three_digit_vocabulary():
    """A vocabulary of more than 2^22 rows is sorted in three passes."""
    vocab = (1 << 22) + 1000
    for n in (100, 5000, 9000, 70000):
        tokens = torch.randint(0, vocab, (n,), device="cuda")
        tokens[:3] = torch.tensor([vocab - 1, 0, vocab - 1])
        g = randn(n, 4)
        got = fs.flagsparse_embedding_grad(tokens, g, vocab)
        want = torch.zeros(vocab, 4, dtype=torch.float64, device="cuda")
        want.index_add_(0, tokens, g.double())
        assert (got - want).abs().max() < 1e-5       # at most a few rows of a token, each below 6
        assert torch.equal(got != 0, want != 0)
    fs.check_selection_ids()


def test_embedding_grad_shapes():
    g = randn(4, 6, 10)
    tokens = torch.randint(0, 9, (4, 6), device="cuda")
    want = fs.flagsparse_embedding_grad(tokens.reshape(-1), g.reshape(24, 10), 9)
    assert torch.equal(fs.flagsparse_embedding_grad(tokens, g, 9), want)
    turned = g.permute(2, 0, 1).contiguous().permute(1, 2, 0)
    assert torch.equal(fs.flagsparse_embedding_grad(tokens, turned, 9), want)
    assert torch.equal(fs.flagsparse_embedding_grad(tokens.t(), g.transpose(0, 1), 9),
                       fs.flagsparse_embedding_grad(tokens.t().contiguous(),
                                                    g.transpose(0, 1).contiguous(), 9))
    spread = g[:, :, :1].expand(4, 6, 10)
    assert torch.equal(fs.flagsparse_embedding_grad(tokens, spread, 9),
                       fs.flagsparse_embedding_grad(tokens, spread.contiguous(), 9))
    cols = torch.full((10, 9), 1.0, device="cuda").t()
    fs.flagsparse_embedding_grad(tokens, g, 9, out=cols, beta=1.0)
    assert_close(cols, cpu(want) + 1.0, cpu(want).abs() * 24 + 1.0, 2)
    none = fs.flagsparse_embedding_grad(tokens[:0], g[:0], 9)
    assert none.shape == (9, 10) and not none.any()
    assert fs.flagsparse_embedding_grad(tokens, g[..., :0], 9).shape == (9, 0)
    gone = torch.full((4, 6), -1, device="cuda")
    assert fs.flagsparse_embedding_grad(gone, g, 0, ignore_index=-1).shape == (0, 10)


# ------------------------------------------------------------------------------------------------
# token route
# ------------------------------------------------------------------------------------------------
def random_experts(n, k, n_experts, drop=0.0, seed=0, index=torch.int64):
    rng = np.random.default_rng(seed)
    skew = rng.random(n_experts) ** 4 + 1e-3
    e = rng.choice(n_experts, size=(n, k), p=skew / skew.sum()) if n * k else np.zeros((n, k))
    e = np.where(rng.random((n, k)) < drop, -1, e)
    return torch.from_numpy(e).to(index).cuda()


def plain_route(experts, n_experts):
    flat = experts.reshape(-1).long().cpu()
    key = torch.where(flat < 0, n_experts, flat)
    order = torch.sort(key, stable=True)[1]
    slots = torch.empty_like(order)
    slots[order] = torch.arange(flat.numel())
    slots[flat < 0] = -1
    indptr = torch.zeros(n_experts + 1, dtype=torch.long)
    indptr[1:] = torch.bincount(key, minlength=n_experts + 1)[:n_experts].cumsum(0)
    return slots.reshape(experts.shape), indptr, order // max(experts.shape[1], 1)


ROUTES = [(1, 1, 1, 0.0), (1024, 1, 9, 0.1), (1025, 1, 9, 0.1), (1024, 4, 500, 0.0),
          (8192, 1, 70, 0.2),
          (8193, 1, 64, 0.2), (8192, 2, 2047, 0.0), (16385, 2, 2047, 0.1), (1, 8, 8, 0.0),
          (7, 3, 5, 0.3), (64, 8, 256, 0.0), (100, 2, 2047, 0.1),
          (513, 8, 3, 0.0), (2100, 2, 64, 0.05), (16384, 1, 128, 0.0), (17000, 8, 60, 0.1),
          (50, 40, 64, 0.0), (6, 4, 10, 1.0), (0, 4, 10, 0.0), (5, 0, 10, 0.0)]


@pytest.mark.parametrize("n, k, n_experts, drop", ROUTES)
def test_route_plan(n, k, n_experts, drop):
    for index in (torch.int32, torch.int64):
        experts = random_experts(n, k, n_experts, drop, seed=n, index=index)
        r = fs.prepare_token_route(experts, n_experts)
        slots, indptr, indices = plain_route(experts, n_experts)
        held = int(indptr[-1])
        assert torch.equal(r.slots.cpu().long(), slots)
        assert torch.equal(r.indptr.cpu().long(), indptr)
        assert torch.equal(r.indices.cpu().long()[:held], indices[:held])
        assert (r.n_tokens, r.k, r.n_rows) == (n, k, n * k)
    turned = random_experts(k, n, n_experts, drop, seed=1).t()
    assert torch.equal(fs.prepare_token_route(turned, n_experts).slots,
                       fs.prepare_token_route(turned.contiguous(), n_experts).slots)
    fs.check_selection_ids()


def test_route_is_a_csr_matrix():
    """(indptr, indices) multiplies as the experts x tokens matrix."""
    experts = random_experts(200, 3, 9, 0.2)
    r, x = fs.prepare_token_route(experts, 9), randn(200, 8, dtype=torch.float64)
    held = int(r.indptr[-1])
    ones = torch.ones(held, dtype=torch.float64, device="cuda")
    per_expert = fs.flagsparse_spmm_csr(ones, r.indices[:held].contiguous(), r.indptr, x, (9, 200))
    rows = fs.flagsparse_token_dispatch(x, r)
    for e in range(9):
        a, b = int(r.indptr[e]), int(r.indptr[e + 1])
        assert torch.allclose(per_expert[e], rows[a:b].sum(0), rtol=0, atol=1e-12)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("n, k, n_experts, drop, dim, pad", [
    (1, 1, 1, 0.0, 1, 0), (1, 8, 8, 0.0, 4096, 0), (7, 3, 5, 0.3, 255, 0), (64, 8, 256, 0.0, 264, 8),
    (513, 8, 3, 0.0, 40, 0), (1100, 2, 64, 0.05, 1025, 2), (50, 37, 64, 0.1, 96, 1),
    (6, 4, 10, 1.0, 24, 0), (300, 5, 16, 0.5, 520, 0)])
def test_route_operators(dtype, n, k, n_experts, drop, dim, pad):
    experts = random_experts(n, k, n_experts, drop, seed=dim)
    r = fs.prepare_token_route(experts, n_experts)
    slots, indptr, _ = plain_route(experts, n_experts)
    held, live = int(indptr[-1]), slots >= 0
    place = torch.where(live, slots, 0)
    nan = float("nan")

    # there
    x = randn(n, dim, dtype=dtype, seed=1, pad=pad)
    rows = fs.flagsparse_token_dispatch(x, r)
    want = torch.zeros(n * k, dim, dtype=torch.float64)
    want[slots[live]] = cpu(x)[:, None].expand(n, k, dim)[live]
    assert torch.equal(cpu(rows), want)
    out = torch.full((n * k, dim + pad), nan, dtype=dtype, device="cuda")[:, :dim]
    assert fs.flagsparse_token_dispatch(x, r, out=out) is out and torch.equal(out, rows)

    # back, with each kind of weights; rows that belong to nobody are never read
    y = randn(n * k, dim, dtype=dtype, seed=2, pad=pad)
    y[held:] = nan
    picked = torch.where(live[:, :, None], cpu(y)[place], 0.0)
    grad = randn(n, dim, dtype=dtype, seed=3, pad=pad)
    for weights in (None, randn(n, k, dtype=dtype, seed=4), randn(n, k, seed=4)):
        if weights is not None:
            weights[experts < 0] = nan
        w = torch.ones(n, k, dtype=torch.float64) if weights is None else cpu(weights)
        w = torch.where(live, w, 0.0)
        total, terms = (w[..., None] * picked).sum(1), (w[..., None] * picked).abs().sum(1)
        got = fs.flagsparse_token_combine(y, r, weights)
        assert got.dtype == dtype and got.shape == (n, dim)
        assert_close(got, total, terms, 2 * k)
        out = randn(n, dim, dtype=dtype, seed=5, pad=pad)
        before = cpu(out)
        fs.flagsparse_token_combine(y, r, weights, alpha=1.5, beta=0.5, out=out)
        assert_close(out, 1.5 * total + 0.5 * before, 1.5 * terms + 0.5 * before.abs(), 2 * k)
        gy, gw = fs.flagsparse_token_combine_grad(grad, y, r, weights, alpha=0.75)
        want = torch.zeros(n * k, dim, dtype=torch.float64)
        want[slots[live]] = (0.75 * w[..., None] * cpu(grad)[:, None])[live]
        assert_close(gy, want, want.abs(), 1)
        if weights is None:
            assert gw is None
            only, _ = fs.flagsparse_token_combine_grad(grad, None, r, alpha=0.75)
            assert torch.equal(only, gy)
        else:
            assert gw.dtype == weights.dtype
            dots = 0.75 * picked * cpu(grad)[:, None]
            assert_close(gw, dots.sum(2), dots.abs().sum(2), 2 * dim, acc=dtype)
            assert not gw[experts < 0].any()

    # the gradient of the way there
    got = fs.flagsparse_token_dispatch_grad(y, r)
    assert_close(got, picked.sum(1), picked.abs().sum(1), k)
    out = randn(n, dim, dtype=dtype, seed=6)
    before = cpu(out)
    fs.flagsparse_token_dispatch_grad(y, r, out=out, beta=1.0)
    assert_close(out, picked.sum(1) + before, picked.abs().sum(1) + before.abs(), k)
    fs.check_selection_ids()


def test_route_operators_empty():
    for n, k in ((0, 4), (5, 0), (0, 0)):
        r = fs.prepare_token_route(torch.zeros(n, k, dtype=torch.int64, device="cuda"), 3)
        assert r.indptr.tolist() == [0, 0, 0, 0]
        assert fs.flagsparse_token_dispatch(randn(n, 8), r).shape == (n * k, 8)
        out = fs.flagsparse_token_combine(randn(n * k, 8), r, randn(n, k))
        assert out.shape == (n, 8) and not out.any()
        kept = torch.full((n, 8), 2.0, device="cuda")
        fs.flagsparse_token_combine(randn(n * k, 8), r, out=kept, beta=0.5)
        assert torch.equal(kept, torch.ones_like(kept))
        gy, gw = fs.flagsparse_token_combine_grad(randn(n, 8), randn(n * k, 8), r, randn(n, k))
        assert gy.shape == (n * k, 8) and gw.shape == (n, k)
    r = fs.prepare_token_route(torch.zeros(4, 2, dtype=torch.int64, device="cuda"), 1)
    assert fs.flagsparse_token_dispatch(randn(4, 0), r).shape == (8, 0)
    gy, gw = fs.flagsparse_token_combine_grad(randn(4, 0), randn(8, 0), r, randn(4, 2))
    assert gy.shape == (8, 0) and not gw.any()


def test_route_layouts():
    r = fs.prepare_token_route(random_experts(30, 3, 7, 0.1), 7)
    x, y, w = randn(30, 20), randn(90, 20, seed=1), randn(30, 3, seed=2)
    rows, out = fs.flagsparse_token_dispatch(x, r), fs.flagsparse_token_combine(y, r, w)
    turn = lambda t: t.t().contiguous().t()  # noqa: E731
    assert torch.equal(fs.flagsparse_token_dispatch(turn(x), r), rows)
    assert torch.equal(fs.flagsparse_token_combine(turn(y), r, turn(w)), out)
    there, back = turn(torch.zeros_like(rows)), turn(torch.zeros_like(out))
    assert fs.flagsparse_token_dispatch(x, r, out=there) is there and torch.equal(there, rows)
    assert fs.flagsparse_token_combine(y, r, w, out=back) is back and torch.equal(back, out)
    g = randn(30, 1).expand(30, 20)
    for a, b in zip(fs.flagsparse_token_combine_grad(g, turn(y), r, turn(w)),
                    fs.flagsparse_token_combine_grad(g.contiguous(), y, r, w)):
        assert torch.equal(a, b)


def test_route_rows_behind_two_to_the_31_elements():
    n, k, dim = 66000, 8, 4096
    experts = torch.zeros(n, k, dtype=torch.int32, device="cuda")
    experts[-1] = torch.arange(1, 9)
    r = fs.prepare_token_route(experts, 9)
    x = torch.zeros(n, dim, dtype=torch.float16, device="cuda")
    x[-1] = randn(1, dim, dtype=torch.float16)
    rows = fs.flagsparse_token_dispatch(x, r)
    assert rows.numel() > 2**31 and torch.equal(rows[-8:], x[-1:].expand(8, dim))
    assert not rows[-9].any()
    out = fs.flagsparse_token_combine(rows, r)
    assert torch.equal(out[-1], x[-1] * 8) and not out[:-1].any()
    del out
    gy, gw = fs.flagsparse_token_combine_grad(x, rows, r, torch.ones(n, k, device="cuda"))
    assert torch.equal(gy[-8:], x[-1:].expand(8, dim))
    dot = float((cpu(x[-1]) ** 2).sum())
    assert (gw[-1].double().cpu() - dot).abs().max() <= 2 * dim * 2.0**-24 * dot


# ------------------------------------------------------------------------------------------------
# gradients, streams, graphs
# ------------------------------------------------------------------------------------------------
def test_gradients_against_differences():
    """Central differences in float64 (torch.autograd.gradcheck)."""
    torch.manual_seed(0)
    f64 = dict(dtype=torch.float64, device="cuda")
    tokens = torch.tensor([[1, 4, 1], [-1, 0, 4]], device="cuda")
    table = torch.randn(6, 5, **f64, requires_grad=True)
    assert torch.autograd.gradcheck(
        lambda t: fs.flagsparse_embedding(tokens, t, alpha=1.5, ignore_index=-1), (table,))
    r = fs.prepare_token_route(torch.tensor([[0, 2], [2, -1], [1, 1], [-1, -1]], device="cuda"), 3)
    x = torch.randn(4, 3, **f64, requires_grad=True)
    assert torch.autograd.gradcheck(lambda v: fs.flagsparse_token_dispatch(v, r), (x,))
    y = torch.randn(8, 3, **f64, requires_grad=True)
    w = torch.randn(4, 2, **f64, requires_grad=True)
    combine = lambda *a: fs.flagsparse_token_combine(a[0], r, a[1], alpha=0.5)  # noqa: E731
    assert torch.autograd.gradcheck(combine, (y, w))
    assert torch.autograd.gradcheck(combine, (y.detach(), w))
    assert torch.autograd.gradcheck(combine, (y, w.detach()))
    assert torch.autograd.gradcheck(lambda v: fs.flagsparse_token_combine(v, r), (y,))


def experts_layer(x, experts, w, mats, own):
    """Tokens through the experts they are sent to: by the route, or expert by expert."""
    n, k = experts.shape
    if own:
        r = fs.prepare_token_route(experts, len(mats))
        rows = fs.flagsparse_token_dispatch(x, r)
        at = r.indptr.tolist()
        parts = [rows[a:b] @ m for a, b, m in zip(at, at[1:], mats)]
        parts.append(rows[at[-1]:])                  # rows that belong to nobody
        return fs.flagsparse_token_combine(torch.cat(parts), r, w)
    out = torch.zeros_like(x)
    for e, m in enumerate(mats):
        share = torch.where(experts == e, w, 0).sum(1, keepdim=True)
        out = out + share.to(x.dtype) * (x @ m)
    return out


@pytest.mark.parametrize("dtype, tol", [(torch.float64, 1e-12), (torch.float32, 2e-5)], ids=ids)
def test_embedding_and_experts_together(dtype, tol):
    """Lookup, route, experts and back in one training step, gradients of everything.

    float32: sums of at most 48 * 3 products per element and three such steps in a row: the norm
    of the error stays below 3 * 144 * 2^-24 = 2.6e-5 of terms that do not cancel by more than the
    square root of their number, 12: 2.6e-5 / 12 * 2 (both sides) = 4.3e-6, held to 2e-5."""
    torch.manual_seed(1)
    vocab, dim, n, k, n_experts = 90, 48, 200, 3, 7
    tokens = torch.randint(0, vocab, (n,), device="cuda")
    tokens[::9] = -1
    experts = random_experts(n, k, n_experts, 0.1)
    table = torch.randn(vocab, dim, dtype=torch.float64, device="cuda")
    score = torch.randn(n, k, dtype=torch.float64, device="cuda")
    mats = [torch.randn(dim, dim, dtype=torch.float64, device="cuda") / dim**0.5
            for _ in range(n_experts)]
    target = torch.randn(n, dim, dtype=torch.float64, device="cuda")
    results = []
    for own, t in ((True, dtype), (False, torch.float64)):
        leaves = [v.to(t).requires_grad_() for v in (table, score, *mats)]
        tab, sc, ms = leaves[0], leaves[1], leaves[2:]
        if own:
            x = fs.flagsparse_embedding(tokens, tab, alpha=2.0, ignore_index=-1)
        else:
            x = torch.where((tokens >= 0)[:, None], tab[tokens.clamp(min=0)] * 2.0, 0)
        w = torch.softmax(sc, dim=1)
        out = x + experts_layer(x, experts, w, ms, own)
        (out * target.to(t)).sum().backward()
        results.append([out.detach(), *(v.grad for v in leaves)])
    for a, b in zip(*results):
        assert torch.linalg.norm(a.double() - b) <= tol * torch.linalg.norm(b)
    fs.check_selection_ids()


def test_only_what_needs_a_gradient_is_recorded():
    tokens, table = torch.tensor([1, 2], device="cuda"), randn(4, 8).requires_grad_()
    with torch.no_grad():
        assert not fs.flagsparse_embedding(tokens, table).requires_grad
        out = torch.zeros(2, 8, device="cuda")
        fs.flagsparse_embedding(tokens, table, out=out)
    y = fs.flagsparse_embedding(tokens, table)
    y.sum().backward()                               # an expanded gradient
    assert torch.equal(table.grad, torch.tensor([0., 1, 1, 0], device="cuda")[:, None].expand(4, 8))
    y = fs.flagsparse_embedding(tokens, table)
    g, = torch.autograd.grad(y.sum(), table, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()                           # once differentiable


def test_scalars_outputs_and_inference_tensors():
    table, tokens = randn(20, 16), torch.randint(0, 20, (9,), device="cuda")
    for alpha in (2, np.float32(2), np.float64(2), torch.tensor(2.0), torch.tensor(2, device="cuda"),
                  2 + 0j):
        assert torch.equal(fs.flagsparse_embedding(tokens, table, alpha=alpha), table[tokens] * 2)
    with torch.inference_mode():
        frozen, grad = table.clone(), torch.zeros(20, 16, device="cuda")
        y = fs.flagsparse_embedding(tokens, frozen)
        fs.flagsparse_embedding_grad(tokens, y, 20, out=grad, beta=1.0)
    fs.flagsparse_embedding_grad(tokens, y, 20, out=grad, beta=1.0)
    assert torch.equal(y, table[tokens])
    assert torch.equal(grad, 2 * fs.flagsparse_embedding_grad(tokens, y, 20))
    watched = torch.zeros(20, 16, device="cuda")
    version = watched._version
    fs.flagsparse_embedding_grad(tokens, y, 20, out=watched, beta=1.0)
    assert watched._version > version
    both = randn(20, 32)
    with pytest.raises(ValueError, match="must not overlap"):
        fs.flagsparse_embedding_grad(torch.arange(20, device="cuda"), both[:, :20], 20,
                                     out=both[:, 12:], beta=1.0)
    want = fs.flagsparse_embedding_grad(torch.arange(20, device="cuda"), both[:, :16].clone(), 20)
    fs.flagsparse_embedding_grad(torch.arange(20, device="cuda"), both[:, :16], 20,
                                 out=both[:, 16:])
    assert torch.equal(both[:, 16:], want)


def test_other_streams_and_a_freed_route():
    n, k, dim = 4000, 4, 512
    experts = random_experts(n, k, 16)
    x = randn(n, dim, dtype=torch.bfloat16)
    r = fs.prepare_token_route(experts, 16)
    want = fs.flagsparse_token_dispatch(x, r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        rows = fs.flagsparse_token_dispatch(x, r)
        back = fs.flagsparse_token_combine(rows, r)
    del r                                            # its memory stays until `side` has read it
    other = [torch.zeros(n * k, dtype=torch.int32, device="cuda") for _ in range(8)]
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(rows, want) and len(other) == 8
    assert torch.equal(back, (x.float() * 4).bfloat16())


def test_kernels_wait_for_the_ones_before_them():
    """Kernels are put in place while their inputs are still being written: long ones in front of
    short ones, and inputs that change between calls."""
    n, k, dim, vocab = 8192, 8, 1024, 9000
    experts = random_experts(n, k, 32)
    x = torch.zeros(n, dim, dtype=torch.bfloat16, device="cuda")
    tokens = torch.randperm(vocab, device="cuda")[:n]
    table = torch.zeros(vocab, dim, dtype=torch.bfloat16, device="cuda")
    results = []
    for turn in range(1, 9):
        x.fill_(turn)
        table.fill_(2 * turn)
        r = fs.prepare_token_route(experts, 32)
        rows = fs.flagsparse_token_dispatch(x, r)
        out = fs.flagsparse_token_combine(rows, r)
        gy, gw = fs.flagsparse_token_combine_grad(out, rows, r, torch.ones(n, k, device="cuda"))
        picked = fs.flagsparse_embedding(tokens, table)
        grad = fs.flagsparse_embedding_grad(tokens, picked, vocab)
        results.append((turn, out, gy, gw, picked, grad))
        experts = experts.roll(1, 0)
    for turn, out, gy, gw, picked, grad in results:
        assert torch.equal(out, torch.full_like(out, 8 * turn))
        assert torch.equal(gy, torch.full_like(gy, 8 * turn))
        assert torch.equal(gw, torch.full_like(gw, 8 * turn * turn * dim))
        assert torch.equal(picked, torch.full_like(picked, 2 * turn))
        want = torch.zeros_like(grad)
        want[tokens] = 2 * turn
        assert torch.equal(grad, want)


def test_random_calls():
    """Sizes, types, layouts and masks at random (the calls above, held to the same bounds)."""
    import random
    for seed in range(150):
        rng = random.Random(seed)
        torch.manual_seed(seed)
        dtype, index = rng.choice(TYPES), rng.choice([torch.int32, torch.int64])
        dim = rng.choice([1, 2, 7, 8, 33, 64, 100, 255, 256, 257, 512, 513, 1030])

        def matrix(rows):
            pad, off = rng.choice([0, 0, 1, 3, 8]), rng.choice([0, 0, 1, 2, 8])
            return torch.randn(rows, off + dim + pad, device="cuda").to(dtype)[:, off:off + dim]

        if seed % 2:
            n, vocab = int(2**rng.uniform(0, 14)), int(2**rng.uniform(0, 12))
            tokens = (torch.rand(n, device="cuda")**rng.choice([1, 4, 20]) * vocab).to(index)
            ignore = rng.choice([None, rng.randrange(vocab)])
            g = matrix(n)
            got = fs.flagsparse_embedding_grad(tokens, g, vocab, alpha=0.5, ignore_index=ignore)
            total, terms, m = plain_grad(tokens, g, vocab, 0.5, ignore=ignore)
            assert_close(got, total, terms, m)
            continue
        n, k, n_experts = int(2**rng.uniform(0, 10)), rng.choice([1, 2, 3, 8, 33]), 64
        experts = random_experts(n, k, n_experts, rng.choice([0.0, 0.2, 1.0]), seed, index)
        r = fs.prepare_token_route(experts, n_experts)
        slots, indptr, _ = plain_route(experts, n_experts)
        assert torch.equal(r.slots.cpu().long(), slots)
        live, held = slots >= 0, int(indptr[-1])
        y, w = matrix(n * k), torch.randn(n, k, device="cuda")
        y[held:] = float("nan")
        picked = torch.where(live[..., None], cpu(y)[torch.where(live, slots, 0)], 0.0)
        parts = torch.where(live, cpu(w), 0.0)[..., None] * picked
        assert_close(fs.flagsparse_token_combine(y, r, w), parts.sum(1), parts.abs().sum(1), 2 * k)
        assert_close(fs.flagsparse_token_dispatch_grad(y, r), picked.sum(1), picked.abs().sum(1), k)
    fs.check_selection_ids()


def test_captured_and_replayed_with_new_inputs():
    """Two graphs of the same calls, replayed in turn on changed inputs, keep their own
    workspaces; ids outside their range are reported after a replay."""
    n, vocab, dim, k, n_experts = 6000, 3000, 256, 4, 32
    graphs = []
    for seed in range(2):
        tokens = torch.zeros(n, dtype=torch.int64, device="cuda")
        experts = torch.zeros(n, k, dtype=torch.int64, device="cuda")
        table = randn(vocab, dim, dtype=torch.bfloat16, seed=seed)
        weights = randn(n, k, seed=seed)

        def step(tokens=tokens, experts=experts, table=table, weights=weights):
            x = fs.flagsparse_embedding(tokens, table)
            r = fs.prepare_token_route(experts, n_experts)
            y = fs.flagsparse_token_dispatch(x, r)
            out = fs.flagsparse_token_combine(y, r, weights)
            gy, gw = fs.flagsparse_token_combine_grad(out, y, r, weights)
            gx = fs.flagsparse_token_dispatch_grad(gy, r)
            return (r.slots, r.indptr, y, out, gy, gw, gx,
                    fs.flagsparse_embedding_grad(tokens, gx, vocab, out_dtype=torch.float32))

        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        graphs.append((graph, tokens, experts, held, step))
    for turn in range(3):
        for seed, (graph, tokens, experts, held, step) in enumerate(graphs):
            rng = np.random.default_rng(10 * turn + seed)
            tokens.copy_(torch.from_numpy(rng.zipf(1.3, n) % vocab))
            experts.copy_(torch.from_numpy(rng.integers(-1, n_experts, (n, k))))
        for graph, *_ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for graph, tokens, experts, held, step in graphs:
            for a, b in zip(held, step()):
                assert torch.equal(a, b)
    fs.check_selection_ids()
    graphs[0][1][5] = vocab
    graphs[0][0].replay()
    with pytest.raises(IndexError):
        fs.check_selection_ids()


def test_capture_of_differentiable_calls_is_refused():
    tokens, table = torch.tensor([1, 2], device="cuda"), randn(4, 8).requires_grad_()
    r = fs.prepare_token_route(torch.tensor([[0, 1]], device="cuda"), 2)
    x, y = randn(1, 8).requires_grad_(), randn(2, 8).requires_grad_()
    alive = fs.flagsparse_embedding(tokens, table)   # an eager graph of the same leaf
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        graph.capture_begin()
        for call in (lambda: fs.flagsparse_embedding(tokens, table),
                     lambda: fs.flagsparse_token_dispatch(x, r),
                     lambda: fs.flagsparse_token_combine(y, r)):
            with pytest.raises(RuntimeError, match="not recorded inside a CUDA graph capture"):
                call()
        with torch.no_grad():
            held = fs.flagsparse_embedding(tokens, table)
        graph.capture_end()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(held, table.detach()[tokens])
    alive.sum().backward()
    assert float(table.grad.sum()) == 16


def test_first_call_of_a_process_may_be_captured():
    """The word the kernels report to is made by the first call, also inside a capture."""
    import subprocess
    import sys
    from conftest import ROOT
    code = """
import torch, flagsparse_b200 as fs
table, tokens = torch.ones(4, 8, device="cuda"), torch.tensor([1, 3], device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = fs.flagsparse_embedding(tokens, table, alpha=2.0)
graph.replay(); torch.cuda.synchronize()
assert float(out.sum()) == 32
tokens[0] = 9
graph.replay()
try:
    fs.check_selection_ids()
except IndexError:
    print("reported")
"""
    res = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True,
                         timeout=300)
    assert res.returncode == 0 and "reported" in res.stdout, res.stdout[-500:] + res.stderr[-1500:]


def test_calls_from_two_threads():
    import threading
    n, vocab, dim = 20000, 4000, 128
    g = randn(n, dim)
    tokens = [torch.randint(0, vocab, (n,), device="cuda") for _ in range(2)]
    want = [fs.flagsparse_embedding_grad(t, g, vocab) for t in tokens]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                if not torch.equal(fs.flagsparse_embedding_grad(tokens[i], g, vocab), want[i]):
                    wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
