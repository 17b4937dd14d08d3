"""Selection products on the GPU: calls beside the usual one.  What has to be refused, what a mask
leaves, views of other tensors, the interpreter during a launch, and the forms of the gradient and
of the combine that take 16 bytes at a time.  Bounds as in test_selection_gpu.py."""

import numpy as np
import pytest
import torch

import flagsparse_b200 as fs
from flagsparse_b200 import selection
from test_selection_gpu import (PATTERNS, TYPES, assert_close, cpu, ids, plain_grad, plain_route,
                                randn, random_experts)

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, params=["host module", "python"])
def way(request, monkeypatch):
    """Every test runs with the calls made by the C++ host module and by the Python code."""
    if request.param == "python":
        monkeypatch.setattr(selection, "_host", None)
    else:
        assert selection._host.embedding is not selection._not_here      # it is built
    return request.param


def test_tangents_are_refused():
    """A result without the tangent of its input would stand for a derivative of zero."""
    import torch.autograd.forward_ad as forward
    tokens = torch.tensor([1, 3, 3], device="cuda")
    r = fs.prepare_token_route(torch.tensor([[0, 1], [1, -1], [1, 0]], device="cuda"), 2)
    table, x, y, w = randn(4, 8), randn(3, 8, seed=1), randn(6, 8, seed=2), randn(3, 2, seed=3)
    fs.flagsparse_embedding(tokens, table)                   # (the usual call is bound by now)
    with forward.dual_level():
        dual = lambda t: forward.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: fs.flagsparse_embedding(tokens, dual(table)),
                     lambda: fs.flagsparse_embedding(tokens, dual(torch.nn.Parameter(table))),
                     lambda: fs.flagsparse_embedding_grad(tokens, dual(x), 4),
                     lambda: fs.flagsparse_token_dispatch(dual(x), r),
                     lambda: fs.flagsparse_token_dispatch_grad(dual(y), r),
                     lambda: fs.flagsparse_token_combine(dual(y), r, w),
                     lambda: fs.flagsparse_token_combine(y, r, dual(w)),
                     lambda: fs.flagsparse_token_combine_grad(dual(x), y, r, w),
                     lambda: fs.flagsparse_token_combine_grad(x, dual(y), r, w),
                     lambda: fs.flagsparse_token_combine_grad(x, y, r, dual(w)),
                     lambda: fs.flagsparse_embedding(tokens, table, out=dual(x)),
                     lambda: fs.flagsparse_embedding_grad(tokens, x, 4, out=dual(table)),
                     lambda: fs.flagsparse_token_dispatch(x, r, out=dual(y)),
                     lambda: fs.flagsparse_token_combine(y, r, out=dual(x))):
            with pytest.raises(NotImplementedError, match="tangent"):
                call()
        assert torch.equal(fs.flagsparse_embedding(tokens, table), table[tokens])
        assert torch.equal(fs.flagsparse_token_dispatch(x, r)[0], x[0])
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: fs.flagsparse_embedding(tokens, t), (table,),
                       (torch.ones_like(table),))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: fs.flagsparse_embedding(tokens, t))(table[None])
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: fs.flagsparse_embedding(tokens, t).sum())(table)


@pytest.mark.parametrize("alpha", [float("inf"), float("nan"), -2.0])
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("n, k, dim", [(3, 2, 264), (3, 2, 33), (6000, 5, 264), (900, 37, 5),
                                       (40, 3, 4096), (4, 0, 16)])
def test_a_mask_that_leaves_nothing_meets_no_alpha(dtype, alpha, n, k, dim):
    """A token without assignments gets beta * out, the weight of a masked one a gradient of zero,
    also where alpha is not finite.  The other tokens' sums are a quarter at least: alpha decides
    on which side of beta * out they lie."""
    rng = np.random.default_rng(n + k)
    experts = random_experts(n, k, 7, 0.3, seed=n)
    experts[torch.from_numpy(rng.random(n) < 0.5).cuda()] = -1
    r = fs.prepare_token_route(experts, 7)
    none = (experts < 0).all(1)
    y = randn(n * k, dim, dtype=dtype).abs() + 0.5
    w = randn(n, k, dtype=dtype, seed=1).abs() + 0.5
    for weights in (None, w, w.float()):
        got = fs.flagsparse_token_combine(y, r, weights, alpha=alpha)
        assert torch.equal(got[none], torch.zeros_like(got[none]))
        out = torch.full((n, dim), 3.0, dtype=dtype, device="cuda")
        fs.flagsparse_token_combine(y, r, weights, alpha=alpha, beta=0.5, out=out)
        assert torch.equal(out[none], torch.full_like(out[none], 1.5))
        for rest, beside in ((got[~none], 0.0), (out[~none], 1.5)):
            assert (rest.isnan() if alpha != alpha
                    else rest == alpha if alpha > 0 else rest < beside).all()
        if weights is not None:
            g = torch.ones(n, dim, dtype=dtype, device="cuda")
            gy, gw = fs.flagsparse_token_combine_grad(g, y, r, weights, alpha=alpha)
            gone = experts < 0
            assert torch.equal(gw[gone], torch.zeros_like(gw[gone]))
            assert (gw[~gone].isnan() if alpha != alpha
                    else gw[~gone].sign() == np.sign(alpha)).all()
            held = int(r.indptr[-1])
            assert not gy[held:].any() and gy[:held].all()


def test_views_that_stand_for_the_negative():
    """The imaginary part of a conjugate is a view with a sign that only PyTorch knows of."""
    view = lambda n, seed: torch.complex(randn(n, 1, seed=seed),  # noqa: E731
                                         randn(n, 1, seed=seed + 1)).conj().imag
    table, x, y = view(9, 0), view(4, 2), view(8, 4)
    assert table.is_neg() and table.stride(0) == 2
    plain = lambda t: t.resolve_neg().contiguous()  # noqa: E731
    tokens = torch.tensor([1, 8, 1, 4], device="cuda")
    r = fs.prepare_token_route(torch.tensor([[0, 1], [1, -1], [1, 0], [0, 0]], device="cuda"), 2)
    w = randn(4, 2)
    same = lambda fn, *args: torch.equal(fn(*args), fn(*map(  # noqa: E731
        lambda a: plain(a) if isinstance(a, torch.Tensor) and a.is_neg() else a, args)))
    assert torch.equal(fs.flagsparse_embedding(tokens, table), plain(table)[tokens])
    assert same(fs.flagsparse_embedding_grad, tokens, x, 9)
    assert same(fs.flagsparse_token_dispatch, x, r)
    assert same(fs.flagsparse_token_dispatch_grad, y, r)
    assert same(fs.flagsparse_token_combine, y, r, w)
    assert same(fs.flagsparse_token_combine, y, r, torch._neg_view(w))
    for a, b in zip(fs.flagsparse_token_combine_grad(x, y, r, w),
                    fs.flagsparse_token_combine_grad(plain(x), plain(y), r, w)):
        assert torch.equal(a, b)
    for beta in (0.0, 0.5):
        out, want = view(4, 6), plain(view(4, 6))
        assert fs.flagsparse_embedding(tokens, plain(table), out=out, beta=beta) is out
        assert torch.equal(out, fs.flagsparse_embedding(tokens, plain(table), out=want, beta=beta))
        out, want = view(9, 6), plain(view(9, 6))
        assert fs.flagsparse_embedding_grad(tokens, plain(x), 9, out=out, beta=beta) is out
        assert torch.equal(out, fs.flagsparse_embedding_grad(tokens, plain(x), 9, out=want,
                                                             beta=beta))


def test_out_may_not_be_what_is_read_under_another_name():
    """The addresses decide, not which storage object a tensor was made from."""
    other = torch.from_dlpack
    table, tokens = randn(20, 8), torch.arange(20, device="cuda")

    def refused(fn, *args, **kwargs):
        with pytest.raises(ValueError, match="must not overlap"):
            fn(*args, **kwargs)

    refused(fs.flagsparse_embedding_grad, tokens, table, 20, out=other(table), beta=1.0)
    refused(fs.flagsparse_embedding_grad, tokens[:15], table[5:], 20, out=other(table))
    refused(fs.flagsparse_embedding, tokens[:15], table, out=other(table[5:]))
    words = torch.zeros(20, 2, dtype=torch.int32, device="cuda")
    refused(fs.flagsparse_embedding, words[:10].view(-1), randn(3, 2), out=words.view(torch.float32))
    r = fs.prepare_token_route(torch.zeros(10, 2, dtype=torch.int64, device="cuda"), 2)
    refused(fs.flagsparse_token_dispatch, table[:10], r, out=other(table))
    slots = r.slots.view(torch.float32)
    refused(fs.flagsparse_token_combine, randn(20, 2), r, out=slots)
    refused(fs.flagsparse_token_dispatch_grad, randn(20, 2), r, out=slots)
    refused(fs.flagsparse_token_dispatch, randn(10, 1), r, out=slots.view(20, 1))
    row = randn(1, 8).expand(20, 8)
    refused(fs.flagsparse_embedding, tokens, row, out=row)
    into = torch.zeros(20, 8, device="cuda")                 # neighbours are taken as before
    both = torch.zeros(40, 8, device="cuda")
    both[:20] = table
    fs.flagsparse_embedding_grad(tokens, both[:20], 20, out=other(both[20:]))
    fs.flagsparse_embedding_grad(tokens, table, 20, out=into)
    assert torch.equal(both[20:], table) and torch.equal(into, table)


def test_other_threads_run_while_a_launch_waits():
    """A launch that finds the queue of launches full waits for the GPU, not with the interpreter's
    lock.  The GPU sleeps for some 0.7 seconds here, behind it there are more calls than the queue
    takes; a thread that looks at the clock every millisecond may not miss half of the sleep."""
    import threading
    import time
    n, k = 8, 2
    table, tokens, y = randn(16, 8), torch.arange(n, device="cuda"), randn(n * k, 8)
    experts, w = torch.zeros(n, k, dtype=torch.int64, device="cuda"), randn(n, k)
    r = fs.prepare_token_route(experts, 2)
    calls = [lambda: fs.flagsparse_embedding(tokens, table),
             lambda: fs.flagsparse_embedding_grad(tokens, table[:n], 16),
             lambda: fs.prepare_token_route(experts, 2),
             lambda: fs.flagsparse_token_dispatch(table[:n], r),
             lambda: fs.flagsparse_token_combine(y, r, w),
             lambda: fs.flagsparse_token_combine_grad(table[:n], y, r, w)]
    for call in calls:
        call()
    torch.cuda.synchronize()
    start = time.perf_counter()
    torch.cuda._sleep(100_000_000)
    torch.cuda.synchronize()
    cycles = int(0.7 / (time.perf_counter() - start) * 100_000_000)

    def watch(stop, gaps):
        last = time.perf_counter()
        while not stop.is_set():
            time.sleep(0.001)
            now = time.perf_counter()
            gaps.append(now - last)
            last = now

    for call in calls:
        stop, gaps = threading.Event(), []
        watcher = threading.Thread(target=watch, args=(stop, gaps))
        watcher.start()
        start = time.perf_counter()
        torch.cuda._sleep(cycles)
        for _ in range(4000):
            call()
        issued = time.perf_counter() - start
        torch.cuda.synchronize()
        stop.set()
        watcher.join()
        assert issued > 0.4, "the queue took every launch: more calls are needed"
        assert max(gaps) < 0.35


@pytest.mark.parametrize("pattern", PATTERNS)
@pytest.mark.parametrize("dtype, out_dtype, dim", [
    (torch.float32, torch.float32, 264), (torch.bfloat16, torch.bfloat16, 264),
    (torch.float16, torch.float16, 392), (torch.bfloat16, torch.float32, 264),
    (torch.bfloat16, torch.float32, 4104), (torch.float16, torch.float32, 392),
    (torch.float64, torch.float64, 130)], ids=ids)
def test_embedding_grad_into_rows_taken_16_bytes_at_a_time(pattern, dtype, out_dtype, dim):
    """Added to (rows that no token names stay as they are), scaled, written over: into an out whose
    rows the kernels take 16 bytes at a time, with and without a pitch of its own."""
    tokens, vocab = PATTERNS[pattern]
    n = tokens.numel()
    if n * dim > 1 << 24 or vocab * dim > 1 << 24:
        dim = 392 if dim > 392 else 40
    g, tok = randn(n, dim, dtype=dtype, seed=n), tokens.cuda()
    named = torch.bincount(tokens, minlength=vocab) > 0
    for pad, alpha, beta in ((0, 1.5, 1.0), (8, 1.0, 1.0), (8, 0.75, 0.5), (0, 1.0, -2.0),
                             (8, 1.0, 0.0)):
        out = randn(vocab, dim, dtype=out_dtype, seed=2, pad=pad)
        if beta == 0.0:
            out.fill_(float("nan"))
        elif beta == 1.0:
            out[~named.cuda()] = float("nan")
        before, again = cpu(out), out.clone()
        assert fs.flagsparse_embedding_grad(tok, g, vocab, alpha=alpha, beta=beta, out=out) is out
        fs.flagsparse_embedding_grad(tok.int(), g, vocab, alpha=alpha, beta=beta, out=again)
        assert torch.equal(again[named.cuda()], out[named.cuda()])       # one order of the sums
        total, terms, m = plain_grad(tokens, g, vocab, alpha, before, beta)
        if beta == 1.0:
            assert torch.isnan(out[~named.cuda()]).all()
            total, terms, m, out = total[named], terms[named], m[named], out[named.cuda()]
        assert_close(out, total, terms, m, acc=dtype)
    fs.check_selection_ids()


def test_embedding_grad_random_calls():
    """Sizes, types, layouts, masks, scalars and places of the result at random."""
    import random
    for seed in range(120):
        rng = random.Random(1000 + seed)
        torch.manual_seed(seed)
        dtype, index = rng.choice(TYPES), rng.choice([torch.int32, torch.int64])
        out_dtype = rng.choice([dtype, torch.float32]) if dtype.itemsize == 2 else dtype
        dim = rng.choice([1, 2, 8, 33, 64, 256, 257, 512, 520, 1032])
        n, vocab = int(2**rng.uniform(0, 14)), int(2**rng.uniform(0, 12))
        tokens = (torch.rand(n, device="cuda")**rng.choice([1, 4, 20]) * vocab).to(index)
        ignore = rng.choice([None, rng.randrange(vocab)])
        alpha, beta = rng.choice([1.0, -0.5]), rng.choice([0.0, 1.0, 0.25])

        def matrix(rows, kind):
            pad, off = rng.choice([0, 0, 8, 3]), rng.choice([0, 0, 8, 1])
            return torch.randn(rows, off + dim + pad, device="cuda").to(kind)[:, off:off + dim]

        g, out = matrix(n, dtype), matrix(vocab, out_dtype)
        before = cpu(out)
        fs.flagsparse_embedding_grad(tokens, g, vocab, alpha=alpha, ignore_index=ignore, out=out,
                                     beta=beta)
        total, terms, m = plain_grad(tokens, g, vocab, alpha, before, beta, ignore)
        assert_close(out, total, terms, m, acc=dtype)
    fs.check_selection_ids()


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("n, k, dim", [(9000, 3, 264), (20000, 2, 72), (11000, 1, 40),
                                       (5000, 9, 8), (400, 70, 520)])
def test_combine_of_several_tokens_a_warp(dtype, n, k, dim):
    """More tokens than warps fit the GPU: a warp's queue goes on from token to token, with rows
    that differ and tokens whose assignments are masked in part or all."""
    experts = random_experts(n, k, 11, 0.2, seed=n)
    experts[::17] = -1
    r = fs.prepare_token_route(experts, 11)
    slots, indptr, _ = plain_route(experts, 11)
    live = slots >= 0
    y, w = randn(n * k, dim, dtype=dtype, seed=1), randn(n, k, seed=2)
    y[int(indptr[-1]):] = float("nan")
    w[experts < 0] = float("nan")
    picked = torch.where(live[..., None], cpu(y)[torch.where(live, slots, 0)], 0.0)
    parts = torch.where(live, cpu(w), 0.0)[..., None] * picked
    assert_close(fs.flagsparse_token_combine(y, r, w), parts.sum(1), parts.abs().sum(1), 2 * k)
    out = randn(n, dim, dtype=dtype, seed=3)
    before = cpu(out)
    fs.flagsparse_token_combine(y, r, w, alpha=-0.5, beta=2.0, out=out)
    assert_close(out, -0.5 * parts.sum(1) + 2.0 * before,
                 0.5 * parts.abs().sum(1) + 2.0 * before.abs(), 2 * k)
    assert_close(fs.flagsparse_token_dispatch_grad(y, r), picked.sum(1), picked.abs().sum(1), k)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float64], ids=ids)
def test_embedding_grad_and_the_transposed_product(dtype):
    """The SpMM of this package with S written out: both within their bound of the 64-bit sum, so
    within two of them of each other (the SpMM has the same: products and additions in any order in
    float32 or float64, one rounding)."""
    n, vocab, dim = 300, 90, 64
    g = randn(n, dim, dtype=dtype, seed=1)
    tokens = torch.randint(0, vocab, (n,), device="cuda")
    ones, ptr = torch.ones(n, dtype=dtype, device="cuda"), torch.arange(n + 1, device="cuda")
    dense = fs.flagsparse_spmm_csr(ones, tokens, ptr, g, (n, vocab), op="trans")
    total, terms, m = plain_grad(tokens, g, vocab)
    for got in (dense, fs.flagsparse_embedding_grad(tokens, g, vocab)):
        assert_close(got, total, terms, m)


def test_two_threads_each_finish_their_calls():
    """Gradients, routes and the way there and back from two threads, each on a stream of its own
    or both on one; what goes wrong in a thread fails the test."""
    import threading
    n, vocab, dim, k = 9000, 4000, 128, 2
    g = randn(n, dim)
    tokens = [torch.randint(0, vocab, (n,), device="cuda") for _ in range(2)]
    experts = [random_experts(n, k, 16, 0.1, seed=i) for i in range(2)]

    def calls(i):
        r = fs.prepare_token_route(experts[i], 16)
        rows = fs.flagsparse_token_dispatch(g, r)
        return (fs.flagsparse_embedding_grad(tokens[i], g, vocab), r.slots, rows,
                fs.flagsparse_token_combine(rows, r), fs.flagsparse_embedding(tokens[i], g[:vocab]))

    want = [calls(i) for i in range(2)]
    torch.cuda.synchronize()
    for shared in (None, torch.cuda.Stream()):
        done, wrong = [0, 0], []

        def work(i):
            try:
                with torch.cuda.stream(shared or torch.cuda.Stream()):
                    for _ in range(20):
                        for a, b in zip(calls(i), want[i]):
                            assert torch.equal(a, b)
                        done[i] += 1
            except BaseException as error:  # noqa: BLE001
                wrong.append(error)

        threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert not wrong and done == [20, 20]
