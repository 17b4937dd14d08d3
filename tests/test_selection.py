"""Selection products (embedding, token route) on the CPU: what they refuse before anything
touches a device, the status codes of the C entry points, and the work split of the gradient
kernel restated in Python."""

import ctypes
import random

import pytest
import torch

import flagsparse_b200 as fs
from flagsparse_b200 import _lib, selection

TOK = torch.zeros(3, dtype=torch.int64)
TABLE = torch.zeros(5, 4)


def test_public_names():
    for name in ("flagsparse_embedding", "flagsparse_embedding_grad", "prepare_token_route",
                 "TokenRoute", "flagsparse_token_dispatch", "flagsparse_token_dispatch_grad",
                 "flagsparse_token_combine", "flagsparse_token_combine_grad",
                 "check_selection_ids"):
        assert name in fs.__all__ and callable(getattr(fs, name))


@pytest.mark.parametrize("args, kwargs, error, message", [
    ((TOK.float(), TABLE), {}, TypeError, "tokens dtype must be torch.int32 or torch.int64"),
    (([0, 1], TABLE), {}, TypeError, "tokens must be a torch.Tensor"),
    ((TOK, TABLE.to(torch.complex64)), {}, TypeError, "table dtype must be one of"),
    ((TOK, TABLE.long()), {}, TypeError, "table dtype must be one of"),
    ((TOK, TABLE[0]), {}, ValueError, "table must be a 2D tensor"),
    ((TOK, TABLE), {"alpha": 1j}, TypeError, "alpha is complex"),
    ((TOK, TABLE), {"alpha": torch.ones(2)}, ValueError, "alpha must be a scalar"),
    ((TOK, TABLE), {"alpha": "two"}, ValueError, "could not convert"),
    ((TOK, TABLE), {"ignore_index": 1.0}, TypeError, "ignore_index must be an integer"),
    ((TOK, TABLE), {"ignore_index": True}, TypeError, "ignore_index must be an integer"),
    ((TOK, TABLE), {"ignore_index": 2**63}, ValueError, "ignore_index must fit int64"),
    ((TOK, TABLE), {}, ValueError, "table must be a CUDA tensor"),
    ((TOK, TABLE.clone().requires_grad_()), {"out": torch.zeros(3, 4)}, RuntimeError,
     "does not support automatic differentiation"),
])
def test_embedding_refuses(args, kwargs, error, message):
    with pytest.raises(error, match=message):
        fs.flagsparse_embedding(*args, **kwargs)


@pytest.mark.parametrize("args, kwargs, error, message", [
    ((TOK, torch.zeros(3, 4), -1), {}, ValueError, "n_rows must be non-negative"),
    ((TOK, torch.zeros(3, 4), 2.0), {}, TypeError, "n_rows must be an integer"),
    ((TOK, torch.zeros(4, 4), 5), {}, ValueError, "grad shape must be tokens.shape"),
    ((TOK, torch.zeros(3), 5), {}, ValueError, "grad shape must be tokens.shape"),
    ((TOK, torch.zeros(3, 4), 5), {"out_dtype": torch.bfloat16}, TypeError, "out dtype must be"),
    ((TOK, torch.zeros(3, 4, dtype=torch.float64), 5), {"out_dtype": torch.float32}, TypeError,
     "out dtype must be"),
    ((TOK, torch.zeros(3, 4, dtype=torch.half), 5), {"out": torch.zeros(5, 4).bfloat16()},
     TypeError, "out dtype must be"),
    ((TOK, torch.zeros(3, 4), 5), {}, ValueError, "grad must be a CUDA tensor"),
])
def test_embedding_grad_refuses(args, kwargs, error, message):
    with pytest.raises(error, match=message):
        fs.flagsparse_embedding_grad(*args, **kwargs)


@pytest.mark.parametrize("args, error, message", [
    ((TOK, 4), ValueError, "experts must be a 2D tensor"),
    ((TOK[None].float(), 4), TypeError, "experts dtype must be"),
    ((TOK[None], 4.0), TypeError, "n_experts must be an integer"),
    ((TOK[None], -1), ValueError, "n_experts must be between 0 and 2047"),
    ((TOK[None], 2048), ValueError, "n_experts must be between 0 and 2047"),
    ((TOK[None], 4), ValueError, "experts must be a CUDA tensor"),
])
def test_route_refuses(args, error, message):
    with pytest.raises(error, match=message):
        fs.prepare_token_route(*args)


def _route(n_tokens=3, k=2, n_experts=4):
    """A route on the CPU: enough for the checks in front of a launch."""
    buffer = torch.arange(2 * n_tokens * k + n_experts + 1, dtype=torch.int32)
    return fs.TokenRoute(buffer, n_tokens, k, n_experts, 0)


def test_route_arrays_are_views_of_one_buffer():
    r = _route()
    assert r.slots.tolist() == [[0, 1], [2, 3], [4, 5]] and r.slots is r.slots
    assert r.indptr.tolist() == [6, 7, 8, 9, 10]
    assert r.indices.tolist() == [11, 12, 13, 14, 15, 16]
    assert (r.n_rows, r.n_tokens, r.k, r.n_experts) == (6, 3, 2, 4)
    assert "n_tokens=3, k=2, n_experts=4" in repr(r)


def test_route_operators_refuse():
    r, x, y = _route(), torch.zeros(3, 4), torch.zeros(6, 4)
    with pytest.raises(TypeError, match="route must be a TokenRoute"):
        fs.flagsparse_token_dispatch(x, (1, 2))
    with pytest.raises(ValueError, match=r"x.shape\[0\] must be n_tokens=3"):
        fs.flagsparse_token_dispatch(y, r)
    with pytest.raises(ValueError, match="x must be a 2D tensor"):
        fs.flagsparse_token_dispatch(x[None], r)
    with pytest.raises(TypeError, match="x dtype must be one of"):
        fs.flagsparse_token_dispatch(x.int(), r)
    with pytest.raises(ValueError, match=r"y.shape\[0\] must be n_tokens \* k=6"):
        fs.flagsparse_token_combine(x, r)
    with pytest.raises(ValueError, match="weights shape must be"):
        fs.flagsparse_token_combine(y, r, torch.zeros(2, 3))
    with pytest.raises(TypeError, match="weights dtype must be the dtype of the rows"):
        fs.flagsparse_token_combine(y, r, torch.zeros(3, 2).half())
    with pytest.raises(ValueError, match=r"grad.shape\[0\] must be n_tokens \* k=6"):
        fs.flagsparse_token_dispatch_grad(x, r)
    with pytest.raises(ValueError, match="y is needed"):
        fs.flagsparse_token_combine_grad(x, None, r, torch.zeros(3, 2))
    with pytest.raises(TypeError, match="y dtype must match"):
        fs.flagsparse_token_combine_grad(x, y.half(), r)
    with pytest.raises(ValueError, match="same number of columns"):
        fs.flagsparse_token_combine_grad(x, torch.zeros(6, 5), r)
    with pytest.raises(ValueError, match="route must be a CUDA tensor"):
        fs.flagsparse_token_dispatch(x, r)
    with pytest.raises(RuntimeError, match="does not support automatic differentiation"):
        fs.flagsparse_token_combine(y.requires_grad_(), r, out=torch.zeros(3, 4))


def test_the_host_module_is_built_and_leaves_what_it_does_not_take():
    """It makes the usual calls on CUDA tensors; for any other it answers None."""
    host = selection._host
    assert host is not None, "_b2s_host.so not built (python -m flagsparse_b200._build)"
    r = _route()
    parts = (r._buffer, r.n_tokens, r.k, r.n_experts, r._stream)
    x, y = torch.zeros(3, 4), torch.zeros(6, 4)
    assert host.embedding(TOK, TABLE, 1.0, None) is None
    assert host.embedding(None, TABLE, 1.0, None) is None
    assert host.embedding(TOK, TABLE, 1.0) is None
    assert host.embedding(TOK, TABLE, "1", 2**70) is None
    assert host.embedding_grad(TOK, x, 5, 1.0, None, None, 0.0, None) is None
    assert host.embedding_grad(TOK, x, -5, 1.0, None, None, 0.0, "float") is None
    assert host.route_plan(TOK[None], 4) is None and host.route_plan(TOK, 4.0) is None
    assert host.dispatch(*parts, x) is None and host.dispatch(x) is None
    assert host.combine(*parts, y, None, 1.0) is None
    assert host.combine_grad(*parts, x, y, torch.zeros(3, 2), 1.0) is None
    with pytest.raises(TypeError):
        host.bind(1, 2)
    with pytest.raises(TypeError):
        host.bind_status("0", 1)


def test_result_places():
    """out that the kernels can write is written in place; another layout gets a stand-in."""
    f32, like = torch.float32, torch.zeros(1)
    with pytest.raises(ValueError, match="beta != 0 requires out="):
        selection._result(None, (3, 4), like, f32, 1.0)
    for bad in (torch.zeros(4, 3), torch.zeros(3, 4).half()):
        with pytest.raises(ValueError, match="out shape/dtype must match result"):
            selection._result(bad, (3, 4), like, f32, 0.0)
    flat, address, pitch = selection._result(None, (2, 3, 4), like, f32, 0.0)
    assert flat.shape == (2, 3, 4) and address == flat.data_ptr() and pitch == 4
    wide = torch.zeros(3, 9)[:, :4]
    flat, address, pitch = selection._result(wide, (3, 4), like, f32, 0.0)
    assert address == wide.data_ptr() and pitch == 9
    version = wide._version
    assert selection._finish(wide, flat) is wide and wide._version > version
    cols = torch.arange(12.0).reshape(4, 3).t()
    flat, address, pitch = selection._result(cols, (3, 4), like, f32, 1.0)
    assert address != cols.data_ptr() and pitch == 4 and torch.equal(flat, cols)   # beta reads it
    flat.zero_()
    assert selection._finish(cols, flat) is cols and not cols.any()
    deep = torch.zeros(2, 3, 9)[:, :, :4]                # rows of one pitch: a view will do
    flat, address, pitch = selection._result(deep, (2, 3, 4), like, f32, 0.0)
    assert address == deep.data_ptr() and pitch == 9
    deep = torch.zeros(3, 2, 4).transpose(0, 1)
    flat, address, pitch = selection._result(deep, (2, 3, 4), like, f32, 0.0)
    assert address != deep.data_ptr() and pitch == 4
    for empty in (torch.zeros(0, 3, 4), torch.zeros(2, 3, 0)):
        flat, _, _ = selection._result(empty, tuple(empty.shape), like, f32, 0.0)
        assert selection._finish(empty, flat) is empty


def test_overlap_of_out_and_what_is_read():
    wide = torch.zeros(6, 10)
    refuse = lambda out, *t: pytest.raises(ValueError, selection._refuse_overlap, out, *t)  # noqa: E731
    selection._refuse_overlap(wide, None, torch.zeros(6, 10), wide[:0])
    selection._refuse_overlap(wide[:3], wide[3:])
    selection._refuse_overlap(wide[:, :4], wide[:, 4:])      # columns side by side
    selection._refuse_overlap(wide[:, 6:], wide[:, :6], wide[:, 2:6])
    selection._refuse_overlap(wide[2:, 6:], wide[:, :6])
    refuse(wide, wide)
    refuse(wide[:4], wide[3:])
    refuse(wide[:, :5], wide[:, 4:])
    refuse(wide[:, 4:], wide[:, :5])
    refuse(wide[1:, :5], wide[:, 4:])
    refuse(wide[:, :4], wide.view(-1))
    refuse(wide, torch.zeros(1), wide[2])


def test_c_entry_points_answer_before_any_launch():
    lib, d = _lib.load(), ctypes.c_void_p(4096)          # never read: every call below is refused
    odd = ctypes.c_void_p(4097)
    ok, dtype, arg, align, ws, rng = 0, 1, 2, 3, 6, 7
    rows = lambda v=0, i=0, idx=d, n=4, t=d, r=5, ld=8, dim=8, o=d, ldo=8: lib.b2s_select_rows(  # noqa: E731
        v, i, idx, n, 0, 0, t, r, ld, dim, o, ldo, 1.0, 0.0, None, None)
    assert rows(v=2) == dtype and rows(v=9) == dtype and rows(i=7) == dtype
    assert rows(n=-1) == arg and rows(idx=None) == arg and rows(t=None) == arg
    assert rows(o=None) == arg and rows(ld=7) == arg and rows(ldo=7) == arg
    assert rows(n=2**31) == rng and rows(r=2**31) == rng and rows(dim=2**23) == rng
    assert rows(idx=odd) == align and rows(t=odd) == align and rows(o=odd) == align
    assert rows(n=0) == ok and rows(dim=0) == ok
    grad = lambda v=5, o=5, n=4, r=5, b=1 << 30, w=d, ld=8: lib.b2s_select_grad(  # noqa: E731
        v, o, 0, d, n, 0, 0, d, ld, r, 8, d, 8, 1.0, 0.0, w, b, None, None)
    assert grad(v=3) == dtype and grad(v=0, o=5) == dtype and grad(v=1, o=0) == dtype
    assert grad(o=4) == dtype and grad(n=-1) == arg and grad(ld=4) == arg
    assert grad(b=16) == ws and grad(w=None) == ws and grad(w=odd) == align
    assert grad(r=0) == ok
    assert lib.b2s_select_grad_bytes(2, 4, 4, 4) == 0 and lib.b2s_select_grad_bytes(0, -1, 4, 4) == 0
    plan = lambda i=1, e=d, t=4, k=2, n=8, b=1 << 30: lib.b2s_route_plan(  # noqa: E731
        i, e, t, k, n, d, d, d, d, b, None, None)
    assert plan(i=2) == dtype and plan(e=None) == arg and plan(n=-1) == arg
    assert plan(n=2048) == rng and plan(t=2**31, k=2) == rng and plan(t=9000, b=0) == ws
    assert plan(e=ctypes.c_void_p(4100)) == align
    disp = lambda v=0, x=d, s=d, h=d, t=4, ld=8: lib.b2s_route_dispatch(  # noqa: E731
        v, x, ld, t, 2, 8, s, h, d, 8, None)
    assert disp(v=3) == dtype and disp(x=None) == arg and disp(s=None) == arg
    assert disp(h=None) == arg and disp(ld=1) == arg and disp(t=0) == ok
    comb = lambda v=0, w=0, p=d, y=d: lib.b2s_route_combine(  # noqa: E731
        v, y, 8, d, w, p, 4, 2, 8, d, 8, 1.0, 0.0, None)
    assert comb(v=2) == dtype and comb(w=4) == dtype and comb(y=None) == arg
    assert comb(p=ctypes.c_void_p(4098)) == align
    back = lambda w=d, gw=d, y=d, wt=0: lib.b2s_route_combine_grad(  # noqa: E731
        0, d, 8, y, 8, d, d, wt, w, 4, 2, 8, 1.0, d, 8, gw, None)
    assert back(w=None) == arg and back(y=None) == arg and back(wt=5) == dtype


# ---- the ranges of the gradient: every entry is summed once, by one owner --------------------------
CROSS = 32


def _first(n, below):
    """The first index in [0, n) that `below` does not hold for, 32 places at a time."""
    lo, length = 0, n
    while length > 1:
        step, end = -(-length // 32), lo + length
        hits = sum(lo + i * step < end and below(lo + i * step) for i in range(32))
        if hits == 0:
            break
        lo += (hits - 1) * step + 1
        length = min(end - lo, step)
    return lo


def _held(keys, none):
    if keys[-1] < none:
        return len(keys)
    lo, length = 0, len(keys)
    while length > 0:
        step, end = -(-length // 32), lo + length
        hits = sum(lo + i * step < end and keys[lo + i * step] < none for i in range(32))
        if hits == 0:
            break
        lo += (hits - 1) * step + 1
        length = min(end - lo, step - 1)
    return lo


def _ranges(keys, none, most):
    """The decisions of the warps that sum ranges of the sorted entries, and of the kernel that
    joins the runs they cut (b2s_select.cu); `none`: masked."""
    m = _held(keys, none)
    assert m == sum(k < none for k in keys)
    if m == 0:
        return {}, 0
    size = max(2, -(-m // most))
    rows, head, tail, runs = {}, {}, {}, []

    def crossing(x):
        if x <= 0 or x >= m:
            return 0
        return sum(x + i < m and keys[x + i] == keys[x - 1] for i in range(CROSS))

    for r in range(-(-m // size)):
        a, b = r * size, min((r + 1) * size, m)
        into, out = crossing(a), crossing(b)
        lo = a + (0 if into == CROSS else into)
        hi = b + (0 if out == CROSS else out)
        first, acc = into == CROSS, []
        for i in range(lo, hi):
            acc.append(i)
            if i + 1 < hi and keys[i + 1] == keys[i]:
                continue
            goes_on = out == CROSS and i + 1 == hi
            where, name = (head, r) if first else (tail, r) if goes_on else (rows, keys[i])
            assert name not in where
            where[name], acc = acc, []
            if first and not goes_on:
                runs.append((_first(lo, lambda j: keys[j] < keys[i]) // size, r, keys[i]))
            first = False
    for begin, end, key in runs:
        assert key not in rows
        rows[key] = sum((tail.pop(r) if r == begin else head.pop(r)
                         for r in range(begin, end + 1)), [])
    assert not head and not tail
    return rows, len(runs)


def test_gradient_ranges_cover_every_entry_once():
    rng = random.Random(3)
    cut = 0
    for _ in range(3000):
        none = rng.choice([1, 2, 5, 50])
        n = rng.choice([1, 7, 8, 9, 31, 32, 33, 40, 64, 65, 97, 130, 700, 2000])
        hot = rng.choice([0.1, 0.9])
        keys = sorted(min(none, int(rng.expovariate(1.0))) if rng.random() < hot
                      else rng.randrange(none + 1) for _ in range(n))
        rows, runs = _ranges(keys, none, rng.choice([1, 2, 3, 10, n, n // 2 + 1, n // 24 + 1]))
        cut += runs
        want = {}
        for i, k in enumerate(keys):
            if k < none:
                want.setdefault(k, []).append(i)
        assert rows == want
    assert cut > 100
