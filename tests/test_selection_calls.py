"""Selection products on the CPU: calls beside the usual one, up to where the device begins."""

import pytest
import torch

import flagsparse_b200 as fs
from flagsparse_b200 import selection

TOK = torch.zeros(3, dtype=torch.int64)
TABLE = torch.zeros(5, 4)


def _route(n_tokens=3, k=2, n_experts=4):
    n = n_tokens * k
    return fs.TokenRoute(torch.zeros(2 * n + n_experts + 1, dtype=torch.int32), n_tokens, k,
                         n_experts, 0)


def test_tangents_are_refused():
    import torch.autograd.forward_ad as forward
    r, x, y, w = _route(), torch.zeros(3, 4), torch.zeros(6, 4), torch.zeros(3, 2)
    with forward.dual_level():
        dual = lambda t: forward.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: fs.flagsparse_embedding(TOK, dual(TABLE)),
                     lambda: fs.flagsparse_embedding_grad(TOK, dual(x), 5),
                     lambda: fs.flagsparse_token_dispatch(dual(x), r),
                     lambda: fs.flagsparse_token_dispatch_grad(dual(y), r),
                     lambda: fs.flagsparse_token_combine(dual(y), r, w),
                     lambda: fs.flagsparse_token_combine(y, r, dual(w)),
                     lambda: fs.flagsparse_token_combine_grad(dual(x), y, r, w),
                     lambda: fs.flagsparse_token_combine_grad(x, y, r, dual(w)),
                     lambda: fs.flagsparse_embedding(TOK, TABLE, out=dual(x))):
            with pytest.raises(NotImplementedError, match="tangent"):
                call()
        with pytest.raises(ValueError, match="must be a CUDA tensor"):
            fs.flagsparse_embedding(TOK, TABLE)


def test_views_that_stand_for_the_negative_are_written_out():
    z = torch.complex(torch.arange(6.0).reshape(6, 1), torch.arange(6.0).reshape(6, 1) + 1)
    view = z.conj().imag                                     # rows that a kernel could read as they lie
    assert view.is_neg() and selection._row_major_ok(view)
    for rows in (selection._rows(view), selection._as_stored(torch._neg_view((-view).resolve_neg()))):
        assert not rows.is_neg() and torch.equal(rows, view)
    assert selection._rows(TABLE) is TABLE
    flat, address, _ = selection._result(view, (6, 1), view, torch.float32, 1.0)
    assert address != view.data_ptr() and not flat.is_neg() and torch.equal(flat, view)
    flat.fill_(5.0)
    assert selection._finish(view, flat) is view and (view == 5).all() and (z.imag == -5).all()


def test_overlap_is_a_matter_of_addresses():
    refuse = lambda out, *t: pytest.raises(ValueError, selection._refuse_overlap, out, *t)  # noqa: E731
    wide = torch.zeros(6, 10)
    alias = torch.from_dlpack(wide[1:])                      # the same memory, another storage
    assert alias.untyped_storage().data_ptr() != wide.untyped_storage().data_ptr()
    refuse(wide, alias)
    refuse(alias, wide[:2])
    selection._refuse_overlap(alias, wide[:1])
    selection._refuse_overlap(alias[:, :4], wide[:, 4:])
    row = torch.zeros(1, 8).expand(5, 8)
    refuse(row, row)
    words = torch.zeros(16)                                  # sizes of both types count
    halves = words.view(torch.float16)
    refuse(halves[16:20].view(2, 2), words[:12].view(6, 2))
    refuse(words[:8].view(4, 2), halves[12:18].view(3, 2))
    selection._refuse_overlap(halves[16:20].view(2, 2), words[:8].view(4, 2))


@pytest.mark.parametrize("call", [
    lambda r, t: fs.flagsparse_token_dispatch(torch.zeros(3, 1), r, out=t.view(6, 1)),
    lambda r, t: fs.flagsparse_token_combine(torch.zeros(6, 2), r, out=t),
    lambda r, t: fs.flagsparse_token_dispatch_grad(torch.zeros(6, 2), r, out=t)])
def test_out_may_not_be_the_route(call, monkeypatch):
    monkeypatch.setattr(selection, "_check_first_device", lambda t, name: t.get_device())
    r = _route()
    with pytest.raises(ValueError, match="must not overlap"):
        call(r, r.slots.view(torch.float32))


def test_out_may_not_be_the_tokens(monkeypatch):
    monkeypatch.setattr(selection, "_check_first_device", lambda t, name: t.get_device())
    words = torch.zeros(8, 2, dtype=torch.int64)
    with pytest.raises(ValueError, match="must not overlap"):
        fs.flagsparse_embedding(words[0], TABLE[:, :2], out=words.view(torch.float32)[:2, :2])
