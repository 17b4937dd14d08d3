"""Products with a selection matrix: the embedding lookup and its gradient, and tokens sorted by
expert and back.

The sparse matrices of a language model select rows.  ``tokens`` stands for the matrix S with
S[i, tokens[i]] = 1; ``experts`` (n_tokens x k) for the matrix R that has a one for every
assignment of a token to an expert.  The calls here are the products that ``flagsparse_spmm_csr``
computes when such a matrix is written out as CSR, without writing it out, checking it or keeping
a plan of it, together with the gradients that training needs:

    flagsparse_embedding        alpha * S @ table + beta * out
    flagsparse_embedding_grad   alpha * S.T @ grad + beta * out
    prepare_token_route         the rows of R sorted by expert: slots, indptr, indices
    flagsparse_token_dispatch   the tokens' rows in that order (and flagsparse_token_dispatch_grad)
    flagsparse_token_combine    the weighted sum of a token's rows (and ..._combine_grad)

FlagSparse has no counterpart (its gather / scatter take one vector, gather_scatter.py:22-81).

The lookup, the dispatch and the combine are differentiable: when an input requires a gradient
and gradients are enabled they record themselves for ``torch.autograd``.  Inside a CUDA graph
capture that is refused (autograd may run a leaf's accumulation on a stream outside the capture);
captured training steps call the ``*_grad`` functions.  Forward-mode derivatives are not
supported: a tensor with a tangent is refused.

Nothing synchronises.  Ids are checked by the kernels: one outside its range selects nothing, and
IndexError is raised by the next call on that device that takes ids (a lookup, its gradient, a
route), or by ``check_selection_ids()``, which waits for the device.
"""

from __future__ import annotations

import ctypes
import threading
import warnings
from types import SimpleNamespace

import torch
from torch.autograd.forward_ad import unpack_dual
from torch.autograd.function import once_differentiable

from . import _lib
from ._contract import SUPPORTED_INDEX_DTYPES, check_scalar
from .spmm import _row_major_ok

SUPPORTED_SELECTION_VALUE_DTYPES = (torch.float16, torch.bfloat16, torch.float32, torch.float64)
MAX_EXPERTS = 2047               # the plan sorts by one digit of 11 bits
MAX_ENTRIES = 2**31 - 1 - 2**25  # positions are int32
MAX_ROWS = 2**31 - 2
MAX_DIM = 1 << 22


class _Host:
    """The usual call (plain strided tensors, a new result, nothing to record) is made by a C++
    module (csrc/host/b2s_host.cpp): it returns None for every other one, which then takes the way
    below.  Without the module all calls do; the kernels are the same.

    The module and the library are loaded by the first call and not when the package is imported:
    a library that lacks an entry point can be built anew by the package that it belongs to.  Then
    the module takes this object's place (an attribute of it costs a call 0.3 us less)."""

    def __getattr__(self, name):
        global _host
        if name.startswith("__"):
            raise AttributeError(name)
        if not _lib.LIB_PATH.exists():  # the call itself will say so, behind its own checks
            return _not_here
        with _HOST_LOCK:
            host = _bound_host()
            if _host is self:
                _host = host
        return getattr(host, name)


def _not_here(*args):
    return None


# in the place of a module that has not been built
_NO_HOST = SimpleNamespace(**dict.fromkeys(
    ("embedding", "embedding_grad", "route_plan", "dispatch", "combine", "combine_grad",
     "bind_status"), _not_here))


def _bound_host():
    lib = _lib.load()
    try:
        from . import _b2s_host
    except ImportError:
        return _NO_HOST
    if _b2s_host.torch_version != torch.__version__:     # it reads PyTorch's own structures
        warnings.warn(f"flagsparse_b200/_b2s_host.so was built for PyTorch "
                      f"{_b2s_host.torch_version}, this is {torch.__version__}: calls are made "
                      "without it (run `python -m flagsparse_b200._build`)", stacklevel=4)
        return _NO_HOST
    address = [ctypes.cast(getattr(lib, name), ctypes.c_void_p).value for name in (
        "b2s_select_rows", "b2s_select_grad_bytes", "b2s_select_grad", "b2s_route_plan_bytes",
        "b2s_route_plan", "b2s_route_dispatch", "b2s_route_combine", "b2s_route_combine_grad")]
    _b2s_host.bind(*address, torch.nn.Parameter, torch.OutOfMemoryError)
    return _b2s_host


_host = _Host()
_HOST_LOCK = threading.Lock()

_WORDS = {}
_WORDS_LOCK = threading.Lock()


# -------------------------------------------------------------------------------------------------
# errors that kernels report
# -------------------------------------------------------------------------------------------------
class _StatusWord:
    """One int32 in pinned host memory per device; the kernels set it when they meet an id
    outside its range, and the host reads it without a copy or a synchronisation."""

    def __init__(self):
        self.memory = torch.zeros(1, dtype=torch.int32).pin_memory()
        self.address = self.memory.data_ptr()
        self.value = ctypes.c_int32.from_address(self.address)

    def check(self):
        if self.value.value:
            self.value.value = 0
            raise IndexError("a token or expert id given to an earlier call on this device lies "
                             "outside its range")


def _status_word(index):
    word = _WORDS.get(index)
    if word is None:
        with _WORDS_LOCK:
            word = _WORDS.get(index)
            if word is None:
                word = _WORDS[index] = _StatusWord()
                if _host is not None:
                    _host.bind_status(index, word.address)
    word.check()
    return word.address


def check_selection_ids(device=None):
    """Wait for `device` (default: the current one) and raise IndexError if a kernel of this
    module met an id outside its range since the last check."""
    index = torch.device("cuda" if device is None else device).index
    if index is None:
        index = torch.cuda.current_device()
    torch.cuda.synchronize(index)
    word = _WORDS.get(index)
    if word is not None:
        word.check()


# -------------------------------------------------------------------------------------------------
# arguments.  A decoding step makes these calls on a few rows, where the host's time is all there
# is: what every call checks is spelled out instead of looped over.
# -------------------------------------------------------------------------------------------------
_Tensor = torch.Tensor
# the stream's handle without a Stream object around it
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream",
                      lambda index: torch.cuda.current_stream(index).cuda_stream)


def _check_ids(t, name):
    if not isinstance(t, _Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype not in SUPPORTED_INDEX_DTYPES:
        raise TypeError(f"{name} dtype must be torch.int32 or torch.int64")


def _check_values(t, name):
    if not isinstance(t, _Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype not in SUPPORTED_SELECTION_VALUE_DTYPES:
        raise TypeError(f"{name} dtype must be one of: float16, bfloat16, float32, float64")
    _refuse_tangent(t, name)


def _refuse_tangent(t, name):
    # (such a tensor does not require a gradient: without this its tangent would be lost)
    if unpack_dual(t).tangent is not None:
        raise NotImplementedError(
            f"{name} has a tangent: forward-mode derivatives are not supported")


def _check_first_device(t, name):
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    return t.get_device()


def _check_same_device(t, name, index, first):
    if t is not None and t.get_device() != index:
        if not t.is_cuda:
            raise ValueError(f"{name} must be a CUDA tensor")
        raise ValueError(f"{name} must be on the same CUDA device as {first}")


def _check_size(name, value, limit):
    if value > limit:
        raise ValueError(f"{name} must be at most {limit}, got {value}")


def _as_int(value, name):
    if isinstance(value, bool) or not hasattr(value, "__index__"):
        raise TypeError(f"{name} must be an integer")
    return value.__index__()


def _scalar(value, dtype, name):
    return value if type(value) is float else float(check_scalar(value, dtype, name))


def _wants_grad(t, other=None):
    return ((t.requires_grad or (other is not None and other.requires_grad))
            and torch.is_grad_enabled())


def _capturing(index):
    """Whether the current stream of device `index` is captured into a graph."""
    if torch.cuda.current_device() == index:
        return torch.cuda.is_current_stream_capturing()
    with torch.cuda.device(index):
        return torch.cuda.is_current_stream_capturing()


def _refuse_capture(index):
    if _capturing(index):
        raise RuntimeError(
            "differentiable calls are not recorded inside a CUDA graph capture: call them under "
            "torch.no_grad() and take the gradients with the *_grad functions")


def _refuse_out(out, t, other=None):
    _refuse_tangent(out, "out")
    if _wants_grad(out, t) or _wants_grad(out, other):
        raise RuntimeError("out= does not support automatic differentiation, but one of the "
                           "arguments requires grad")


def _refuse_overlap(out, *inputs):
    """The kernels read their inputs while they write `out`.  Addresses are compared: one memory
    can have several storage objects (DLPack)."""
    for t in inputs:
        if t is None or not t.numel() or not out.numel():
            continue
        ends = [(v.data_ptr(), v.data_ptr() + v.element_size() * (1 + sum(
            (n - 1) * s for n, s in zip(v.shape, v.stride())))) for v in (out, t)]
        if ends[0][1] <= ends[1][0] or ends[1][1] <= ends[0][0]:
            continue
        # rows of one array side by side: columns that do not meet
        if out.dim() == t.dim() == 2 and t.dtype == out.dtype and out.stride() == t.stride():
            pitch = out.stride(0)
            if pitch > 0 and out.stride(1) == 1:
                apart = (ends[1][0] - ends[0][0]) // out.element_size() % pitch
                if out.shape[1] <= apart <= pitch - t.shape[1]:
                    continue
        raise ValueError("out must not overlap the tensors that are read")


def _rows(t):
    """`t` (2-D) with unit stride inside a row and rows that do not overlap; copied if need be."""
    t = _as_stored(t)
    return t if t.is_contiguous() or _row_major_ok(t) else t.contiguous()


def _as_stored(t):
    """`t` with the values that its memory holds: a view that stands for the negative of them (the
    imaginary part of a conjugate) is written out."""
    return t.resolve_neg() if t.is_neg() else t


def _pitch(t):
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _result(out, shape, like, dtype, beta):
    """(tensor the kernels write, its address, its pitch) for the result of a call: a new tensor,
    `out` itself, or (when the kernels cannot write it as it lies) a contiguous stand-in, which
    _finish copies into `out`.  `like`: a tensor on the device."""
    if out is None:
        if beta != 0:
            raise ValueError("beta != 0 requires out= holding the rows to scale")
        out = like.new_empty(shape, dtype=dtype)
        return out, out.data_ptr(), shape[-1]
    if tuple(out.shape) != tuple(shape) or out.dtype != dtype:
        raise ValueError("out shape/dtype must match result")
    flat = out
    if len(shape) != 2:
        try:
            flat = out.view(-1 if out.numel() else 0, shape[-1])
        except RuntimeError:
            flat = None
    if flat is None or out.is_neg() or not _row_major_ok(flat):
        flat = out.clone(memory_format=torch.contiguous_format) if beta != 0 else like.new_empty(
            shape, dtype=dtype)
        return flat, flat.data_ptr(), shape[-1]
    return flat, flat.data_ptr(), _pitch(flat)


def _finish(out, flat):
    """What the call returns: `flat` if the caller gave no `out`."""
    if out is None:
        return flat
    if out.numel() and flat.data_ptr() != out.data_ptr():
        out.copy_(flat)
    else:  # written by a kernel: tell autograd and whoever else watches the counter
        torch.autograd.graph.increment_version(out)
    return out


def _call(index, fn, *args):
    """fn(*args, current stream of device `index`) with that device current; raise on a non-zero
    status."""
    if torch.cuda.current_device() == index:
        st = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            st = fn(*args, _raw_stream(index))
    if st:
        _lib.check(st, fn.__name__)


# -------------------------------------------------------------------------------------------------
# embedding
# -------------------------------------------------------------------------------------------------
def _ignored(ignore_index):
    if ignore_index is None:
        return 0, 0
    value = _as_int(ignore_index, "ignore_index")
    if not -2**63 <= value < 2**63:
        raise ValueError("ignore_index must fit int64")
    return 1, value


def flagsparse_embedding(tokens, table, alpha=1.0, ignore_index=None, out=None, beta=0.0):
    """alpha * table[tokens] + beta * out: the rows of `table` that `tokens` names, scaled.

    tokens: integer tensor of any shape; table: (n_rows, dim), float16 / bfloat16 / float32 /
    float64.  The result has the shape tokens.shape + (dim,) and the table's dtype; the product is
    formed in float32 (float64) and rounded once.  Where a token equals `ignore_index` (any
    integer, inside the table or not) nothing is selected: the row is beta * out, zero for beta = 0.
    alpha, beta are numbers; beta != 0 needs `out`.
    Differentiable in `table` (a dense gradient, see flagsparse_embedding_grad).
    """
    if _host is not None and out is None and type(beta) in (float, int) and beta == 0:
        result = _host.embedding(tokens, table, alpha, ignore_index)
        if result is not None:
            return result
    _check_ids(tokens, "tokens")
    _check_values(table, "table")
    if table.dim() != 2:
        raise ValueError("table must be a 2D tensor: (n_rows, dim)")
    alpha = _scalar(alpha, table.dtype, "alpha")
    beta = _scalar(beta, table.dtype, "beta")
    has_ignore, ignore = _ignored(ignore_index)
    if out is not None:
        _refuse_out(out, table)
    index = _check_first_device(table, "table")
    _check_same_device(tokens, "tokens", index, "table")
    _check_same_device(out, "out", index, "table")
    if _wants_grad(table):
        _refuse_capture(index)
        if beta != 0:
            raise ValueError("beta != 0 requires out= holding the rows to scale")
        return _Embedding.apply(tokens, table, alpha, ignore_index)
    return _embedding(tokens, table, alpha, has_ignore, ignore, out, beta, index)


def _embedding(tokens, table, alpha, has_ignore, ignore, out, beta, index):
    n_rows, dim = table.shape
    n = tokens.numel()
    if n > MAX_ENTRIES or n_rows > MAX_ROWS or dim > MAX_DIM:
        _check_size("the number of tokens", n, MAX_ENTRIES)
        _check_size("the number of rows of table", n_rows, MAX_ROWS)
        _check_size("dim", dim, MAX_DIM)
    flat, address, pitch = _result(out, (*tokens.shape, dim), table, table.dtype, beta)
    if not tokens.is_contiguous():
        tokens = tokens.contiguous()
    if out is not None:
        _refuse_overlap(out, table, tokens)
    table = _rows(table)
    _call(index, _lib.load().b2s_select_rows, _lib.VALUE_CODE[table.dtype],
          _lib.INDEX_CODE[tokens.dtype], tokens.data_ptr(), n, has_ignore, ignore,
          table.data_ptr(), n_rows, _pitch(table), dim, address, pitch, alpha, beta,
          _status_word(index))
    return flat if out is None else _finish(out, flat)


def flagsparse_embedding_grad(tokens, grad, n_rows, alpha=1.0, ignore_index=None, out=None,
                              beta=0.0, out_dtype=None):
    """alpha * (sum of grad over equal tokens) + beta * out: the gradient of an embedding table
    of `n_rows` rows from the gradient of its looked-up rows.

    grad: tokens.shape + (dim,).  The result is (n_rows, dim), of grad's dtype or, for float16 and
    bfloat16, of float32 (`out_dtype`, or the dtype of `out`).  beta = 0 writes every row (zero
    where no token names it); beta = 1 adds to `out` and touches the named rows only.
    The tokens are sorted, and the rows of one token are summed in float32 (float64) in a fixed
    order: the result is the same from run to run.  The call itself is not differentiable.
    """
    if _host is not None:
        result = _host.embedding_grad(tokens, grad, n_rows, alpha, ignore_index, out, beta,
                                      out_dtype)
        if result is not None:
            return result
    _check_ids(tokens, "tokens")
    _check_values(grad, "grad")
    n_rows = _as_int(n_rows, "n_rows")
    if n_rows < 0:
        raise ValueError("n_rows must be non-negative")
    shape = grad.shape
    if len(shape) != tokens.dim() + 1 or shape[:-1] != tokens.shape:
        raise ValueError(f"grad shape must be tokens.shape + (dim,), got {tuple(shape)} for "
                         f"tokens of shape {tuple(tokens.shape)}")
    dtype = grad.dtype
    if out_dtype is None:
        out_dtype = dtype if out is None else out.dtype
    if out_dtype != dtype and not (out_dtype == torch.float32 and grad.element_size() == 2):
        raise TypeError("out dtype must be the dtype of grad, or float32 for float16 / bfloat16")
    alpha = _scalar(alpha, dtype, "alpha")
    beta = _scalar(beta, dtype, "beta")
    has_ignore, ignore = _ignored(ignore_index)
    if out is not None:
        _refuse_out(out, grad)
    index = _check_first_device(grad, "grad")
    _check_same_device(tokens, "tokens", index, "grad")
    _check_same_device(out, "out", index, "grad")
    dim = shape[-1]
    n = tokens.numel()
    _check_size("the number of tokens", n, MAX_ENTRIES)
    _check_size("n_rows", n_rows, MAX_ROWS)
    _check_size("dim", dim, MAX_DIM)
    flat, address, pitch = _result(out, (n_rows, dim), grad, out_dtype, beta)
    if out is not None:     # (the tokens have been read before a row is written)
        _refuse_overlap(out, grad)
    if not tokens.is_contiguous():
        tokens = tokens.contiguous()
    grad = _rows(grad if grad.dim() == 2 else grad.reshape(n, dim))
    lib = _lib.load()
    vcode = _lib.VALUE_CODE[dtype]
    nbytes = lib.b2s_select_grad_bytes(vcode, n, n_rows, dim)
    ws = grad.new_empty(nbytes, dtype=torch.uint8)
    _call(index, lib.b2s_select_grad, vcode, _lib.VALUE_CODE[out_dtype],
          _lib.INDEX_CODE[tokens.dtype], tokens.data_ptr(), n, has_ignore, ignore,
          grad.data_ptr(), _pitch(grad), n_rows, dim, address, pitch, alpha, beta,
          ws.data_ptr(), nbytes, _status_word(index))
    return flat if out is None else _finish(out, flat)


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, table, alpha, ignore_index):   # (gradients are disabled in here)
        ctx.save_for_backward(tokens)
        ctx.args = (table.shape[0], alpha, ignore_index)
        return flagsparse_embedding(tokens, table, alpha, ignore_index)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        _refuse_capture(grad.get_device())
        n_rows, alpha, ignore = ctx.args
        grad_table = flagsparse_embedding_grad(ctx.saved_tensors[0], grad, n_rows, alpha=alpha,
                                               ignore_index=ignore)
        return None, grad_table, None, None


# -------------------------------------------------------------------------------------------------
# tokens to experts and back
# -------------------------------------------------------------------------------------------------
class TokenRoute:
    """Where every assignment of a token to an expert stands when they are sorted by expert.

    slots    int32 (n_tokens, k): the row of assignment (t, j) among the sorted rows, -1 if masked
    indptr   int32 (n_experts + 1,): the rows of expert e are indptr[e] .. indptr[e + 1] - 1
    indices  int32 (n_tokens * k,): the token of each row (of the first indptr[-1] rows)

    (indptr, indices) is the experts x tokens matrix of the route in CSR form.  Masked assignments
    have no row: the rows from indptr[-1] on belong to nobody and are kept zero.
    """

    __slots__ = ("n_tokens", "k", "n_experts", "_buffer", "_stream", "_views")

    def __init__(self, buffer, n_tokens, k, n_experts, stream):
        """`buffer` (int32): slots, indptr and indices one behind the other."""
        self.n_tokens, self.k, self.n_experts = n_tokens, k, n_experts
        self._buffer, self._stream = buffer, stream
        self._views = {}

    @property
    def n_rows(self):
        """Rows of the sorted array: n_tokens * k, whatever is masked."""
        return self.n_tokens * self.k

    @property
    def device(self):
        return self._buffer.device

    @property
    def _index(self):
        return self._buffer.get_device()

    @property
    def _address(self):     # of slots
        return self._buffer.data_ptr()

    @property
    def _held(self):        # of indptr[-1]
        return self._buffer.data_ptr() + 4 * (self.n_tokens * self.k + self.n_experts)

    def _view(self, which, shape, stride, at):
        view = self._views.get(which)
        if view is None:
            view = self._views[which] = self._buffer.as_strided(shape, stride, at)
        return view

    @property
    def slots(self):
        return self._view(0, (self.n_tokens, self.k), (self.k, 1), 0)

    @property
    def indptr(self):
        return self._view(1, (self.n_experts + 1,), (1,), self.n_rows)

    @property
    def indices(self):
        return self._view(2, (self.n_rows,), (1,), self.n_rows + self.n_experts + 1)

    def _use(self):
        """Called before a launch: keeps the arrays from being reused while a stream other than
        the one they were made on still reads them."""
        if _raw_stream(self._index) != self._stream:
            if not _capturing(self._index):
                self._buffer.record_stream(torch.cuda.current_stream(self._index))

    def __repr__(self):
        return (f"TokenRoute(n_tokens={self.n_tokens}, k={self.k}, n_experts={self.n_experts}, "
                f"device={self.device})")


def prepare_token_route(experts, n_experts):
    """Sort the assignments experts[t, j] (int32 / int64, -1: masked) by expert, keeping their
    order within an expert, and return the TokenRoute.  Nothing is read back to the host."""
    if _host is not None:
        made = _host.route_plan(experts, n_experts)
        if made is not None:
            n_tokens, k = experts.shape
            return TokenRoute(made[0], n_tokens, k, n_experts, made[1])
    _check_ids(experts, "experts")
    if experts.dim() != 2:
        raise ValueError("experts must be a 2D tensor: (n_tokens, k)")
    n_experts = _as_int(n_experts, "n_experts")
    if not 0 <= n_experts <= MAX_EXPERTS:
        raise ValueError(f"n_experts must be between 0 and {MAX_EXPERTS}, got {n_experts}")
    n_tokens, k = experts.shape
    n = n_tokens * k
    _check_size("n_tokens * k", n, MAX_ENTRIES)
    index = _check_first_device(experts, "experts")
    if not experts.is_contiguous():
        experts = experts.contiguous()
    lib = _lib.load()
    nbytes = lib.b2s_route_plan_bytes(n_tokens, k, n_experts)
    scratch = -(-(2 * n + n_experts + 1) // 64) * 64     # behind the arrays, 256-byte aligned
    buffer = experts.new_empty(scratch + nbytes // 4, dtype=torch.int32)
    stream = _raw_stream(index)
    route = TokenRoute(buffer, n_tokens, k, n_experts, stream)
    address = route._address
    _call(index, lib.b2s_route_plan, _lib.INDEX_CODE[experts.dtype], experts.data_ptr(), n_tokens,
          k, n_experts, address, address + 4 * n, route._held + 4, address + 4 * scratch, nbytes,
          _status_word(index))
    return route


def _check_route(route):
    if not isinstance(route, TokenRoute):
        raise TypeError("route must be a TokenRoute (prepare_token_route)")


def _check_matrix(t, name, rows, what):
    _check_values(t, name)
    if t.dim() != 2:
        raise ValueError(f"{name} must be a 2D tensor: ({what}, dim)")
    if t.shape[0] != rows:
        raise ValueError(f"{name}.shape[0] must be {what}={rows}, got {t.shape[0]}")
    _check_size("dim", t.shape[1], MAX_DIM)


def _check_weights(weights, route, dtype):
    if weights is None:
        return
    _check_values(weights, "weights")
    if weights.dtype != dtype and weights.dtype != torch.float32:
        raise TypeError("weights dtype must be the dtype of the rows, or float32")
    if tuple(weights.shape) != (route.n_tokens, route.k):
        raise ValueError(f"weights shape must be {(route.n_tokens, route.k)}, got "
                         f"{tuple(weights.shape)}")


def flagsparse_token_dispatch(x, route, out=None):
    """The tokens' rows sorted by expert: row route.slots[t, j] of the result is x[t].

    x: (n_tokens, dim); the result is (n_tokens * k, dim) of x's dtype, its rows from
    route.indptr[-1] on (left by masked assignments) zero.  Differentiable in x.
    """
    _check_route(route)
    if _host is not None and out is None:
        result = _host.dispatch(route._buffer, route.n_tokens, route.k, route.n_experts,
                                route._stream, x)
        if result is not None:
            return result
    _check_matrix(x, "x", route.n_tokens, "n_tokens")
    if out is not None:
        _refuse_out(out, x)
    index = _check_first_device(route._buffer, "route")
    _check_same_device(x, "x", index, "route")
    _check_same_device(out, "out", index, "route")
    if _wants_grad(x):
        _refuse_capture(index)
        return _Dispatch.apply(x, route)
    return _dispatch(x, route, out)


def _dispatch(x, route, out):
    dim = x.shape[1]
    flat, address, pitch = _result(out, (route.n_rows, dim), x, x.dtype, 0.0)
    if out is not None:
        _refuse_overlap(out, x, route._buffer)
    x = _rows(x)
    route._use()
    _call(route._index, _lib.load().b2s_route_dispatch, _lib.VALUE_CODE[x.dtype], x.data_ptr(),
          _pitch(x), route.n_tokens, route.k, dim, route._address, route._held, address, pitch)
    return flat if out is None else _finish(out, flat)


def flagsparse_token_dispatch_grad(grad, route, out=None, beta=0.0):
    """The gradient of flagsparse_token_dispatch: row t is the sum of grad[route.slots[t, j]] over
    the j that are not masked (float32 / float64 sums, one rounding), plus beta * out.

    grad: (n_tokens * k, dim); its rows from route.indptr[-1] on are not read.  The call itself is
    not differentiable.
    """
    _check_route(route)
    if _host is not None and out is None and type(beta) in (float, int) and beta == 0:
        result = _host.combine(route._buffer, route.n_tokens, route.k, route.n_experts,
                               route._stream, grad, None, 1.0)
        if result is not None:
            return result
    _check_matrix(grad, "grad", route.n_rows, "n_tokens * k")
    beta = _scalar(beta, grad.dtype, "beta")
    if out is not None:
        _refuse_out(out, grad)
    index = _check_first_device(route._buffer, "route")
    _check_same_device(grad, "grad", index, "route")
    _check_same_device(out, "out", index, "route")
    return _combine(grad, route, None, 1.0, out, beta)


def flagsparse_token_combine(y, route, weights=None, alpha=1.0, out=None, beta=0.0):
    """The rows of each token brought back and summed with their weights:
    alpha * sum_j weights[t, j] * y[route.slots[t, j]] + beta * out[t], without the masked j.

    y: (n_tokens * k, dim); weights: (n_tokens, k) of y's dtype or float32, None for ones.  The
    result is (n_tokens, dim) of y's dtype: float32 (float64) sums, one rounding; a token whose
    assignments are all masked gets beta * out, whatever alpha is.  Differentiable in y and weights.
    """
    _check_route(route)
    if _host is not None and out is None and type(beta) in (float, int) and beta == 0:
        result = _host.combine(route._buffer, route.n_tokens, route.k, route.n_experts,
                               route._stream, y, weights, alpha)
        if result is not None:
            return result
    _check_matrix(y, "y", route.n_rows, "n_tokens * k")
    _check_weights(weights, route, y.dtype)
    alpha = _scalar(alpha, y.dtype, "alpha")
    beta = _scalar(beta, y.dtype, "beta")
    if out is not None:
        _refuse_out(out, y, weights)
    index = _check_first_device(route._buffer, "route")
    _check_same_device(y, "y", index, "route")
    _check_same_device(weights, "weights", index, "route")
    _check_same_device(out, "out", index, "route")
    if _wants_grad(y, weights):
        _refuse_capture(index)
        if beta != 0:
            raise ValueError("beta != 0 requires out= holding the rows to scale")
        return _Combine.apply(y, weights, route, alpha)
    return _combine(y, route, weights, alpha, out, beta)


def _combine(y, route, weights, alpha, out, beta):
    dim = y.shape[1]
    flat, address, pitch = _result(out, (route.n_tokens, dim), y, y.dtype, beta)
    if out is not None:
        _refuse_overlap(out, y, weights, route._buffer)
    y = _rows(y)
    wcode, waddress = 0, None
    if weights is not None:
        weights = _as_stored(weights).contiguous()
        wcode, waddress = _lib.VALUE_CODE[weights.dtype], weights.data_ptr()
    route._use()
    _call(route._index, _lib.load().b2s_route_combine, _lib.VALUE_CODE[y.dtype], y.data_ptr(),
          _pitch(y), route._address, wcode, waddress, route.n_tokens, route.k, dim, address, pitch,
          alpha, beta)
    return flat if out is None else _finish(out, flat)


def flagsparse_token_combine_grad(grad, y, route, weights=None, alpha=1.0):
    """The gradients of flagsparse_token_combine: (grad_y, grad_weights).

    grad: (n_tokens, dim).  grad_y[route.slots[t, j]] = alpha * weights[t, j] * grad[t] (rows that
    belong to nobody are zero); grad_weights[t, j] = alpha * <grad[t], y[route.slots[t, j]]> in the
    dtype of weights, zero where masked.  Without weights, y may be None and grad_weights is None.
    The call itself is not differentiable.
    """
    _check_route(route)
    if _host is not None and weights is not None:
        result = _host.combine_grad(route._buffer, route.n_tokens, route.k, route.n_experts,
                                    route._stream, grad, y, weights, alpha)
        if result is not None:
            return result
    _check_matrix(grad, "grad", route.n_tokens, "n_tokens")
    _check_weights(weights, route, grad.dtype)
    if weights is not None:
        if y is None:
            raise ValueError("y is needed for the gradient of weights")
    if y is not None:
        _check_matrix(y, "y", route.n_rows, "n_tokens * k")
        if y.dtype != grad.dtype:
            raise TypeError("y dtype must match grad dtype")
        if y.shape[1] != grad.shape[1]:
            raise ValueError("y and grad must have the same number of columns")
    alpha = _scalar(alpha, grad.dtype, "alpha")
    index = _check_first_device(route._buffer, "route")
    _check_same_device(grad, "grad", index, "route")
    _check_same_device(y, "y", index, "route")
    _check_same_device(weights, "weights", index, "route")
    return _combine_grad(grad, y, route, weights, alpha, weights is not None)


def _combine_grad(grad, y, route, weights, alpha, want_weights):
    dim = grad.shape[1]
    grad = _rows(grad)
    grad_y = grad.new_empty((route.n_rows, dim))
    grad_w, wcode, waddress, gaddress = None, 0, None, None
    yaddress, ypitch = None, 0
    if weights is not None:
        weights = _as_stored(weights).contiguous()
        wcode, waddress = _lib.VALUE_CODE[weights.dtype], weights.data_ptr()
        if want_weights:
            y = _rows(y)
            yaddress, ypitch = y.data_ptr(), _pitch(y)
            grad_w = weights.new_empty((route.n_tokens, route.k))
            gaddress = grad_w.data_ptr()
    route._use()
    _call(route._index, _lib.load().b2s_route_combine_grad, _lib.VALUE_CODE[grad.dtype],
          grad.data_ptr(), _pitch(grad), yaddress, ypitch, route._address, route._held, wcode,
          waddress, route.n_tokens, route.k, dim, alpha, grad_y.data_ptr(), dim, gaddress)
    return grad_y, grad_w


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, route):
        ctx.route = route
        return flagsparse_token_dispatch(x, route)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        _refuse_capture(grad.get_device())
        return flagsparse_token_dispatch_grad(grad, ctx.route), None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weights, route, alpha):
        ctx.route, ctx.alpha = route, alpha
        wants_weights = ctx.needs_input_grad[1]
        ctx.wants_weights = wants_weights
        # y is read by the gradient of the weights only
        ctx.save_for_backward(y if wants_weights else None, weights)
        return flagsparse_token_combine(y, route, weights, alpha)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        _refuse_capture(grad.get_device())
        y, weights = ctx.saved_tensors
        if ctx.wants_weights:
            grad_y, grad_w = flagsparse_token_combine_grad(grad, y, ctx.route, weights, ctx.alpha)
        else:
            grad_y, grad_w = _combine_grad(grad, None, ctx.route, weights, ctx.alpha, False)
        return grad_y, grad_w, None, None
