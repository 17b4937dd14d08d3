"""Selection products on the CPU: calls beside the usual one, up to where the device begins."""

import contextlib
import shutil
import subprocess
import sys
from types import SimpleNamespace

import pytest
import torch

import flagsparse_b200 as fs
from conftest import ROOT
from flagsparse_b200 import _lib, selection

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
    view = z.conj().imag                                 # rows that a kernel could read as they lie
    assert view.is_neg() and selection._row_major_ok(view)
    same = torch._neg_view((-view).resolve_neg())
    for rows in (selection._rows(view), selection._as_stored(same)):
        assert not rows.is_neg() and torch.equal(rows, view)
    assert selection._rows(TABLE) is TABLE
    flat, address, _ = selection._result(view, (6, 1), view, torch.float32, 1.0)
    assert address != view.data_ptr() and not flat.is_neg() and torch.equal(flat, view)
    flat.fill_(5.0)
    assert selection._finish(view, flat) is view and (view == 5).all() and (z.imag == -5).all()


def test_overlap_is_a_matter_of_addresses():
    wide = torch.zeros(6, 10)

    def refuse(*tensors):
        with pytest.raises(ValueError, match="must not overlap"):
            selection._refuse_overlap(*tensors)

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


def _run(code, cwd):
    return subprocess.run([sys.executable, "-c", code], cwd=cwd, capture_output=True, text=True,
                          timeout=300)


def test_importing_the_package_loads_no_library():
    """The libraries come with the first call: whoever imports the package for something else (its
    build command, a workload's description) does not depend on them."""
    res = _run("import flagsparse_b200, flagsparse_b200._build\n"
               "maps = open('/proc/self/maps').read()\n"
               "assert 'libb200sparse' not in maps and '_b2s_host' not in maps\n"
               "from flagsparse_b200 import selection\n"
               "assert selection._host.embedding(1, 2, 3) is None\n"
               "maps = open('/proc/self/maps').read()\n"
               "assert 'libb200sparse' in maps and '_b2s_host' in maps\n", ROOT)
    assert res.returncode == 0, res.stderr[-1500:]


def test_a_library_without_an_entry_point_can_be_built_anew(tmp_path):
    """Importing the package, and with it the build command, works beside a library that is older
    than its declarations; the first call says what the library lacks."""
    package = tmp_path / "flagsparse_b200"
    package.mkdir()
    for path in (ROOT / "flagsparse_b200").iterdir():
        if path.suffix == ".py":
            shutil.copy(path, package / path.name)
        elif path.suffix == ".so":
            (package / path.name).symlink_to(path)
    with open(package / "_lib.py", "a") as f:
        f.write("\nSIGNATURES['b2s_of_a_later_version'] = (c_int, [])\n")
    res = _run("import torch, flagsparse_b200, flagsparse_b200._build\n"
               "assert flagsparse_b200.__file__.startswith(%r)\n"
               "try:\n"
               "    flagsparse_b200.flagsparse_embedding(torch.zeros(1).long(), torch.zeros(1, 1))\n"
               "except AttributeError as e:\n"
               "    print(e)\n" % str(tmp_path), tmp_path)
    assert res.returncode == 0 and "b2s_of_a_later_version" in res.stdout, res.stderr[-1500:]


def test_without_the_host_module_or_the_library(tmp_path, monkeypatch):
    monkeypatch.setitem(sys.modules, "flagsparse_b200._b2s_host", None)    # an ImportError
    monkeypatch.delattr(fs, "_b2s_host", raising=False)
    monkeypatch.setattr(selection, "_host", selection._Host())
    assert selection._host.embedding(TOK, TABLE, 1.0, None) is None
    assert selection._host is selection._NO_HOST             # for good: no call asks again
    assert selection._host.bind_status(0, 0) is None
    monkeypatch.setattr(selection, "_host", selection._Host())
    monkeypatch.setattr(_lib, "LIB_PATH", tmp_path / "libb200sparse.so")
    assert selection._host.combine() is None and type(selection._host) is selection._Host


def test_a_host_module_of_another_pytorch_is_not_used(monkeypatch):
    """It reads PyTorch's structures by the headers it was built with."""
    other = SimpleNamespace(torch_version="1.0", bind=lambda *a: pytest.fail("called"))
    monkeypatch.setitem(sys.modules, "flagsparse_b200._b2s_host", other)
    monkeypatch.setattr(fs, "_b2s_host", other, raising=False)
    monkeypatch.setattr(selection, "_host", selection._Host())
    with pytest.warns(UserWarning, match="built for PyTorch 1.0"):
        assert selection._host.embedding(TOK, TABLE, 1.0, None) is None
    assert selection._host is selection._NO_HOST


def test_the_host_module_is_built_anew_for_another_pytorch(monkeypatch, tmp_path):
    from flagsparse_b200 import _build
    built = []

    def run(cmd, **kwargs):
        built.append(cmd)
        return SimpleNamespace(returncode=0, stdout="", stderr="")

    lib = tmp_path / "_b2s_host.so"
    monkeypatch.setattr(_build, "HOST_LIB_PATH", lib)
    monkeypatch.setattr(_build, "BUILD_DIR", tmp_path / "build")
    monkeypatch.setattr(_build.subprocess, "run", run)
    monkeypatch.setattr(_build, "_nvcc", lambda: "/usr/local/cuda/bin/nvcc")
    _build.build_host()
    assert len(built) == 1 and f'-DB2S_TORCH_VERSION="{torch.__version__}"' in built[0]
    lib.touch()
    _build.build_host()
    assert len(built) == 1                                   # nothing has changed
    monkeypatch.setattr(torch, "__version__", "99.0")
    _build.build_host()
    assert len(built) == 2 and '-DB2S_TORCH_VERSION="99.0"' in built[1]


class _FakeCuda:
    """Two devices; the current stream of the second is captured."""

    def __init__(self, monkeypatch):
        self.index = 0
        for name in ("current_device", "is_current_stream_capturing", "device"):
            monkeypatch.setattr(torch.cuda, name, getattr(self, name))

    def current_device(self):
        return self.index

    def is_current_stream_capturing(self):
        return self.index == 1

    @contextlib.contextmanager
    def device(self, index):
        before, self.index = self.index, index
        yield
        self.index = before


def test_the_stream_of_the_tensors_decides_whether_it_is_a_capture(monkeypatch):
    """Recorded calls are refused where their own device's stream is captured, whichever device is
    current; and a route's memory is not marked as used by a stream that is."""
    cuda = _FakeCuda(monkeypatch)
    monkeypatch.setattr(selection, "_check_first_device", lambda t, name: 1)
    monkeypatch.setattr(selection, "_check_same_device", lambda *args: None)
    x, y = torch.zeros(3, 4).requires_grad_(), torch.zeros(6, 4).requires_grad_()
    for current in (0, 1):
        cuda.index = current
        for call in (lambda: fs.flagsparse_embedding(TOK, x), lambda: fs.flagsparse_token_dispatch(
                x, _route()), lambda: fs.flagsparse_token_combine(y, _route())):
            with pytest.raises(RuntimeError, match="not recorded inside a CUDA graph capture"):
                call()
        assert cuda.index == current
    cuda.index = 1                                           # (the other device is free to record)
    assert not selection._capturing(0) and selection._capturing(1)
    marked = []
    monkeypatch.setattr(selection, "_raw_stream", lambda index: 5)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda index: "stream")
    for index, times in ((1, 0), (0, 1)):
        for cuda.index in (0, 1):
            fake = SimpleNamespace(get_device=lambda: index, record_stream=marked.append)
            fs.TokenRoute(fake, 3, 2, 4, 0)._use()
        assert len(marked) == 2 * times
