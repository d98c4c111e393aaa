"""The Python host's side of a call without a GPU: where scratch memory comes from."""
import contextlib
import types

import pytest
import torch

from ax_dsl_kernels_b200 import _lib


class FakeCuda:
    """two devices, streams by handle (0: the default one), some of them capturing; records what is allocated where"""

    def __init__(self, monkeypatch, capturing=()):
        self.dev, self.stream, self.capturing, self.made = 0, {0: 0, 1: 0}, set(capturing), []
        for name, f in (("current_device", lambda: self.dev),
                        ("is_current_stream_capturing", lambda: (self.dev, self.stream[self.dev]) in self.capturing),
                        ("ExternalStream", self.external), ("default_stream", lambda d: types.SimpleNamespace(handle=0, dev=d)),
                        ("stream", self.use)):
            monkeypatch.setattr(torch.cuda, name, f)
        monkeypatch.setattr(torch, "empty", self.empty)
        monkeypatch.setattr(_lib, "_raw_stream", lambda d: self.stream[d])
        monkeypatch.setattr(_lib, "_ws_cache", {})

    @staticmethod
    def external(handle, device):
        assert handle, "handle 0 would name a stream of the pool"
        return types.SimpleNamespace(handle=handle, dev=device)

    @contextlib.contextmanager
    def use(self, s):
        old = self.dev, self.stream[s.dev]
        self.dev, self.stream[s.dev] = s.dev, s.handle
        try:
            yield
        finally:
            self.dev, self.stream[s.dev] = old

    def empty(self, n, dtype=None, device=None):
        self.made.append((device.index, self.stream[device.index], n))
        address = 4096 * len(self.made)
        return types.SimpleNamespace(numel=lambda: n, data_ptr=lambda: address)


MB = 1 << 20


@pytest.mark.parametrize("dev,handle", [(0, 0), (0, 7), (1, 0), (1, 7)])
@pytest.mark.parametrize("current", [0, 5])
def test_scratch_belongs_to_the_stream_of_the_call(monkeypatch, dev, handle, current):
    cuda = FakeCuda(monkeypatch)
    cuda.stream[0] = current
    at, _ = _lib._scratch(dev, 10, handle)
    assert cuda.made == [(dev, handle, MB)]
    assert _lib._scratch(dev, MB, handle)[0] == at and len(cuda.made) == 1  # kept
    assert _lib._scratch(dev, MB + 1, handle)[0] != at
    assert cuda.made[1:] == [(dev, handle, MB + 1)]  # the old buffer goes back to this stream's memory too
    assert (cuda.dev, cuda.stream[0]) == (0, current)


@pytest.mark.parametrize("dev,handle,current", [(0, 7, 0), (0, 7, 5), (1, 7, 0), (1, 7, 7), (0, 5, 5)])
def test_a_capture_on_the_calls_stream_takes_the_graphs_memory(monkeypatch, dev, handle, current):
    """whatever stream and device are current"""
    cuda = FakeCuda(monkeypatch, capturing=[(dev, handle)])
    cuda.stream[dev] = current
    _lib._scratch(dev, 10, handle)
    _lib._scratch(dev, 20, handle)
    assert cuda.made == [(dev, handle, 10), (dev, handle, 20)] and not _lib._ws_cache


@pytest.mark.parametrize("handle", [0, 7])
def test_a_capture_on_another_stream_is_no_matter(monkeypatch, handle):
    """the current stream captures, the call goes elsewhere: its buffer is that stream's, not the graph's"""
    cuda = FakeCuda(monkeypatch, capturing=[(0, 5)])
    cuda.stream[0] = 5
    at = _lib._scratch(0, 10, handle)[0]
    assert cuda.made == [(0, handle, MB)] and _lib._ws_cache[0, handle][1] == at


@pytest.mark.parametrize("current,capturing", [(0, [(1, 0)]), (0, [(0, 0)]), (1, [(1, 0)]), (1, [])])
def test_counts_first_used_in_a_capture_on_another_device(monkeypatch, current, capturing):
    """(first, last) pairs of select_pages and evict_keys: copied from the host and kept, or set by the graph that the tensors'
    device captures"""
    from ax_dsl_kernels_b200 import long_context as lc
    cuda = FakeCuda(monkeypatch, capturing)
    cuda.dev = current

    @contextlib.contextmanager
    def device(d):
        old, cuda.dev = cuda.dev, d
        yield
        cuda.dev = old

    class Filled:
        def __getitem__(self, _):
            return self

        def fill_(self, _):
            made.append("set by the graph")

    made = []
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch, "tensor", lambda *a, **k: made.append("copied"))
    monkeypatch.setattr(torch, "full", lambda *a, **k: Filled())
    monkeypatch.setattr(lc, "_keep", {})
    lc._keep_pair(6, 2, torch.device("cuda", 1))
    assert made == ["set by the graph" if (1, 0) in capturing else "copied"]
    assert bool(lc._keep) == ((1, 0) not in capturing) and cuda.dev == current


# ------------------------------------------------------------------------------------------- the fast path and its build
def test_the_fast_path_of_another_torch_is_not_used(monkeypatch):
    import sys

    import ax_dsl_kernels_b200 as q35
    other = types.SimpleNamespace(built_for="1.0.0", init=lambda *a: pytest.fail("initialised"), run=None)
    monkeypatch.setitem(sys.modules, "ax_dsl_kernels_b200._bind", other)
    monkeypatch.setattr(q35, "_bind", other, raising=False)
    assert _lib._fast_run() is _lib.run_checked


def test_the_fast_path_is_built_for_this_torch():
    _bind = pytest.importorskip("ax_dsl_kernels_b200._bind")
    assert _bind.built_for == torch.__version__
    assert _lib._fast_run() is _bind.run


def build_in(monkeypatch, tmp_path, compiler):
    from ax_dsl_kernels_b200 import build
    source = tmp_path / "bind.cc"
    source.write_text("")
    monkeypatch.setattr(build, "HERE", str(tmp_path))
    monkeypatch.setattr(build, "OBJ", str(tmp_path))
    monkeypatch.setattr(build, "BIND", str(tmp_path / "_bind.this.so"))
    monkeypatch.setattr(build.subprocess, "run", compiler)
    return lambda **k: build.binding([str(source)], **k)


def test_a_binding_that_does_not_compile_is_a_warning(monkeypatch, tmp_path):
    binding = build_in(monkeypatch, tmp_path, lambda *a, **k: types.SimpleNamespace(returncode=1, stdout="", stderr="no such header"))
    (tmp_path / "_bind.this.so").write_text("of an older torch")
    with pytest.warns(UserWarning, match="no such header"):
        binding()
    assert not (tmp_path / "_bind.this.so").exists()  # nothing old is left to be imported

    def no_compiler(*a, **k):
        raise FileNotFoundError("g++")

    binding = build_in(monkeypatch, tmp_path, no_compiler)
    with pytest.warns(UserWarning, match="g[+][+]"):
        binding()


def test_another_torch_makes_the_binding_stale(monkeypatch, tmp_path):
    built = []

    def compiler(cmd, **k):
        built.append(torch.__version__)
        assert f'-DQ35_BUILT_FOR="{torch.__version__}"' in cmd
        (tmp_path / "_bind.this.so").write_text("")
        return types.SimpleNamespace(returncode=0, stdout="", stderr="")

    binding = build_in(monkeypatch, tmp_path, compiler)
    (tmp_path / "_bind.so").write_text("for any Python")
    here = torch.__version__
    binding()
    binding()
    assert built == [here] and not (tmp_path / "_bind.so").exists()
    monkeypatch.setattr(torch, "__version__", "99.0")
    binding()
    binding()
    assert built == [here, "99.0"]
    binding(force=True)
    assert len(built) == 3
