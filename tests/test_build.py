"""What each part of the build needs, and what is rebuilt when."""
import subprocess
import sysconfig

import numpy as np
import pytest
import torch

from rnn_kernel_b200 import _lib, build, optim


@pytest.fixture
def no_compiler(monkeypatch, tmp_path):
    """No module for this torch, and nothing to build one with; the library is as built."""
    _lib.load()
    monkeypatch.setattr(build, "host_path", lambda: tmp_path / "_host.so")

    def run(cmd, **kw):
        raise subprocess.CalledProcessError(1, cmd)

    monkeypatch.setattr(build.subprocess, "run", run)
    monkeypatch.setattr(_lib, "_lib", None)
    monkeypatch.setattr(_lib, "_host", None)
    optim._reader.cache_clear()
    yield
    optim._reader.cache_clear()


def test_the_library_needs_no_cpp_module(no_compiler):
    assert not build.needs_build()
    assert _lib.load().gru_stash_bytes(1, 2, 3) > 0


def test_adamw_reads_in_python_where_the_module_cannot_be_built(no_compiler):
    with pytest.raises(subprocess.CalledProcessError):
        _lib.host()
    with pytest.warns(UserWarning, match="in Python"):
        assert optim._reader() is None


def test_the_module_belongs_to_one_torch_and_one_python(monkeypatch):
    here = build.host_path()
    assert torch.__version__ in here.name and here.name.endswith(sysconfig.get_config_var("EXT_SUFFIX"))
    monkeypatch.setattr(torch, "__version__", "99.0")
    assert build.host_path() != here


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_python_and_cpp_readers_step_alike(no_compiler, bits, monkeypatch):
    def run():
        torch.manual_seed(0)
        ps = [torch.nn.Parameter(torch.randn(n, device="cuda")) for n in (300, 7, 2049)]
        opt = optim.AdamW(ps, lr=1e-2, state_bits=bits)
        for t in range(3):
            for p in ps:
                p.grad = torch.randn_like(p)
            opt.step()
        return [p.detach() for p in ps], opt

    with pytest.warns(UserWarning, match="in Python"):
        slow, opt = run()
    assert opt._tables[0].addresses is None
    monkeypatch.undo()
    optim._reader.cache_clear()
    fast, opt = run()
    assert opt._tables[0].addresses is not None
    assert all(np.array_equal(a.cpu(), b.cpu()) for a, b in zip(slow, fast))
