"""A copied or unpickled AdamW is an optimizer of its own: it reads and writes none of the original's memory."""
import copy
import io
import pickle
import types

import numpy as np
import pytest
import torch

from rnn_kernel_b200 import AdamW, optim

SIZES = [300, 5, 2049]


def by_pickle(x):
    return pickle.loads(pickle.dumps(x))


def by_torch_save(x):
    f = io.BytesIO()
    torch.save(x, f)
    f.seek(0)
    return torch.load(f, weights_only=False)


COPIES = [copy.deepcopy, by_pickle, by_torch_save]


@pytest.mark.parametrize("make", [copy.copy, *COPIES])
def test_table_points_at_its_own_entries(make):
    params = [torch.nn.Parameter(torch.zeros(n)) for n in SIZES]
    owner = types.SimpleNamespace(params=params, _sizes=np.array(SIZES), _offsets=np.array([0, 512, 768]))
    table = optim._TypeTable(owner, torch.float32, np.zeros(3, dtype=np.int64))
    other = make(table)
    assert other.address == other.entries.ctypes.data
    assert table.address == table.entries.ctypes.data
    assert other.entries.tolist() == table.entries.tolist()


def fresh(**kw):
    torch.manual_seed(1)
    ps = [torch.nn.Parameter(torch.randn(n, device="cuda")) for n in SIZES]
    return ps, AdamW(ps, lr=1e-2, **kw)


def gradients(ps, step):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(step)
    for p in ps:
        p.grad = torch.randn(p.shape, device="cuda", generator=gen)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("steps", [0, 2])
@pytest.mark.parametrize("make", COPIES)
def test_copy_steps_as_the_original_would(make, steps, bits):
    ps, opt = fresh(state_bits=bits, seed=5)
    for t in range(steps):
        gradients(ps, t)
        opt.step()
    other = make(opt)
    mine = other.params
    start = [p.detach().clone() for p in ps]
    assert all(p.data_ptr() != q.data_ptr() and torch.equal(p, q) for p, q in zip(ps, mine))
    # the copy first: the original's tensors and table stay as they are
    for t in range(steps, steps + 3):
        gradients(mine, t)
        other.step()
    assert all(torch.equal(p.detach(), s) for p, s in zip(ps, start))
    for t in range(steps, steps + 3):
        gradients(ps, t)
        opt.step()
    for p, q in zip(ps, mine):
        assert torch.equal(p.detach(), q.detach())
    assert all(torch.equal(a, b) for a, b in zip(opt.moments(), other.moments()))
