"""What of the gated delta rule and AdamW needs no GPU: sizes, refusals of the C entry points and of the Python ones."""
import numpy as np
import pytest
import torch

from rnn_kernel_b200 import AdamW, DataParallelTrainer, GatedDelta, _lib, gated_delta_rule, gated_delta_step
from rnn_kernel_b200 import optim


def pack(dtype=0, B=2, T=100, Hk=2, Hv=4, dk=64, dv=64, pointers=(0,) * 6):
    return _lib.DELTA_ARGS.pack(dtype, B, T, Hk, Hv, dk, dv, 1.0, *pointers, *[0] * 15)


def test_sizes_without_gpu():
    lib = _lib.load()
    for dtype in (0, 1):
        one = lib.gru_delta_stash_bytes(pack(dtype, T=64))
        assert one > 0 and one % 256 == 0
        assert lib.gru_delta_stash_bytes(pack(dtype, T=65)) > one
        # a forward without a gradient keeps no more than a training one
        assert 0 < lib.gru_delta_workspace_bytes(pack(dtype), 0) <= lib.gru_delta_stash_bytes(pack(dtype))
        assert lib.gru_delta_workspace_bytes(pack(dtype), 1) > 0
    assert lib.gru_delta_stash_bytes(pack(T=0)) == 0
    # the states alone of this one pass 32 bits
    assert lib.gru_delta_stash_bytes(pack(B=1, T=1 << 20, Hk=16, Hv=16, dk=128, dv=128)) > 1 << 34


@pytest.mark.parametrize("bad", [dict(dtype=2), dict(B=-1), dict(T=-1), dict(Hk=0), dict(Hk=3), dict(dk=0), dict(dk=129),
                                 dict(dv=0), dict(dv=129), dict(B=1 << 20, T=1 << 20, Hk=64, Hv=64)])
def test_c_entries_refuse(bad):
    lib = _lib.load()
    a = pack(**bad)
    assert lib.gru_delta_stash_bytes(a) == 0 and _lib.last_error()
    assert lib.gru_delta_forward(a, 0, 0, 0, 0, 0, 0, 0) in (_lib.GRU_ERR_INVALID, _lib.GRU_ERR_UNSUPPORTED)
    assert lib.gru_delta_backward(a, *[0] * 3, 0, *[0] * 7, 0, 0) in (_lib.GRU_ERR_INVALID, _lib.GRU_ERR_UNSUPPORTED)
    assert lib.gru_delta_step(a, 0, 0, 0) in (_lib.GRU_ERR_INVALID, _lib.GRU_ERR_UNSUPPORTED)


def test_c_entries_refuse_null_misaligned_and_small():
    lib = _lib.load()
    p = (64,) * 6  # addresses that are never read: the calls fail before
    assert lib.gru_delta_forward(pack(), 64, 64, 64, 1 << 40, 0, 0, 0) == _lib.GRU_ERR_INVALID  # null tensors
    a = pack(pointers=p)
    assert lib.gru_delta_forward(a, 64, 0, 64, 1 << 40, 0, 0, 0) == _lib.GRU_ERR_INVALID  # no final state
    assert lib.gru_delta_forward(a, 64, 64, 64, 16, 0, 0, 0) == _lib.GRU_ERR_INVALID  # a small stash
    assert lib.gru_delta_forward(a, 64, 64, 0, 0, 64, 16, 0) == _lib.GRU_ERR_INVALID  # a small workspace
    assert lib.gru_delta_forward(a, 64, 64, 72, 1 << 40, 0, 0, 0) == _lib.GRU_ERR_INVALID  # not aligned
    assert lib.gru_delta_forward(pack(pointers=(66,) + p[1:]), 64, 64, 64, 1 << 40, 0, 0, 0) == _lib.GRU_ERR_INVALID
    assert lib.gru_delta_backward(a, 64, 64, 64, 1 << 40, 64, 64, 64, 64, 64, 64, 64, 16, 0) == _lib.GRU_ERR_INVALID
    assert lib.gru_delta_backward(a, 64, 64, 64, 1 << 40, 0, 64, 64, 64, 64, 64, 64, 1 << 40, 0) == _lib.GRU_ERR_INVALID
    assert lib.gru_delta_step(a, 64, 64, 0) == _lib.GRU_ERR_INVALID  # T is not 1
    assert "T must be 1" in _lib.last_error()
    assert lib.gru_delta_step(pack(T=1, pointers=p), 0, 64, 0) == _lib.GRU_ERR_INVALID
    # nothing to do
    assert lib.gru_delta_step(pack(T=1, B=0), 0, 0, 0) == _lib.GRU_OK
    assert lib.gru_delta_forward(pack(B=0), 0, 0, 0, 0, 0, 0, 0) == _lib.GRU_OK


def entry(**kw):
    e = np.zeros(1, dtype=optim._ENTRY)
    e["param"], e["grad"], e["n"] = 64, 64, 10
    for k, v in kw.items():
        e[k] = v
    return e


def step(e, dtype=0, bits=32, elems=256, beta1=0.9, beta2=0.999, eps=1e-8, m=64, v=64, sm=64, sv=64, step=0, scalars=0):
    return _lib.load().gru_adamw_step(e.ctypes.data, len(e), dtype, bits, m, v, sm, sv, elems, beta1, beta2, eps, 1.0, 0, 1,
                                      step, scalars, 0)


def test_adamw_c_entry_refuses():
    assert optim._ENTRY.itemsize == 48
    assert step(entry(), dtype=2) == step(entry(), bits=16) == _lib.GRU_ERR_UNSUPPORTED
    assert step(entry(), beta1=1.0) == step(entry(), eps=-1.0) == step(entry(), beta2=float("nan")) == _lib.GRU_ERR_INVALID
    assert step(entry(n=-1)) == step(entry(param=0)) == step(entry(param=66)) == _lib.GRU_ERR_INVALID
    assert step(entry(state_offset=1)) == step(entry(n=257)) == step(entry(state_offset=512)) == _lib.GRU_ERR_INVALID
    assert step(entry(), m=0) == step(entry(), v=72) == step(entry(), bits=8, sm=0) == _lib.GRU_ERR_INVALID
    assert step(entry(), step=64) == _lib.GRU_ERR_INVALID and "device_scalars" in _lib.last_error()
    assert step(entry(n=0)) == _lib.GRU_OK
    lib = _lib.load()
    assert lib.gru_adamw_decode(64, 64, 64, 64, 100, 64, 64, 0) == _lib.GRU_ERR_INVALID
    assert lib.gru_adamw_decode(64, 64, 64, 64, 256, 0, 64, 0) == _lib.GRU_ERR_INVALID
    assert lib.gru_adamw_decode(64, 64, 64, 64, 0, 0, 0, 0) == _lib.GRU_OK


def test_python_entries_refuse_cpu_tensors():
    q, v, g = torch.zeros(1, 4, 2, 8), torch.zeros(1, 4, 2, 8), torch.zeros(1, 4, 2)
    with pytest.raises(RuntimeError, match="CUDA"):
        gated_delta_rule(q, q, v, g, g)
    with pytest.raises(RuntimeError, match="CUDA"):
        gated_delta_step(q[:, 0], q[:, 0], v[:, 0], g[:, 0], g[:, 0], torch.zeros(1, 2, 8, 8))
    with pytest.raises(ValueError, match="leading"):
        gated_delta_rule(q, q, v, g[..., None], g)
    with pytest.raises(RuntimeError, match="CUDA"):
        AdamW([torch.nn.Parameter(torch.zeros(3))])
    with pytest.raises(ValueError, match="optimizer"):
        DataParallelTrainer(torch.nn.GRU(2, 2, batch_first=True), optimizer="adam")
    with pytest.raises(ValueError):
        GatedDelta(8, num_heads=2, num_key_heads=4)
    with pytest.raises(ValueError):
        GatedDelta(8, head_size=129)


def test_layer_state_dict_names():
    layer = GatedDelta(16, num_heads=4, head_size=8, num_key_heads=2, output_size=5)
    assert {k: tuple(v.shape) for k, v in layer.state_dict().items()} == {
        "in_proj.weight": (2 * 2 * 8 + 4 * 8 + 8, 16), "out_proj.weight": (5, 32), "norm_weight": (8,), "log_rate": (4,)}


def test_tensor_addresses_only_of_what_the_table_holds():
    """The C++ reader of parameters refuses, and reads nothing of, what is not a CUDA tensor of the entry's size."""
    read = _lib.host().adamw_addresses
    p = torch.nn.Parameter(torch.zeros(5))
    p.grad = torch.zeros(5)
    entries = np.zeros(1, dtype=optim._ENTRY)
    entries["n"] = 5
    before = entries.copy()
    assert read([p], entries.ctypes.data, _lib.GRU_F32, 0) is False  # not on the device
    assert read(["p"], entries.ctypes.data, _lib.GRU_F32, 0) is False
    assert read([], entries.ctypes.data, _lib.GRU_F32, 0) is True
    assert (entries == before).all()
    with pytest.raises(TypeError):
        read((p,), entries.ctypes.data, _lib.GRU_F32, 0)

