"""What of the selective scan, the causal convolution and the layer norm needs no GPU: sizes, refusals of the C entry points
and of the Python ones, the layers' parameters."""
import pytest
import torch

from rnn_kernel_b200 import (LayerNorm, RecurrentStack, SelectiveScan, _lib, build, causal_conv, causal_conv_step, layer_norm,
                             selective_scan, selective_step)

BAD = (_lib.GRU_ERR_INVALID, _lib.GRU_ERR_UNSUPPORTED)


def scan(dtype=0, B=2, T=100, D=64, N=16, G=2, softplus=1, pointers=(0,) * 9):
    return _lib.SCAN_ARGS.pack(dtype, B, T, D, N, G, softplus, *pointers, *[0] * 12)


def conv(dtype=0, wtype=0, B=2, T=10, D=64, W=4, act=1, pointers=(0,) * 4):
    return _lib.CONV_ARGS.pack(dtype, wtype, B, T, D, W, act, *pointers, 0, 0)


def norm(dtype=0, rtype=0, wtype=0, width=64, eps=1e-5, rows=10):
    return _lib.NORM_ARGS.pack(dtype, rtype, wtype, width, eps, rows, width, width)


def test_struct_sizes_match_the_header():
    assert (_lib.SCAN_ARGS.size, _lib.CONV_ARGS.size, _lib.NORM_ARGS.size) == (200, 80, 48)


def test_sizes_without_gpu():
    lib = _lib.load()
    one = lib.gru_scan_stash_bytes(scan(T=64))
    assert one > 0 and one % 256 == 0 and one < lib.gru_scan_stash_bytes(scan(T=65)) < 2 * one
    # a gate keeps what it multiplies
    assert lib.gru_scan_stash_bytes(scan(T=64, pointers=(0,) * 4 + (64,) + (0,) * 4)) == one + 4 * 2 * 64 * 64
    assert lib.gru_scan_workspace_bytes(scan(), 1) > 0
    # long sequences of few channels are cut into segments, which a forward remembers too
    assert lib.gru_scan_workspace_bytes(scan(T=5), 0) == 0 < lib.gru_scan_workspace_bytes(scan(T=5000), 0)
    assert lib.gru_scan_stash_bytes(scan(B=64, T=1 << 16, D=4096)) >= 1 << 34
    assert lib.gru_conv_workspace_bytes(conv()) > 0 and lib.gru_layer_norm_workspace_bytes(norm()) > 0


@pytest.mark.parametrize("bad", [dict(dtype=2), dict(B=-1), dict(T=-1), dict(D=0), dict(G=0), dict(G=3), dict(N=0), dict(N=65),
                                 dict(softplus=2), dict(B=1 << 30, D=1 << 20)])
def test_scan_entries_refuse(bad):
    lib = _lib.load()
    a = scan(**bad)
    assert lib.gru_scan_stash_bytes(a) == 0 == lib.gru_scan_workspace_bytes(a, 1) and _lib.last_error()
    assert lib.gru_scan_forward(a, 64, 64, 0, 0, 0, 0, 0) in BAD
    assert lib.gru_scan_backward(a, *[64] * 3, 1 << 40, *[64] * 10, 1 << 40, 0) in BAD
    assert lib.gru_scan_step(a, 64, 64, 0) in BAD


def test_scan_entries_refuse_null_misaligned_and_small():
    lib = _lib.load()
    p = (64,) * 8 + (128,)  # addresses that are never read: the calls fail before
    assert lib.gru_scan_forward(scan(), 64, 64, 0, 0, 0, 0, 0) in BAD  # null tensors
    assert lib.gru_scan_forward(scan(pointers=p), 64, 128, 0, 0, 0, 0, 0) in BAD and "initial state" in _lib.last_error()
    assert lib.gru_scan_forward(scan(pointers=p), 0, 64, 0, 0, 0, 0, 0) in BAD
    assert lib.gru_scan_forward(scan(pointers=p), 64, 0, 0, 0, 0, 0, 0) in BAD
    assert lib.gru_scan_forward(scan(pointers=p), 64, 64, 64, 16, 0, 0, 0) in BAD  # a small stash
    assert lib.gru_scan_forward(scan(pointers=p), 64, 64, 72, 1 << 40, 0, 0, 0) in BAD
    assert lib.gru_scan_forward(scan(pointers=(66,) + p[1:]), 64, 64, 0, 0, 0, 0, 0) in BAD
    assert lib.gru_scan_forward(scan(T=5000, pointers=p), 64, 64, 0, 0, 0, 0, 0) in BAD  # no workspace
    assert lib.gru_scan_forward(scan(T=5000, pointers=p), 64, 64, 0, 0, 64, 16, 0) in BAD
    grads = [64] * 9
    assert lib.gru_scan_backward(scan(pointers=p), 64, 128, 64, 1 << 40, *grads, 64, 16, 0) in BAD
    assert lib.gru_scan_backward(scan(pointers=p), 64, 128, 64, 16, *grads, 64, 1 << 40, 0) in BAD
    assert lib.gru_scan_backward(scan(pointers=p), 64, 64, 64, 1 << 40, *grads, 64, 1 << 40, 0) in BAD and "dfinal" in _lib.last_error()
    for i in (0, 1, 2, 3, 4, 6):  # dx, ddt, da, db, dc, dz
        assert lib.gru_scan_backward(scan(pointers=p), 64, 128, 64, 1 << 40, *grads[:i], 0, *grads[i + 1:], 64, 1 << 40, 0) in BAD
    assert lib.gru_scan_step(scan(pointers=p), 64, 64, 0) in BAD and "T must be 1" in _lib.last_error()
    assert lib.gru_scan_step(scan(T=1, pointers=p), 0, 64, 0) in BAD
    assert lib.gru_scan_step(scan(T=1, B=0), 0, 0, 0) == _lib.GRU_OK == lib.gru_scan_forward(scan(B=0), 0, 0, 0, 0, 0, 0, 0)


@pytest.mark.parametrize("bad", [dict(dtype=2), dict(wtype=1), dict(wtype=3), dict(B=-1), dict(T=-1), dict(D=0), dict(W=1), dict(W=9),
                                 dict(act=2), dict(B=1 << 28, T=1 << 20)])
def test_conv_entries_refuse(bad):
    lib = _lib.load()
    a = conv(**bad)
    assert lib.gru_conv_workspace_bytes(a) == 0 and _lib.last_error()
    assert lib.gru_conv_forward(a, 64, 64, 0) in BAD
    assert lib.gru_conv_backward(a, *[64] * 7, 1 << 40, 0) in BAD
    assert lib.gru_conv_step(a, 64, 64, 0) in BAD


def test_conv_entries_refuse_null_misaligned_and_small():
    lib = _lib.load()
    p = (64,) * 4
    assert lib.gru_conv_forward(conv(), 64, 64, 0) in BAD
    assert lib.gru_conv_forward(conv(pointers=p), 64, 64, 0) in BAD  # the initial state's own memory
    assert lib.gru_conv_forward(conv(pointers=p), 66, 128, 0) in BAD
    assert lib.gru_conv_backward(conv(pointers=p), 64, 64, 64, 64, 64, 64, 64, 16, 0) in BAD
    assert lib.gru_conv_backward(conv(pointers=p), 64, 64, 0, 64, 64, 64, 64, 1 << 40, 0) in BAD
    assert lib.gru_conv_backward(conv(pointers=p), 64, 64, 64, 0, 64, 64, 64, 1 << 40, 0) in BAD
    assert lib.gru_conv_step(conv(pointers=p), 64, 64, 0) in BAD and "T must be 1" in _lib.last_error()
    assert lib.gru_conv_step(conv(T=1, B=0), 0, 0, 0) == _lib.GRU_OK


@pytest.mark.parametrize("bad", [dict(dtype=2), dict(rtype=1), dict(wtype=1), dict(rows=-1), dict(width=0), dict(width=16385),
                                 dict(eps=-1.0), dict(eps=float("nan"))])
def test_norm_entries_refuse(bad):
    lib = _lib.load()
    a = norm(**bad)
    assert lib.gru_layer_norm_workspace_bytes(a) == 0 and _lib.last_error()
    assert lib.gru_layer_norm_forward(a, 64, 0, 64, 64, 64, 0, 0, 0) in BAD
    assert lib.gru_layer_norm_backward(a, *[64] * 10, 1 << 40, 0) in BAD


def test_norm_entries_refuse_null_misaligned_and_small():
    lib = _lib.load()
    ok = [64, 0, 64, 64, 64, 0, 0]
    for i, v in ((0, 0), (2, 0), (4, 0), (0, 66), (1, 64), (5, 64), (6, 66)):  # null; a residual or a sum alone
        assert lib.gru_layer_norm_forward(norm(), *ok[:i], v, *ok[i + 1:], 0) in BAD
    ok = [64] * 10
    for i, v in ((0, 0), (1, 0), (2, 0), (3, 0), (7, 0), (9, 0), (9, 72), (0, 66)):
        assert lib.gru_layer_norm_backward(norm(), *ok[:i], v, *ok[i + 1:], 1 << 40, 0) in BAD
    assert lib.gru_layer_norm_backward(norm(), *ok, 16, 0) in BAD
    assert lib.gru_layer_norm_forward(norm(rows=0), *[0] * 7, 0) == _lib.GRU_OK


def test_python_entries_refuse_shapes_and_cpu_tensors():
    x, A, B = torch.zeros(1, 4, 8), torch.zeros(8, 3), torch.zeros(1, 4, 2, 3)
    with pytest.raises(RuntimeError, match="CUDA"):
        selective_scan(x, x, A, B, B)
    with pytest.raises(RuntimeError, match="CUDA"):
        selective_step(x[:, 0], x[:, 0], A, B[:, 0], B[:, 0], torch.zeros(1, 8, 3))
    for bad in (dict(x=x[0]), dict(dt=x[:, :3]), dict(A=A.t()), dict(B=B[:, :3]), dict(C=B[..., :2]), dict(z=x[:, :1]),
                dict(skip=x[0, 0, :7]), dict(dt_bias=x[0]), dict(initial_state=torch.zeros(1, 3, 8)),
                dict(B=torch.zeros(1, 4, 3, 3), C=torch.zeros(1, 4, 3, 3))):
        with pytest.raises(ValueError):
            selective_scan(**{**dict(x=x, dt=x, A=A, B=B, C=B), **bad})
    with pytest.raises(ValueError, match="states"):
        selective_scan(x, x, torch.zeros(8, 65), torch.zeros(1, 4, 1, 65), torch.zeros(1, 4, 1, 65))
    w = torch.zeros(8, 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        causal_conv(x, w)
    with pytest.raises(RuntimeError, match="CUDA"):
        causal_conv_step(x[:, 0], w, torch.zeros(1, 3, 8))
    for bad in (dict(x=x[0]), dict(weight=w[:7]), dict(weight=w[:, :1]), dict(weight=torch.zeros(8, 9)), dict(bias=w[:7, 0]),
                dict(initial_state=torch.zeros(1, 4, 8)), dict(activation="gelu")):
        with pytest.raises(ValueError):
            causal_conv(**{**dict(x=x, weight=w), **bad})
    with pytest.raises(RuntimeError, match="CUDA"):
        layer_norm(x, torch.zeros(8))
    for bad in (dict(weight=torch.zeros(7)), dict(bias=torch.zeros(1, 8)), dict(residual=x[0]), dict(eps=-1e-5), dict(x=torch.tensor(1.0)),
                dict(x=torch.zeros(2, 0), weight=torch.zeros(0)), dict(x=torch.zeros(1, 16385), weight=torch.zeros(16385))):
        with pytest.raises(ValueError):
            layer_norm(**{**dict(x=x, weight=torch.zeros(8)), **bad})


def test_the_host_module_without_cuda_headers_is_adamws_alone(tmp_path):
    files, flags = build.host_parts(tmp_path)  # no libc10_cuda there
    assert [f.name for f in files] == ["host_tensors.cpp"] and flags == ["-DGRU_TENSORS_ONLY"]


def test_layers():
    m = SelectiveScan(16, 24, state_size=5, conv_size=3, num_groups=2, dt_rank=2, output_size=7)
    assert {k: tuple(v.shape) for k, v in m.state_dict().items()} == {
        "conv_weight": (24, 3), "conv_bias": (24,), "dt_bias": (24,), "log_rate": (24, 5), "skip": (24,), "in_proj.weight": (48, 16),
        "x_proj.weight": (22, 24), "dt_proj.weight": (24, 2), "out_proj.weight": (7, 24)}
    conv, state = m.bfloat16().init_state(3)
    assert conv.shape == (3, 2, 24) and conv.dtype == torch.bfloat16 and state.shape == (3, 24, 5) and state.dtype == torch.float32
    for bad in (dict(inner_size=25, num_groups=2), dict(state_size=65), dict(conv_size=1), dict(conv_size=9), dict(dt_rank=0)):
        with pytest.raises(ValueError):
            SelectiveScan(16, **bad)
    with pytest.raises(ValueError):
        LayerNorm(0)
    with pytest.raises(ValueError):
        LayerNorm(16385)
    stack = RecurrentStack([SelectiveScan(16), SelectiveScan(16)], 16)
    assert len(stack.norms) == 3 and stack.norms[0].weight.shape == (16,)
    with pytest.raises(RuntimeError, match="CUDA"):
        stack(torch.zeros(1, 2, 16))
