"""CPU: the layer operators' checks of arguments (the tests' tensors are on the CPU, whose device number is -1), and the
plain 64-bit forms that the GPU tests compare with, against independent ones.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kernelintrinsics as KI
import layer_reference as ref

CPU = -1


def _refused(call, *args):
    with pytest.raises(KI.KIArgumentError):
        call(*args)


def test_rows_of_any_stride():
    t = torch.zeros(4, 10)
    assert KI._rows("f", "x", t, (4, 10), torch.float32, CPU) == 10
    assert KI._rows("f", "x", t[:, 2:7], (4, 5), torch.float32, CPU) == 10
    assert KI._rows("f", "x", t[1:2], (1, 10), torch.float32, CPU) == 10   # a single row has no stride of its own
    assert KI._rows("f", "x", t[:, :1], (4, 1), torch.float32, CPU) == 10
    for bad, shape, dtype in ((t, (4, 9), torch.float32), (t, (4, 10), torch.float16), (t.t(), (10, 4), torch.float32),
                              (t[:, ::2], (4, 5), torch.float32), (t[:1].expand(4, 10), (4, 10), torch.float32)):
        _refused(KI._rows, "f", "x", bad, shape, dtype, CPU)
    _refused(KI._rows, "f", "x", t, (4, 10), torch.float32, 0)             # another device


def test_flat():
    t = torch.zeros(6, 3)
    assert KI._flat("f", "x", None, (6, 3), torch.float32, CPU) is None
    assert KI._flat("f", "x", t, (6, 3), torch.float32, CPU) == t.data_ptr()
    for bad, shape in ((t[:, :2], (6, 2)), (t.t(), (3, 6)), (t, (3, 6))):
        _refused(KI._flat, "f", "x", bad, shape, torch.float32, CPU)
    _refused(KI._flat, "f", "x", t, (6, 3), torch.int32, CPU)


def test_states_in_slots():
    big = torch.zeros(5, 4, 3, 8)
    slots = torch.zeros(2, dtype=torch.int32)
    ptr, ld, n, at = KI._state("f", big[:, 1], 3, 8, torch.float32, CPU, slots, 2)
    assert (ptr, ld, n, at) == (big[:, 1].data_ptr(), 96, 5, slots.data_ptr())
    assert KI._state("f", big[0], 3, 8, torch.float32, CPU, None, 4)[1:] == (24, 4, None)
    assert KI._state("f", None, 3, 8, torch.float32, CPU, None, 4) == (None, 0, 0, None)
    args = (torch.float32, CPU)
    _refused(KI._state, "f", None, 3, 8, *args, slots, 2)
    _refused(KI._state, "f", big[0], 3, 8, *args, None, 5)                 # fewer slots than sequences
    _refused(KI._state, "f", big[0], 3, 8, *args, slots, 3)
    _refused(KI._state, "f", big[0], 3, 8, *args, slots.long(), 2)
    _refused(KI._state, "f", big[0], 8, 3, *args, None, 4)
    _refused(KI._state, "f", big[0].half(), 3, 8, *args, None, 4)
    _refused(KI._state, "f", big[0].transpose(1, 2), 8, 3, *args, None, 4)  # a slot that is not contiguous
    _refused(KI._state, "f", big[0, :1].expand(4, 3, 8), 3, 8, *args, None, 4)
    _refused(KI._state, "f", big, 3, 8, *args, None, 4)


def test_sequences():
    off = torch.tensor([0, 3, 9], dtype=torch.int32)
    flags = torch.ones(2, dtype=torch.bool)
    assert KI._sequences("f", None, None, None, CPU) == (1, None, None)
    assert KI._sequences("f", off, flags, off, CPU) == (2, off.data_ptr(), flags.data_ptr())
    _refused(KI._sequences, "f", off.long(), None, None, CPU)
    _refused(KI._sequences, "f", off[:0], None, None, CPU)
    _refused(KI._sequences, "f", off[None], None, None, CPU)
    _refused(KI._sequences, "f", off, flags, None, CPU)                    # flags without a state
    _refused(KI._sequences, "f", off, flags[:1], off, CPU)
    _refused(KI._sequences, "f", off, flags.float(), off, CPU)


def test_groups_of_b_and_c():
    t = torch.zeros(6, 40)
    assert KI._per_state("f", "B", t[:, 4:20], 6, 16, torch.float32, CPU) == (40, 1)
    assert KI._per_state("f", "B", t[:, 4:36].unflatten(1, (2, 16)), 6, 16, torch.float32, CPU) == (40, 2)
    for bad in (t[:, :32].unflatten(1, (16, 2)).transpose(1, 2), t[:, :30], t[:, :32].unflatten(1, (4, 8)), t[0],
                t[:1, :32].unflatten(1, (2, 16)).expand(6, 2, 16), t.half()[:, :16]):
        _refused(KI._per_state, "f", "B", bad, 6, 16, torch.float32, CPU)


def test_activation_and_types():
    assert KI._silu("f", None) == 0 and KI._silu("f", "silu") == 1
    _refused(KI._silu, "f", "relu")
    assert [KI._float_code("f", t) for t in (torch.float32, torch.float16, torch.bfloat16)] == [8, 10, 11]
    _refused(KI._float_code, "f", torch.float64)


def test_no_cpu_path():
    x = torch.zeros(4, 8)
    for call in (lambda: KI.quantize_rows(x), lambda: KI.int8_gemm(x.char(), x.char(), x[:, 0], x[:, 0]),
                 lambda: KI.causal_conv(x, x[:, :4]), lambda: KI.causal_conv_step(x, x[:, :4]),
                 lambda: KI.selective_scan(x, x, x, x, x), lambda: KI.selective_scan_step(x, x, x, x, x)):
        _refused(call)


def test_reference_conv_is_conv1d():
    g = torch.Generator().manual_seed(1)
    x, w, b = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((20, 6), (6, 4), (6,)))
    want = torch.nn.functional.silu(torch.nn.functional.conv1d(x.t()[None], w[:, None], b, padding=3, groups=6)[0, :, :20].t())
    y, err, last = ref.conv(x.numpy(), w.numpy(), b.numpy(), [(0, 20)], [np.zeros((3, 6))], True)
    assert np.allclose(y, want.numpy(), rtol=1e-12, atol=1e-12)
    assert np.array_equal(last[0], x[17:].numpy())
    # in two parts, the second from the first one's state
    y1, _, l1 = ref.conv(x[:2].numpy(), w.numpy(), b.numpy(), [(0, 2)], [np.zeros((3, 6))], True)
    y2, _, l2 = ref.conv(x[2:].numpy(), w.numpy(), b.numpy(), [(0, 18)], l1, True)
    assert np.allclose(np.concatenate([y1, y2]), y) and np.array_equal(l2[0], last[0])


def test_reference_scan_is_the_sum_over_earlier_tokens():
    """y_t = sum_n C_t sum_{s <= t} exp(A sum_{s < r <= t} s_r) s_s u_s B_s + D u, gated."""
    g = torch.Generator().manual_seed(2)
    T, D, N = 7, 3, 4
    u, d, z = (torch.randn(T, D, generator=g, dtype=torch.float64) for _ in range(3))
    B, C = (torch.randn(T, 1, N, generator=g, dtype=torch.float64) for _ in range(2))
    A, skip, bias = -torch.rand(D, N, generator=g, dtype=torch.float64), torch.randn(D, generator=g).double(), torch.randn(D, generator=g).double()
    s = torch.nn.functional.softplus(d + bias, threshold=1000)
    total = s.cumsum(0)
    want = torch.zeros(T, D, dtype=torch.float64)
    for t in range(T):
        for r in range(t + 1):
            want[t] += (C[t, 0] * torch.exp(A * (total[t] - total[r])[:, None]) * (s[r] * u[r])[:, None] * B[r, 0]).sum(1)
    want = (want + skip * u) * torch.nn.functional.silu(z)
    y, err, last, lerr = ref.scan(*(v.numpy() for v in (u, d, A, B, C, skip, z, bias)), True, [(0, T)], [np.zeros((D, N))])
    assert np.allclose(y, want.numpy(), rtol=1e-12, atol=1e-12)


def test_reference_quantize():
    x = np.array([[127.0, 0.5, 1.5, 2.5, -0.5, -63.49, 0.0, -127.0], [0] * 8, [np.nan] + [1.0] * 7, [np.inf, -np.inf] + [1.0] * 6],
                 np.float32)
    s, q = ref.quantize(x)
    one = np.float32(127) * (np.float32(1) / np.float32(127))
    assert s[0] == one and s[1] == 0 and np.isnan(s[2]) and np.isinf(s[3])
    assert q[0].tolist() == [127, 0, 2, 2, 0, -63, 0, -127] and not q[1:].any()


def test_reference_product():
    rng = np.random.default_rng(3)
    a, w = rng.integers(-128, 128, (3, 50), dtype=np.int8), rng.integers(-128, 128, (5, 50), dtype=np.int8)
    y, err = ref.product(a, w, np.ones(3), np.full(5, 0.5), np.arange(5.0))
    want = (torch.from_numpy(a).double() @ torch.from_numpy(w).double().t() * 0.5 + torch.arange(5.0)).numpy()
    assert np.array_equal(y, want) and (err >= 0).all()


def test_tensors_that_require_gradients_are_refused():
    """The operators give no gradients, so a tensor that requires one is refused where torch would record it."""
    t = torch.zeros(6, 32, requires_grad=True)
    state = torch.zeros(5, 4, 8, requires_grad=True)
    grouped = t.unflatten(1, (2, 16))
    calls = ((KI._rows, "f", "x", t, (6, 32), torch.float32, CPU), (KI._flat, "f", "x", t, (6, 32), torch.float32, CPU),
             (KI._state, "f", state, 4, 8, torch.float32, CPU, None, 5),
             (KI._per_state, "f", "B", grouped, 6, 16, torch.float32, CPU),
             (KI._per_state, "f", "B", t, 6, 32, torch.float32, CPU))
    for call, *args in calls:
        with pytest.raises(KI.KIArgumentError, match="gradient"):
            call(*args)
        with torch.no_grad():
            call(*args)
        call(*(a.detach() if isinstance(a, torch.Tensor) else a for a in args))


def test_the_gravest_latched_bit_is_reported(tmp_path):
    """A status word with a bad index and an inconsistent state says inconsistent state; a wait that ran out comes first."""
    import subprocess

    from conftest import PKG

    src = tmp_path / "latched.cpp"
    src.write_text('#include <cstdio>\n#include "ki/common.cuh"\n'
                   'int main() { for (unsigned b = 1; b < 8; ++b) std::printf("%d ", ki::latched(b).status); }\n')
    exe = tmp_path / "latched"
    subprocess.run(["g++", "-std=c++17", f"-I{PKG / 'csrc'}", "-I/usr/local/cuda/include", str(src), "-o", str(exe)], check=True)
    # KI_DEV_TIMEOUT 1 -> KI_ERR_TIMEOUT 3, KI_DEV_BAD_STATE 2 -> KI_ERR_CUDA 2, KI_DEV_BAD_INDEX 4 -> KI_ERR_ARG 1
    got = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()
    assert got == ["3", "2", "3", "1", "3", "2", "3"]
