"""GPU: the operators of a state-space layer served in 8 bits (quantize_rows, int8_gemm, causal_conv,
selective_scan and the single-token forms) against plain 64-bit forms, with the bounds of
layer_reference.py; quantize_rows bit for bit.
"""
from __future__ import annotations

import numpy as np
import pytest

import layer_reference as ref

pytestmark = pytest.mark.gpu

TYPES = ["float32", "float16", "bfloat16"]


def _rng(seed):
    import torch

    return torch.Generator().manual_seed(seed)


def _normal(g, *shape, scale=1.0, dtype="float32", dev="cuda"):
    import torch

    return (torch.randn(*shape, generator=g) * scale).to(getattr(torch, dtype)).to(dev)


def _within(got, want, err, dtype):
    import torch

    got = ref.f64(got)
    bound = ref.stored(want, err, dtype)
    off = np.abs(got - want)
    assert np.isfinite(got).all()
    assert (off <= bound).all(), (float((off / bound).max()), np.unravel_index((off / bound).argmax(), off.shape))


# ---------------------------------------------------------------------------------------------
# rows to int8
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 64), (2, 257), (7, 1000), (4, 4096), (3, 8200), (2, 16384),
                                       (1, 16392), (2, 33000), (1030, 24)])
def test_quantize_rows(KI, dev, dtype, rows, cols):
    import torch

    g = _rng(rows * 31 + cols)
    x = _normal(g, rows, cols) * torch.exp(2 * _normal(g, rows, 1))
    x = x.to(getattr(torch, dtype))
    q, s = KI.quantize_rows(x)
    ws, wq = ref.quantize(x.float().cpu().numpy())
    assert np.array_equal(s.cpu().numpy(), ws) and np.array_equal(q.cpu().numpy(), wq)
    # views whose rows start anywhere, into an output whose rows start anywhere
    for lead in (1, 3, 8):
        big = torch.zeros(rows, cols + 21, dtype=x.dtype, device=dev)
        big[:, lead:lead + cols] = x
        out = torch.full((rows, cols + 5), 99, dtype=torch.int8, device=dev)
        q2, s2 = KI.quantize_rows(big[:, lead:lead + cols], out=out[:, 2:2 + cols])
        assert torch.equal(q2, q) and torch.equal(s2, s)
        assert (out[:, :2] == 99).all() and (out[:, 2 + cols:] == 99).all()
    KI.context(0).check()


@pytest.mark.parametrize("cols", [16, 37, 5000, 40000])
def test_quantize_rows_special_values(KI, dev, cols):
    import torch

    g = _rng(cols)
    x = _normal(g, 12, cols, dev="cpu")
    x[0] = 0
    x[1] = -0.0
    x[2, 3] = float("nan")
    x[3, 5] = float("inf")
    x[4, 1], x[4, 2] = float("-inf"), float("nan")
    x[5] *= 1e-38                       # subnormal values and scale
    x[6] = 0
    x[6, 7] = 2.0 ** -149               # the scale underflows to zero
    x[7] = torch.arange(cols) % 255 - 127.0
    x[7, 0], x[8] = 127.0, x[7] / 2     # row 8: half-way points at scale 1, after its own maximum
    x[8] = (torch.arange(cols) % 254) - 126.5
    x[8, 0] = 127.0
    x[9] = torch.finfo(torch.float32).max * torch.sign(x[9])
    x[10] = 190 * 2.0 ** -149           # the scale rounds to one step: q is cut at 127
    q, s = KI.quantize_rows(x.to(dev))
    ws, wq = ref.quantize(x.numpy())
    assert np.array_equal(s.cpu().numpy(), ws, equal_nan=True)
    assert np.array_equal(q.cpu().numpy(), wq)
    assert (q[0] == 0).all() and s[0] == 0 and torch.isnan(s[2]) and torch.isinf(s[3]) and torch.isnan(s[4])


def test_quantize_rows_near_half_way_points(KI, dev):
    """Values one step either side of every half-way point round as the division does."""
    import torch

    rows = []
    for k in range(60):
        scale = np.float32(0.37 + 0.0131 * k)
        top = np.float32(scale * 127)
        mid = ((np.arange(-126, 126) + 0.5) * np.float64(top) / 127).astype(np.float32)
        near = np.concatenate([mid, np.nextafter(mid, np.float32(9e9)), np.nextafter(mid, np.float32(-9e9)), [top]])
        rows.append(near.astype(np.float32))
    x = np.stack(rows)
    q, s = KI.quantize_rows(torch.from_numpy(x).to(dev))
    ws, wq = ref.quantize(x)
    assert np.array_equal(s.cpu().numpy(), ws) and np.array_equal(q.cpu().numpy(), wq)


def test_quantize_rows_empty(KI, dev):
    import torch

    q, s = KI.quantize_rows(torch.empty(0, 5, device=dev))
    assert q.shape == (0, 5) and s.shape == (0,)
    q, s = KI.quantize_rows(torch.empty(3, 0, device=dev))
    assert q.shape == (3, 0) and (s == 0).all()


# ---------------------------------------------------------------------------------------------
# int8 product
# ---------------------------------------------------------------------------------------------
def _operands(seed, M, N, K, dev):
    import torch

    g = _rng(seed)
    a = torch.randint(-128, 128, (M, K), generator=g, dtype=torch.int8).to(dev)
    w = torch.randint(-128, 128, (N, K), generator=g, dtype=torch.int8).to(dev)
    sa = (torch.rand(M, generator=g) * 0.05 + 0.001).to(dev)
    sw = (torch.rand(N, generator=g) * 0.01 + 0.0001).to(dev)
    return a, w, sa, sw, torch.randn(N, generator=g).to(dev)


def _check_product(out, a, w, sa, sw, bias, dtype):
    want, err = ref.product(a.cpu().numpy(), w.cpu().numpy(), ref.f64(sa), ref.f64(sw), None if bias is None else ref.f64(bias))
    _within(out, want, err, dtype)


@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 128, 128), (1, 300, 4096), (2, 129, 48), (15, 64, 1000), (16, 256, 256),
                                   (17, 130, 130), (33, 200, 2064), (48, 1024, 512), (64, 128, 129), (65, 127, 127),
                                   (128, 128, 2048), (129, 257, 255), (200, 700, 640), (256, 512, 384), (300, 2049, 272),
                                   (513, 1040, 144), (1024, 1024, 256), (1111, 515, 257), (2050, 2304, 128), (2049, 2060, 400),
                                   (4100, 1030, 1040)])
def test_int8_gemm(KI, dev, M, N, K):
    import torch

    a, w, sa, sw, bias = _operands(M + 7 * N + 13 * K, M, N, K, dev)
    for dtype, b in ((torch.float32, None), (torch.bfloat16, bias), (torch.float16, bias)):
        sc = sw * (K ** -0.5)  # Float16 outputs stay in range
        out = KI.int8_gemm(a, w, sa, sc, bias=b, dtype=dtype)
        KI.context(0).check()
        _check_product(out, a, w, sa, sc, b, dtype)


@pytest.mark.parametrize("lead_a,lead_w,pad", [(0, 0, 16), (16, 32, 16), (1, 0, 16), (0, 3, 16), (5, 7, 3), (8, 4, 9)])
@pytest.mark.parametrize("M,N,K", [(3, 140, 320), (70, 260, 200), (300, 520, 136)])
def test_int8_gemm_strided(KI, dev, lead_a, lead_w, pad, M, N, K):
    """Operands that are views with any start and stride, and an output that is a view; what surrounds it stays."""
    import torch

    a, w, sa, sw, bias = _operands(M * 3 + N + K, M, N, K, dev)
    av = torch.zeros(M, K + lead_a + pad, dtype=torch.int8, device=dev)[:, lead_a:lead_a + K]
    wv = torch.full((N, K + lead_w + pad), 77, dtype=torch.int8, device=dev)[:, lead_w:lead_w + K]
    av.copy_(a)
    wv.copy_(w)
    for dtype in (torch.float32, torch.bfloat16):
        big = torch.full((M + 2, N + 9), 5.0, dtype=dtype, device=dev)
        out = KI.int8_gemm(av, wv, sa, sw, bias=bias, out=big[1:-1, 3:3 + N])
        KI.context(0).check()
        _check_product(out, a, w, sa, sw, bias, dtype)
        rest = big.clone()
        rest[1:-1, 3:3 + N] = 5.0
        assert (rest == 5.0).all()


@pytest.mark.parametrize("M,N,K", [(1111, 4099, 33), (640, 4099, 65), (513, 4099, 129), (740, 4099, 17), (768, 4100, 300),
                                   (2100, 2049, 129), (769, 4099, 0)])
def test_int8_gemm_tiles_of_other_widths(KI, dev, M, N, K):
    """Rows that TMA cannot take, in more tiles of 128 x 128 than there are SMs; outputs at odd strides."""
    import torch

    a, w, sa, sw, bias = _operands(M + N + K, M, N, K, dev)
    for dtype in (torch.float32, torch.bfloat16):
        big = torch.full((M + 2, N + 5), 5.0, dtype=dtype, device=dev)
        sc = sw * (max(K, 1) ** -0.5)
        out = KI.int8_gemm(a, w, sa, sc, bias=bias, out=big[1:-1, 2:2 + N])
        KI.context(0).check()
        _check_product(out, a, w, sa, sc, bias, dtype)
        big[1:-1, 2:2 + N] = 5.0
        assert (big == 5.0).all()


def test_int8_gemm_extremes(KI, dev):
    """The largest sums that are allowed, and no inner dimension at all."""
    import torch

    K = 131071
    a = torch.full((2, K), -128, dtype=torch.int8, device=dev)
    w = torch.full((3, K), -128, dtype=torch.int8, device=dev)
    w[1] = 127
    one = torch.ones(3, device=dev)
    out = KI.int8_gemm(a, w, one[:2].clone(), one, dtype=torch.float32)
    assert out[0].tolist() == [float(np.float32(128 * 128 * K)), float(np.float32(-128 * 127 * K)),
                               float(np.float32(128 * 128 * K))]
    with pytest.raises(KI.KIArgumentError):
        KI.int8_gemm(torch.zeros(1, K + 1, dtype=torch.int8, device=dev), torch.zeros(1, K + 1, dtype=torch.int8, device=dev),
                     one[:1].clone(), one[:1].clone())
    # (its rows have a stride of one, and may start anywhere)
    e = torch.empty(5, 3, dtype=torch.int8, device=dev)[:, 1:1]
    assert torch.equal(KI.int8_gemm(e, torch.empty(7, 2, dtype=torch.int8, device=dev)[:, 2:], torch.ones(5, device=dev),
                                    torch.ones(7, device=dev), dtype=torch.float32), torch.zeros(5, 7, device=dev))
    e = torch.empty(5, 0, dtype=torch.int8, device=dev)
    bias = torch.arange(7.0, device=dev)
    sc = torch.ones(7, device=dev)
    out = KI.int8_gemm(e, torch.empty(7, 0, dtype=torch.int8, device=dev), sc[:5].clone(), sc, bias=bias, dtype=torch.float32)
    assert torch.equal(out, bias.expand(5, 7))
    assert KI.int8_gemm(torch.empty(0, 16, dtype=torch.int8, device=dev), torch.empty(7, 16, dtype=torch.int8, device=dev),
                        sc[:0].clone(), sc).shape == (0, 7)
    KI.context(0).check()


def test_int8_gemm_shows_a_broken_token(KI, dev):
    """A token whose scale is NaN or infinite gives NaN in its own row only."""
    import torch

    x = torch.randn(4, 64, generator=_rng(3)).to(dev)
    x[1, 5] = float("nan")
    x[2, 7] = float("inf")
    q, s = KI.quantize_rows(x)
    w = torch.randint(-127, 128, (130, 64), generator=_rng(4), dtype=torch.int8).to(dev)
    w[:, 7] = 0
    out = KI.int8_gemm(q, w, s, torch.ones(130, device=dev), dtype=torch.float32)
    assert torch.isfinite(out[0]).all() and torch.isfinite(out[3]).all()
    assert torch.isnan(out[1]).all() and torch.isnan(out[2]).all()


# ---------------------------------------------------------------------------------------------
# causal convolution
# ---------------------------------------------------------------------------------------------
#: offsets of packed sequences: one token, several, empty ones at the start, between and at the end
LAYOUTS = {"one": [0, 1], "two tokens": [0, 2], "long": [0, 333], "several": [0, 1, 3, 4, 40, 41, 170],
           "empty": [0, 0, 0, 5, 5, 37, 37, 37, 64, 64], "runs": [0, 31, 33, 62, 64, 65, 97, 128], "none": [0, 0],
           "inside": [4, 9, 50, 51]}


def _conv_case(seed, offsets, channels, width, dtype, dev, more=7):
    import torch

    g = _rng(seed)
    tokens, n = offsets[-1] + more, len(offsets) - 1
    x = _normal(g, tokens, channels, dtype=dtype)
    w = _normal(g, channels, width, scale=0.5, dtype=dtype)
    bias = _normal(g, channels, scale=0.3, dtype=dtype)
    state = _normal(g, n + 4, width - 1, channels, dtype=dtype)
    slots = torch.randperm(n + 4, generator=g)[:n].to(torch.int32)
    initial = torch.rand(n, generator=g) < 0.6
    return x, w, bias, state, slots, initial, torch.tensor(offsets, dtype=torch.int32)


def _conv_check(KI, dev, x, w, bias, state, slots, initial, offsets, act, dtype):
    import torch

    n = offsets.numel() - 1
    spans = [(int(offsets[i]), int(offsets[i + 1])) for i in range(n)]
    before = state.clone()
    first = [ref.f64(state[int(slots[i])]) * (1.0 if initial is None or initial[i] else 0.0) if slots[i] >= 0 else None
             for i in range(n)]
    live = [i for i in range(n) if slots[i] >= 0]
    want, err, last = ref.conv(ref.f64(x), ref.f64(w), None if bias is None else ref.f64(bias), [spans[i] for i in live],
                               [first[i] for i in live], act == "silu")
    out = torch.full((x.shape[0], x.shape[1]), 3.0, dtype=x.dtype, device=dev)
    got = KI.causal_conv(x, w, bias, state=state, offsets=offsets.to(dev), slots=slots.to(dev),
                         initial=None if initial is None else initial.to(dev), activation=act, out=out)
    KI.context(0).check()
    covered = np.zeros(x.shape[0], bool)
    for i in live:
        covered[spans[i][0]:spans[i][1]] = True
    _within(got[torch.from_numpy(covered).to(dev)], want[covered], err[covered], x.dtype)
    assert (got[torch.from_numpy(~covered).to(dev)] == 3.0).all()  # rows of no sequence
    for i, l in zip(live, last):
        assert np.array_equal(ref.f64(state[int(slots[i])]), l)
    rest = [s for s in range(state.shape[0]) if s not in [int(slots[i]) for i in live]]
    assert torch.equal(state[rest], before[rest])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("channels,width", [(8, 4), (136, 2), (75, 4), (1100, 3), (64, 8)])
def test_causal_conv(KI, dev, dtype, layout, channels, width):
    case = _conv_case(channels + width, LAYOUTS[layout], channels, width, dtype, dev)
    x, w, bias, state, slots, initial, offsets = case
    _conv_check(KI, dev, x, w, bias, state, slots, initial, offsets, "silu", dtype)
    _conv_check(KI, dev, x, w, None, state, slots, None, offsets, None, dtype)


@pytest.mark.parametrize("width", [2, 5, 6, 7, 8])
def test_causal_conv_state_over_run_borders(KI, dev, width):
    """Sequences that begin at every place around the borders of the runs of tokens."""
    for first in range(0, 40):
        offsets = [0, first, first + 1, first + 3, first + 3 + width, 75, 90]
        case = _conv_case(first, offsets, 16, width, "float32", dev, more=0)
        x, w, bias, state, slots, initial, off = case
        _conv_check(KI, dev, x, w, bias, state, slots, initial, off, None, "float32")


def test_causal_conv_padding_and_strides(KI, dev):
    """Padding sequences are skipped; x, y and the state are views with strides of their own."""
    import torch

    x, w, bias, state, slots, initial, offsets = _conv_case(5, LAYOUTS["several"], 96, 4, "bfloat16", dev)
    slots[1], slots[4] = -1, -7
    big = torch.zeros(x.shape[0], 200, dtype=x.dtype, device=dev)
    big[:, 101:197] = x
    cache = torch.zeros(state.shape[0], 2, 3, 96, dtype=x.dtype, device=dev)
    cache[:, 1] = state
    _conv_check(KI, dev, big[:, 101:197], w, bias, cache[:, 1], slots, initial, offsets, "silu", "bfloat16")
    assert (cache[:, 0] == 0).all()


def test_causal_conv_without_state(KI, dev):
    import torch

    x, w, bias, *_ = _conv_case(9, [0, 50], 40, 4, "float32", dev, more=0)
    want, err, _ = ref.conv(ref.f64(x), ref.f64(w), ref.f64(bias), [(0, 50)], [np.zeros((3, 40))], False)
    _within(KI.causal_conv(x, w, bias), want, err, torch.float32)
    off = torch.tensor([0, 20, 50], dtype=torch.int32, device=dev)
    want, err, _ = ref.conv(ref.f64(x), ref.f64(w), ref.f64(bias), [(0, 20), (20, 50)], [np.zeros((3, 40))] * 2, True)
    _within(KI.causal_conv(x, w, bias, offsets=off, activation="silu"), want, err, torch.float32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,channels,width", [(1, 8, 4), (3, 75, 2), (64, 1024, 4), (5, 130, 8)])
def test_causal_conv_steps_continue_a_prompt(KI, dev, dtype, rows, channels, width):
    """Prompt, then single tokens: the same bits as one long prompt, and slots of other requests stay."""
    import torch

    g = _rng(rows + channels)
    T = 9
    x = _normal(g, rows, T, channels, dtype=dtype)
    w = _normal(g, channels, width, scale=0.5, dtype=dtype)
    bias = _normal(g, channels, dtype=dtype)
    slots = torch.randperm(rows + 3, generator=g)[:rows].to(torch.int32).to(dev)
    none = torch.zeros(rows, dtype=torch.bool, device=dev)

    def prompt(n, state):
        off = torch.arange(0, rows * n + 1, n, dtype=torch.int32, device=dev)
        return KI.causal_conv(x[:, :n].reshape(rows * n, channels), w, bias, state=state, offsets=off, slots=slots,
                              initial=none, activation="silu").view(rows, n, channels)

    whole = torch.randn(rows + 3, width - 1, channels, generator=g).to(x.dtype).to(dev)
    parts = whole.clone()
    want = prompt(T, whole)
    got = [prompt(4, parts)]
    for t in range(4, T):
        got.append(KI.causal_conv_step(x[:, t], w, bias, state=parts, slots=slots, activation="silu")[:, None])
    assert torch.equal(torch.cat(got, 1), want) and torch.equal(parts, whole)
    # a padding row is skipped
    keep = parts.clone()
    out = torch.full((rows, channels), 2.0, dtype=x.dtype, device=dev)
    KI.causal_conv_step(x[:, 0], w, bias, state=parts, slots=torch.full_like(slots, -1), out=out)
    assert torch.equal(parts, keep) and (out == 2.0).all()


# ---------------------------------------------------------------------------------------------
# selective scan
# ---------------------------------------------------------------------------------------------
def _scan_case(seed, tokens, n, channels, states, groups, dtype, dev, soft=True, gate=True):
    import torch

    g = _rng(seed)
    c = {"u": _normal(g, tokens, channels, dtype=dtype), "B": _normal(g, tokens, groups, states, dtype=dtype),
         "C": _normal(g, tokens, groups, states, dtype=dtype)}
    if soft:
        c["delta"] = _normal(g, tokens, channels, dtype=dtype)
        c["delta_bias"] = _normal(g, channels, scale=1.0) - 3
    else:
        c["delta"] = (torch.rand(tokens, channels, generator=g) * 0.2).to(getattr(torch, dtype)).to(dev)
        c["delta_bias"] = None
    c["A"] = -torch.exp(_normal(g, channels, states))
    c["D"] = _normal(g, channels)
    c["z"] = _normal(g, tokens, channels, scale=2.0, dtype=dtype) if gate else None
    c["softplus"] = soft
    state = _normal(g, n + 4, channels, states)
    slots = torch.randperm(n + 4, generator=g)[:n].to(torch.int32)
    return c, state, slots, torch.rand(n, generator=g) < 0.6


def _scan_check(KI, dev, c, state, slots, initial, offsets):
    import torch

    n = len(offsets) - 1
    spans = [(offsets[i], offsets[i + 1]) for i in range(n)]
    before = state.clone()
    live = [i for i in range(n) if slots[i] >= 0]
    first = [ref.f64(state[int(slots[i])]) * (1.0 if initial is None or initial[i] else 0.0) for i in live]
    opt = lambda k: None if c[k] is None else ref.f64(c[k])  # noqa: E731
    want, err, last, lasterr = ref.scan(ref.f64(c["u"]), ref.f64(c["delta"]), ref.f64(c["A"]), ref.f64(c["B"]),
                                        ref.f64(c["C"]), opt("D"), opt("z"), opt("delta_bias"), c["softplus"],
                                        [spans[i] for i in live], first)
    out = torch.full(c["u"].shape, 3.0, dtype=c["u"].dtype, device=dev)
    got = KI.selective_scan(**c, state=state, offsets=torch.tensor(offsets, dtype=torch.int32, device=dev),
                            slots=slots.to(dev), initial=None if initial is None else initial.to(dev), out=out)
    KI.context(0).check()
    covered = np.zeros(out.shape[0], bool)
    for i in live:
        covered[spans[i][0]:spans[i][1]] = True
    _within(got[torch.from_numpy(covered).to(dev)], want[covered], err[covered], out.dtype)
    assert (got[torch.from_numpy(~covered).to(dev)] == 3.0).all()
    for i, l, e in zip(live, last, lasterr):
        _within(state[int(slots[i])], l, e, torch.float32)
    rest = [s for s in range(state.shape[0]) if s not in [int(slots[i]) for i in live]]
    assert torch.equal(state[rest], before[rest])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("channels,states,groups", [(16, 16, 1), (70, 16, 2), (36, 13, 1), (5, 1, 1)])
def test_selective_scan(KI, dev, dtype, layout, channels, states, groups):
    offsets = LAYOUTS[layout]
    c, state, slots, initial = _scan_case(channels + states, offsets[-1] + 3, len(offsets) - 1, channels, states, groups,
                                          dtype, dev)
    _scan_check(KI, dev, c, state, slots, initial, offsets)


@pytest.mark.parametrize("states", [1, 2, 4, 7, 8, 15, 16, 17, 24, 32, 33, 64, 65, 100, 128, 129, 200, 256])
def test_selective_scan_states(KI, dev, states):
    offsets = [0, 70, 71, 200]
    c, state, slots, initial = _scan_case(states, 200, 3, 24, states, 2, "float32", dev, soft=False, gate=False)
    c["D"] = None
    _scan_check(KI, dev, c, state, slots, initial, offsets)


@pytest.mark.parametrize("n,channels", [(12, 700), (256, 40), (300, 40)])
def test_selective_scan_longest_first(KI, dev, n, channels):
    """More blocks than SMs: sequences are taken by length, equal ones and empty ones among them."""
    import torch

    lengths = torch.randint(0, 9, (n,), generator=_rng(n)).tolist()
    lengths[n // 2] = 40
    offsets = [0] + np.cumsum(lengths).tolist()
    c, state, slots, initial = _scan_case(n, offsets[-1] + 3, n, channels, 16, 1, "float32", dev)
    slots[3] = -1
    _scan_check(KI, dev, c, state, slots, initial, offsets)


def test_one_slot_named_twice(KI, dev):
    """Not allowed; the call still only touches that slot."""
    import torch

    offsets = torch.tensor([0, 3, 50], dtype=torch.int32, device=dev)
    twice = torch.tensor([2, 2], dtype=torch.int32, device=dev)
    x, w, bias, state, *_ = _conv_case(1, [0, 3, 50], 64, 4, "float32", dev, more=0)
    c, hs, _, _ = _scan_case(4, 50, 2, 64, 16, 1, "float32", dev)
    keep, hkeep = state.clone(), hs.clone()
    KI.causal_conv(x, w, bias, state=state, offsets=offsets, slots=twice)
    KI.causal_conv_step(x[:2], w, bias, state=state, slots=twice)
    KI.selective_scan(**c, state=hs, offsets=offsets, slots=twice)
    step = {k: v[:2] if k in ("u", "delta", "B", "C", "z") else v for k, v in c.items()}
    KI.selective_scan_step(**step, state=hs, slots=twice)
    KI.context(0).check()
    rest = [i for i in range(state.shape[0]) if i != 2]
    assert torch.equal(state[rest], keep[rest]) and torch.equal(hs[rest], hkeep[rest])


def test_selective_scan_padding_and_strides(KI, dev):
    import torch

    offsets = LAYOUTS["several"]
    c, state, slots, initial = _scan_case(3, offsets[-1] + 3, len(offsets) - 1, 48, 16, 2, "bfloat16", dev)
    slots[0], slots[5] = -1, -3
    for key, lead in (("u", 3), ("delta", 16), ("z", 50)):
        big = torch.zeros(c[key].shape[0], 131, dtype=c[key].dtype, device=dev)
        big[:, lead:lead + 48] = c[key]
        c[key] = big[:, lead:lead + 48]
    bc = torch.zeros(c["u"].shape[0], 5 + 64, dtype=c["u"].dtype, device=dev)
    bc[:, 5:37], bc[:, 37:] = c["B"].flatten(1), c["C"].flatten(1)
    c["B"], c["C"] = bc[:, 5:37].unflatten(1, (2, 16)), bc[:, 37:].unflatten(1, (2, 16))
    cache = torch.zeros(state.shape[0], 3, 48, 16, device=dev)
    cache[:, 1] = state
    _scan_check(KI, dev, c, cache[:, 1], slots, initial, offsets)
    assert (cache[:, 0] == 0).all() and (cache[:, 2] == 0).all()


def test_selective_scan_far_values(KI, dev):
    """Large and tiny steps: softplus beyond 20 and far below 0, decays that vanish or stay one."""
    offsets = [0, 64]
    c, state, slots, initial = _scan_case(1, 64, 1, 32, 16, 1, "float32", dev)
    c["delta"][:20] = -40.0
    c["delta"][20:40] = 30.0
    c["delta_bias"][:] = 0.0
    c["A"][:, :4] = 0.0
    c["A"][:, 4:8] = -1e30
    _scan_check(KI, dev, c, state, slots, initial, offsets)


def test_selective_scan_without_state(KI, dev):
    import torch

    c, *_ = _scan_case(2, 100, 1, 40, 16, 1, "float32", dev)
    c["B"], c["C"] = c["B"][:, 0], c["C"][:, 0]
    want, err, _, _ = ref.scan(ref.f64(c["u"]), ref.f64(c["delta"]), ref.f64(c["A"]), ref.f64(c["B"])[:, None],
                               ref.f64(c["C"])[:, None], ref.f64(c["D"]), ref.f64(c["z"]), ref.f64(c["delta_bias"]), True,
                               [(0, 100)], [np.zeros((40, 16))])
    _within(KI.selective_scan(**c), want, err, torch.float32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,channels,states,groups", [(1, 8, 16, 1), (7, 70, 13, 2), (3, 33, 1, 1), (64, 512, 16, 1),
                                                         (5, 24, 64, 2), (2, 9, 100, 1)])
def test_selective_scan_step(KI, dev, dtype, rows, channels, states, groups):
    """Each row is a sequence of one token."""
    import torch

    c, state, slots, _ = _scan_case(rows + states, rows, rows, channels, states, groups, dtype, dev)
    if rows > 2:
        slots[1] = -1
    live = [r for r in range(rows) if slots[r] >= 0]
    want, err, last, lasterr = ref.scan(ref.f64(c["u"]), ref.f64(c["delta"]), ref.f64(c["A"]), ref.f64(c["B"]),
                                        ref.f64(c["C"]), ref.f64(c["D"]), ref.f64(c["z"]), ref.f64(c["delta_bias"]), True,
                                        [(r, r + 1) for r in live], [ref.f64(state[int(slots[r])]) for r in live])
    before = state.clone()
    out = torch.full(c["u"].shape, 3.0, dtype=c["u"].dtype, device=dev)
    got = KI.selective_scan_step(**c, state=state, slots=slots.to(dev), out=out)
    KI.context(0).check()
    _within(got[live], want[live], err[live], out.dtype)
    for r, l, e in zip(live, last, lasterr):
        _within(state[int(slots[r])], l, e, torch.float32)
    rest = [s for s in range(state.shape[0]) if s not in [int(slots[r]) for r in live]]
    assert torch.equal(state[rest], before[rest])
    assert all((got[r] == 3.0).all() for r in range(rows) if r not in live)


# ---------------------------------------------------------------------------------------------
# what a caller may get wrong, streams and graphs
# ---------------------------------------------------------------------------------------------
def test_bad_indices_are_reported_and_touch_nothing(KI, dev):
    """Slot numbers past the cache are padding, offsets past the rows are cut; check() says so once."""
    import torch

    x, w, bias, state, slots, initial, offsets = _conv_case(1, [0, 10, 30], 32, 4, "float32", dev, more=2)
    keep = state.clone()
    bad = torch.tensor([state.shape[0], 2 ** 31 - 1], dtype=torch.int32, device=dev)
    out = torch.full((32, 32), 4.0, device=dev)
    KI.causal_conv(x, w, bias, state=state, offsets=offsets.to(dev), slots=bad, out=out)
    with pytest.raises(KI.KIArgumentError):
        KI.context(0).check()
    KI.context(0).check()
    assert torch.equal(state, keep) and (out == 4.0).all()
    for off in ([0, 10, 99], [-5, 10, 20], [0, 20, 10]):
        guard = torch.full((34, 32), 4.0, device=dev)
        KI.causal_conv(x, w, bias, offsets=torch.tensor(off, dtype=torch.int32, device=dev), out=guard[1:33])
        with pytest.raises(KI.KIArgumentError):
            KI.context(0).check()
        assert (guard[0] == 4.0).all() and (guard[33] == 4.0).all()
    c, st, _, _ = _scan_case(4, 32, 2, 32, 16, 1, "float32", dev)
    keep = st.clone()
    out.fill_(4.0)
    KI.selective_scan(**c, state=st, offsets=offsets.to(dev), slots=bad, out=out)
    with pytest.raises(KI.KIArgumentError):
        KI.context(0).check()
    assert torch.equal(st, keep) and (out == 4.0).all()
    for off in ([0, 10, 99], [-5, 10, 20], [0, 20, 10]):
        guard = torch.full((34, 32), 4.0, device=dev)
        KI.selective_scan(**c, offsets=torch.tensor(off, dtype=torch.int32, device=dev), out=guard[1:33])
        with pytest.raises(KI.KIArgumentError):
            KI.context(0).check()
        assert (guard[0] == 4.0).all() and (guard[33] == 4.0).all()
    KI.selective_scan_step(**{k: v[:2] if k in ("u", "delta", "B", "C", "z") else v for k, v in c.items()}, state=st,
                           slots=bad)
    KI.causal_conv_step(x[:2], w, bias, state=state, slots=bad)
    with pytest.raises(KI.KIArgumentError):
        KI.context(0).check()
    assert torch.equal(st, keep)
    KI.context(0).check()


def test_refusals(KI, dev):
    import torch

    x = torch.randn(8, 32, device=dev)
    w, b = torch.randn(32, 4, device=dev), torch.randn(32, device=dev)
    st = torch.zeros(3, 3, 32, device=dev)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    q = torch.zeros(8, 32, dtype=torch.int8, device=dev)
    s8, s32 = torch.ones(8, device=dev), torch.ones(32, device=dev)
    W = torch.zeros(32, 32, dtype=torch.int8, device=dev)
    A, B = torch.zeros(32, 16, device=dev), torch.zeros(8, 16, device=dev)
    hs = torch.zeros(3, 32, 16, device=dev)
    calls = [
        lambda: KI.quantize_rows(x.double()),
        lambda: KI.quantize_rows(x.t()),
        lambda: KI.quantize_rows(x[0]),
        lambda: KI.quantize_rows(x, out=q[:, :31]),
        lambda: KI.quantize_rows(x, out=q, scale=s32),
        lambda: KI.quantize_rows(x, out=x.view(torch.int8)[:, :32]),
        lambda: KI.quantize_rows(x.cpu()),
        lambda: KI.int8_gemm(q, W[:, :31], s8, s32),
        lambda: KI.int8_gemm(q, W, s32, s32),
        lambda: KI.int8_gemm(q, W, s8, s32, dtype=torch.int32),
        lambda: KI.int8_gemm(q, W, s8, s32, bias=s8),
        lambda: KI.int8_gemm(q, W.t(), s8, s32),
        lambda: KI.int8_gemm(q, W, s8, s32, out=torch.empty(8, 31, device=dev)),
        lambda: KI.int8_gemm(q, W, s8.cpu(), s32),
        lambda: KI.causal_conv(x, w.half(), b),
        lambda: KI.causal_conv(x, w[:, :1].contiguous(), b),
        lambda: KI.causal_conv(x, torch.randn(32, 9, device=dev), b),
        lambda: KI.causal_conv(x, w, b, activation="relu"),
        lambda: KI.causal_conv(x, w, b, state=st.half()),
        lambda: KI.causal_conv(x, w, b, state=st[:, :2]),
        lambda: KI.causal_conv(x, w, b, slots=i32(0)),
        lambda: KI.causal_conv(x, w, b, initial=torch.ones(1, dtype=torch.bool, device=dev)),
        lambda: KI.causal_conv(x, w, b, state=st, initial=torch.ones(2, dtype=torch.bool, device=dev)),
        lambda: KI.causal_conv(x, w, b, offsets=i32(0, 8).long()),
        lambda: KI.causal_conv(x, w, b, state=st, offsets=i32(0, 1, 2, 3, 8)),
        lambda: KI.causal_conv(x, w, b, out=x),
        lambda: KI.causal_conv(x, w, b, state=x[:3].view(1, 3, 32)),
        lambda: KI.causal_conv_step(x, w, b),
        lambda: KI.causal_conv_step(x, w, b, state=st),
        lambda: KI.selective_scan(x, x, A, B, B[:7]),
        lambda: KI.selective_scan(x, x.half(), A, B, B),
        lambda: KI.selective_scan(x, x, A.double(), B, B),
        lambda: KI.selective_scan(x, x, A, B, B, state=hs.half()),
        lambda: KI.selective_scan(x, x, A, B, B, z=x[:, :31]),
        lambda: KI.selective_scan(x, x, A, B.view(8, 2, 8), B.view(8, 2, 8)),
        lambda: KI.selective_scan(x, x, torch.zeros(32, 257, device=dev), torch.zeros(8, 257, device=dev),
                                  torch.zeros(8, 257, device=dev)),
        lambda: KI.selective_scan(x, x, A, torch.zeros(8, 3, 16, device=dev), torch.zeros(8, 3, 16, device=dev)),
        lambda: KI.selective_scan(x, x, A, B, B, out=x),
        lambda: KI.selective_scan_step(x, x, A, B, B),
        lambda: KI.selective_scan_step(x, x, A, B, B, state=hs),
        lambda: KI.reduce(x.half()),      # the new element types belong to the layer's operators only
        lambda: KI.scan(x.bfloat16().view(-1)),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(KI.KIArgumentError):
            call()
            pytest.fail(f"call {i} was accepted")
    KI.context(0).check()


def test_refusals_at_the_c_interface(KI, dev):
    """What the Python layer cannot ask for: null pointers, strides below a row, unknown types."""
    import ctypes

    import torch

    c = KI.context(0)
    x = torch.zeros(64, 64, device=dev)
    p, s = x.data_ptr(), KI._stream_ptr(None, 0)
    q = torch.zeros(64, 64, dtype=torch.int8, device=dev).data_ptr()
    sc = torch.zeros(64, device=dev).data_ptr()
    y = torch.zeros(64, 64, device=dev).data_ptr()

    def refused(name, *args):
        with pytest.raises(KI.KIArgumentError):
            c.call(name, *args)

    refused("ki_quantize_rows", 9, p, 4, 4, 4, q, 4, sc, s)
    refused("ki_quantize_rows", 8, None, 4, 4, 4, q, 4, sc, s)
    refused("ki_quantize_rows", 8, p, 4, 4, 3, q, 4, sc, s)
    refused("ki_quantize_rows", 8, p + 2, 4, 4, 4, q, 4, sc, s)
    refused("ki_gemm_i8", q, 64, q, 64, sc, sc, None, 9, y, 64, 4, 4, 4, s)
    refused("ki_gemm_i8", q, 64, q, 64, None, sc, None, 8, y, 64, 4, 4, 4, s)
    refused("ki_gemm_i8", q, 3, q, 64, sc, sc, None, 8, y, 64, 4, 4, 4, s)
    refused("ki_gemm_i8", q, 64, q, 64, sc, sc, None, 8, y, 3, 4, 4, 4, s)
    refused("ki_gemm_i8", q, 64, q, 64, sc, y, None, 8, y, 64, 4, 4, 4, s)
    refused("ki_causal_conv", 10, None, 64, p, None, None, 0, 0, None, None, None, 1, y, 64, 4, 4, 4, 0, s)
    refused("ki_causal_conv", 8, p, 64, p, None, None, 0, 0, None, None, None, 2, y, 64, 4, 4, 4, 0, s)
    refused("ki_causal_conv", 8, p, 64, p, None, sc, 3, 2, None, None, None, 1, y, 64, 4, 4, 4, 0, s)
    refused("ki_causal_conv_step", 8, p, 64, p, None, None, 0, 0, None, y, 64, 4, 4, 4, 0, s)
    refused("ki_selective_scan", 8, p, 64, p, 64, sc, p, 64, p, 64, None, None, 0, None, 0, None, 0, 0, None, None, None, 1, y,
            64, 4, 6, 4, 4, s)
    refused("ki_selective_scan", 8, p, 64, p, 64, sc, p, 64, p, 64, None, None, 0, None, 0, None, 0, 0, None, None, None, 1, y,
            64, 4, 4, 0, 1, s)
    refused("ki_selective_scan_step", 8, p, 64, p, 64, sc, p, 64, p, 64, None, None, 0, None, 0, None, 0, 0, None, y, 64, 4, 4, 4,
            1, s)
    assert ctypes.sizeof(ctypes.c_void_p) == 8


def test_refuses_rows_at_the_end_of_32_bits(KI, dev):
    """A thread's index passes the row's end by its stride before it stops, so rows end that much below 2^31."""
    import torch

    x = torch.zeros(8, device=dev)
    for cols in (0x7ffff001, 0x7fffffff, 1 << 31, 1 << 40):
        with pytest.raises(KI.KIArgumentError, match="too many columns"):
            KI.context(0).call("ki_quantize_rows", 8, x.data_ptr() + 4, 1, cols, cols, x.data_ptr(), cols, x.data_ptr(),
                               KI._stream_ptr(None, 0))


def test_refuses_sequences_at_the_end_of_32_bits(KI, dev):
    """A thread's index passes the last sequence by its stride before it stops, so their number ends that much below 2^31."""
    import torch

    x = torch.zeros(64, device=dev)
    p, s, c = x.data_ptr(), KI._stream_ptr(None, 0), KI.context(0)
    for n in (0x7ffff001, 0x7ffffffe, 1 << 31, 1 << 40):
        for name, args in (
                ("ki_causal_conv", (8, p, 4, p, None, None, 0, 0, None, None, p, n, p, 4, 4, 4, 4, 0, s)),
                ("ki_causal_conv_step", (8, p, 4, p, None, p, 12, n, None, p, 4, n, 4, 4, 0, s)),
                ("ki_selective_scan", (8, p, 4, p, 4, p, p, 4, p, 4, None, None, 0, None, 0, None, 0, 0, None, None, p, n, p,
                                       4, 4, 4, 4, 1, s)),
                ("ki_selective_scan_step", (8, p, 4, p, 4, p, p, 4, p, 4, None, None, 0, None, 0, p, 16, n, None, p, 4, n, 4, 4,
                                            1, s))):
            with pytest.raises(KI.KIArgumentError, match="too many"):
                c.call(name, *args)


def _layer(dev, seed=11, d=96, inner=160, states=16, rank=8):
    """Weights of one state-space layer: int8 projections with channel scales, convolution and scan parameters."""
    import torch

    g = _rng(seed)

    def lin(n, k):
        return (torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8).to(dev),
                (torch.rand(n, generator=g) * 0.01 + 0.01).to(dev) / k ** 0.5)

    return {"in": lin(2 * inner, d), "x": lin(rank + 2 * states, inner), "dt": lin(inner, rank), "out": lin(d, inner),
            "w": _normal(g, inner, 4, scale=0.5, dtype="bfloat16"), "b": _normal(g, inner, scale=0.1, dtype="bfloat16"),
            "A": -torch.exp(_normal(g, inner, states)), "D": _normal(g, inner), "bias": _normal(g, inner) - 2,
            "inner": inner, "states": states, "rank": rank}


def _linear(KI, x, weight, **kw):
    q, s = KI.quantize_rows(x)
    return KI.int8_gemm(q, weight[0], s, weight[1], **kw)


def _mix(KI, L, h, conv, scan):
    xz = _linear(KI, h, L["in"])
    x = conv(xz[:, :L["inner"]], L["w"], L["b"], activation="silu")
    p = _linear(KI, x, L["x"])
    dt = _linear(KI, p[:, :L["rank"]], L["dt"])
    B, C = p[:, L["rank"]:L["rank"] + L["states"]], p[:, L["rank"] + L["states"]:]
    y = scan(x, dt, L["A"], B, C, D=L["D"], z=xz[:, L["inner"]:], delta_bias=L["bias"], softplus=True)
    return y, _linear(KI, y, L["out"])


def test_layer_prompt_then_tokens(KI, dev):
    """A whole layer over ragged prompts, then token by token: as one pass over everything.

    The first projections, the convolution and their quantisation see the same rows in both and give the same bits; only
    the scan may order its sums otherwise, so y may differ by two half steps of bf16, 2^-7 |y|.  The dequantised y then
    differs by that and by half a quantum on either side, and the last projection by those times |w|, and by the two
    roundings of its own result.  The Float32 states: 46 steps of at most 32 half steps each."""
    import functools

    import torch

    L = _layer(dev)
    lengths, more = [3, 1, 17, 40], 6
    n = len(lengths)
    g = _rng(2)
    h = [_normal(g, l + more, 96, dtype="bfloat16") for l in lengths]
    slots = torch.tensor([5, 0, 3, 1], dtype=torch.int32, device=dev)
    new = torch.zeros(n, dtype=torch.bool, device=dev)

    def caches():
        return (torch.full((6, 3, L["inner"]), 9.0, dtype=torch.bfloat16, device=dev),
                torch.full((6, L["inner"], 16), 9.0, device=dev))

    def prompts(rows, cs, ss):
        off = torch.tensor(np.cumsum([0] + [r.shape[0] for r in rows]), dtype=torch.int32, device=dev)
        kw = dict(offsets=off, slots=slots, initial=new)
        both = _mix(KI, L, torch.cat(rows), functools.partial(KI.causal_conv, state=cs, **kw),
                    functools.partial(KI.selective_scan, state=ss, **kw))
        return list(zip(*(v.split([r.shape[0] for r in rows]) for v in both)))

    c1, s1 = caches()
    whole = prompts(h, c1, s1)
    c2, s2 = caches()
    parts = [[p] for p in prompts([r[:l] for r, l in zip(h, lengths)], c2, s2)]
    for t in range(more):
        step = _mix(KI, L, torch.stack([r[l + t] for r, l in zip(h, lengths)]),
                    functools.partial(KI.causal_conv_step, state=c2, slots=slots),
                    functools.partial(KI.selective_scan_step, state=s2, slots=slots))
        for i in range(n):
            parts[i].append(tuple(v[i:i + 1] for v in step))
    KI.context(0).check()
    assert torch.equal(c1, c2)
    assert float((s1 - s2).abs().max()) <= 46 * 32 * ref.U * float(s1.abs().max())
    assert (s1[[2, 4]] == 9.0).all() and (c1[[2, 4]] == 9.0).all()
    for i in range(n):
        (y1, a), (y2, b) = whole[i], (torch.cat(v) for v in zip(*parts[i]))
        y1, y2, a, b = (v.double() for v in (y1, y2, a, b))
        assert torch.isfinite(a).all() and ((y1 - y2).abs() <= 2.0 ** -7 * y1.abs() + 1e-30).all()
        quantum = y1.abs().amax(1, keepdim=True) * (1 + 2.0 ** -7) / 127
        bound = (2.0 ** -7 * y1.abs() + quantum) @ L["out"][0].double().abs().t() * L["out"][1].double()
        assert ((a - b).abs() <= bound + 2.0 ** -7 * a.abs()).all()


def test_streams_and_graphs(KI, dev):
    """Two streams at once through one context, and two captured graphs replayed in turn: the same results as eager."""
    import torch

    L = _layer(dev, seed=5)
    g = _rng(8)
    h = [_normal(g, 30, 96, dtype="bfloat16") for _ in range(2)]
    import functools

    def state():
        return (torch.zeros(1, 3, L["inner"], dtype=torch.bfloat16, device=dev), torch.zeros(1, L["inner"], 16, device=dev))

    def run(x, c, s):
        return _mix(KI, L, x, functools.partial(KI.causal_conv, state=c), functools.partial(KI.selective_scan, state=s))[1]

    want = []
    for x in h:
        c, s = state()
        want.append((run(x, c, s).clone(), run(x, c, s).clone(), s))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    st = [state() for _ in range(2)]
    got = [[], []]
    torch.cuda.synchronize()
    for _ in range(2):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(run(h[i], *st[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(got[i][0], want[i][0]) and torch.equal(got[i][1], want[i][1])
        assert torch.equal(st[i][1], want[i][2])
    st = [state() for _ in range(2)]
    graphs, outs = [], []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            outs.append(run(h[i], *st[i]))
        graphs.append(graph)
    for step in range(2):
        for i in range(2):
            graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i], want[i][step])
    KI.context(0).check()


def test_stream_argument_owns_the_output(KI, dev):
    """An output made for another stream is that stream's memory: its block is not handed out to the current stream while
    the other stream still writes it."""
    import torch

    s = torch.cuda.Stream(dev)
    x = torch.randn(512, 1024, device=dev)
    torch.cuda.synchronize()
    for _ in range(20):
        q, sc = KI.quantize_rows(x, stream=s)
        del q, sc
        junk = torch.full((512, 1024), 55, dtype=torch.int8, device=dev)
        del junk
    q, sc = KI.quantize_rows(x, stream=s)
    s.synchronize()
    ws, wq = ref.quantize(x.cpu().numpy())
    assert np.array_equal(q.cpu().numpy(), wq)


def test_offsets_beyond_32_bits(KI, dev):
    """Rows so far apart, and a cache so large, that element offsets pass 2^31."""
    import torch

    ld = 1 << 20
    rows = 2200  # 2200 * 2^20 > 2^31 elements
    try:
        big = torch.empty(rows, ld, dtype=torch.bfloat16, device=dev)
    except torch.OutOfMemoryError:
        pytest.skip("needs 5 GB")
    x = big[:, 64:64 + 32]
    x.copy_(_normal(_rng(1), rows, 32, dtype="bfloat16"))
    dense = x.contiguous()
    w = _normal(_rng(2), 32, 4, dtype="bfloat16")
    assert torch.equal(KI.causal_conv(x, w, activation="silu"), KI.causal_conv(dense, w, activation="silu"))
    q, s = KI.quantize_rows(x)
    q2, s2 = KI.quantize_rows(dense)
    assert torch.equal(q, q2) and torch.equal(s, s2)
    c, state, _, _ = _scan_case(1, rows, 1, 32, 16, 1, "bfloat16", dev)
    want = KI.selective_scan(**c)
    c["u"] = x.copy_(c["u"])
    assert torch.equal(KI.selective_scan(**c), want)
    out = torch.empty_like(big)[:, :32]
    assert torch.equal(KI.selective_scan(**c, out=out), want)
    del out
    wide = big.view(torch.int8)
    a = wide[:, 4096:4096 + 48]
    a.copy_(torch.randint(-127, 128, (rows, 48), dtype=torch.int8, generator=_rng(3)))
    ws = torch.ones(40, device=dev)
    wt = torch.randint(-127, 128, (40, 48), dtype=torch.int8, generator=_rng(4)).to(dev)
    sa = torch.ones(rows, device=dev)
    assert torch.equal(KI.int8_gemm(a, wt, sa, ws), KI.int8_gemm(a.contiguous(), wt, sa, ws))
    KI.context(0).check()


# ---------------------------------------------------------------------------------------------
# infinities and NaN
# ---------------------------------------------------------------------------------------------
def _as_defined(got, want, err, dtype):
    """NaN and infinities where the definition has them, and elsewhere within the bound."""
    got = ref.f64(got)
    assert np.array_equal(np.isnan(got), np.isnan(want)), np.argwhere(np.isnan(got) != np.isnan(want))[:5]
    big = np.isinf(want)
    assert np.array_equal(got[big], want[big])
    fin = np.isfinite(want)
    assert (np.abs(got[fin] - want[fin]) <= ref.stored(want[fin], err[fin], dtype)).all()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("soft", [False, True])
@pytest.mark.parametrize("states,channels", [(1, 16), (5, 16), (13, 16), (16, 16), (17, 16), (24, 16), (33, 16), (100, 16),
                                             (200, 16), (5, 2400), (13, 1200), (13, 2400), (24, 1200)])
def test_selective_scan_of_infinities(KI, dev, dtype, soft, states, channels):
    """An infinite input makes its channel infinite, not NaN, whatever the number of states, in the prompt's form and in
    the single token's.  B, C and D are positive, so that no sum has infinities of both signs; decays stay far from zero
    (at most 40 steps of 0.3), so that infinite states stay infinite."""
    import torch

    T = 40
    g = _rng(states + channels)
    c, state, _, _ = _scan_case(states, T, 1, channels, states, 1, dtype, dev, soft=soft)
    c["B"], c["C"] = c["B"].abs() + 0.1, c["C"].abs() + 0.1
    c["D"] = c["D"].abs()
    c["A"] = -(torch.rand(channels, states, generator=g) + 0.5).to(dev)
    if soft:
        c["delta_bias"] = torch.full((channels,), -3.0, device=dev)
        c["delta"] = c["delta"].clamp(-1, 1)
        c["delta"][3, 6] = -1e4  # a step of zero
    inf = float("inf")
    c["u"][5, 0], c["u"][33, 1] = inf, -inf
    c["delta"][9, 2], c["u"][9, 2] = inf, 0.75
    c["z"][11, 3], c["z"][12, 4] = inf, -inf
    c["u"][13, 5] = float("nan")
    c["z"][14, 7] = float("nan")
    with np.errstate(all="ignore"):
        want, err, last, lasterr = ref.scan(*(ref.f64(c[k]) for k in ("u", "delta", "A", "B", "C", "D", "z")),
                                            ref.f64(c["delta_bias"]) if soft else None, soft, [(0, T)], [ref.f64(state[0])])
    assert np.isinf(want[5:, 0]).all() and np.isinf(want[33:, 1]).all() and np.isinf(want[9:, 2]).all()
    held, token = state.clone(), state.clone()
    _as_defined(KI.selective_scan(**c, state=held), want, err, c["u"].dtype)
    _as_defined(held[0], last[0], lasterr[0], torch.float32)
    rows = {k: v for k, v in c.items() if k in ("u", "delta", "B", "C", "z")}
    fixed = {k: v for k, v in c.items() if k not in rows}
    steps = [KI.selective_scan_step(**{k: v[t:t + 1] for k, v in rows.items()}, **fixed, state=token) for t in range(T)]
    _as_defined(torch.cat(steps), want, err, c["u"].dtype)
    _as_defined(token[0], last[0], lasterr[0], torch.float32)
    KI.context(0).check()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("states,channels", [(16, 24), (13, 24), (16, 2400), (64, 24)])
def test_selective_scan_of_the_lowest_decays(KI, dev, dtype, states, channels):
    """A of the lowest value forgets a state at any step, but a step of zero leaves it as it is; so does minus infinity
    where no step is zero."""
    import torch

    T = 37
    c, state, _, _ = _scan_case(states, T, 1, channels, states, 1, dtype, dev, soft=False)
    c["delta"] = c["delta"] + 0.01
    low = dict(c, A=c["A"].clone())
    low["A"][:, 0] = -1e30
    low["A"][:, -1] = -float("inf")
    same = dict(c, A=low["A"].clamp(min=-1e30))
    held = [state.clone(), state.clone()]
    assert torch.equal(KI.selective_scan(**low, state=held[0]), KI.selective_scan(**same, state=held[1]))
    assert torch.equal(*held)
    c["A"][:, 0] = torch.finfo(torch.float32).min
    c["A"][1, -1] = torch.finfo(torch.float32).min
    c["delta"][::3] = 0
    want, err, last, lasterr = ref.scan(*(ref.f64(c[k]) for k in ("u", "delta", "A", "B", "C", "D", "z")), None, False,
                                        [(0, T)], [ref.f64(state[0])])
    held, token = state.clone(), state.clone()
    _within(KI.selective_scan(**c, state=held), want, err, c["u"].dtype)
    _within(held[0], last[0], lasterr[0], torch.float32)
    rows = {k: v for k, v in c.items() if k in ("u", "delta", "B", "C", "z")}
    fixed = {k: v for k, v in c.items() if k not in rows}
    steps = [KI.selective_scan_step(**{k: v[t:t + 1] for k, v in rows.items()}, **fixed, state=token) for t in range(T)]
    _within(torch.cat(steps), want, err, c["u"].dtype)
    _within(token[0], last[0], lasterr[0], torch.float32)
    KI.context(0).check()


# ---------------------------------------------------------------------------------------------
# sizes that reach every layout of lanes, rows per block, run length and a pair's third tile (148 SMs)
# ---------------------------------------------------------------------------------------------
def _as_views(c, channels, dev):
    """u, delta and z as columns of wider rows that start anywhere, B and C as slices of one projection's rows."""
    import torch

    for key, lead in (("u", 1), ("delta", 3), ("z", channels + 1)):
        big = torch.zeros(c[key].shape[0], 2 * channels + 5, dtype=c[key].dtype, device=dev)
        big[:, lead:lead + channels] = c[key]
        c[key] = big[:, lead:lead + channels]
    groups, states = c["B"].shape[1:]
    n = groups * states
    bc = torch.zeros(c["u"].shape[0], 3 + 2 * n, dtype=c["u"].dtype, device=dev)
    bc[:, 3:3 + n], bc[:, 3 + n:] = c["B"].flatten(1), c["C"].flatten(1)
    c["B"], c["C"] = bc[:, 3:3 + n].unflatten(1, (groups, states)), bc[:, 3 + n:].unflatten(1, (groups, states))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("states,channels,groups,views",
                         [(8, 48, 1, False), (5, 1200, 2, True), (8, 1200, 1, False),       # 8 and 4 lanes for 8 states
                          (16, 64, 1, False), (13, 800, 1, True), (16, 800, 2, False),      # 16, 8
                          (16, 1200, 1, False), (16, 1202, 2, True), (13, 1200, 1, False),  # and 4 lanes for 16
                          (32, 64, 1, True), (24, 800, 1, False), (32, 800, 2, True),       # 16 and 8 lanes for 32
                          (64, 40, 1, False), (40, 48, 2, True), (128, 40, 1, True), (100, 24, 1, False),
                          (256, 40, 1, False), (200, 24, 2, True)])
def test_selective_scan_lanes(KI, dev, dtype, states, channels, groups, views):
    """Two sequences of four and two chunks of tokens, on every number of lanes per channel and states per lane."""
    offsets = [0, 37, 140]
    c, state, slots, initial = _scan_case(states + channels, 143, 2, channels, states, groups, dtype, dev)
    if views:
        _as_views(c, channels, dev)
    initial[:] = False
    initial[1] = True
    _scan_check(KI, dev, c, state, slots, initial, offsets)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,channels,states,groups,views",
                         [(127, 1024, 8, 1, False), (131, 1030, 5, 2, True), (131, 1200, 16, 1, False), (130, 1030, 13, 2, True),
                          (67, 1200, 32, 1, False), (66, 1202, 24, 2, True), (35, 600, 64, 1, False), (21, 300, 128, 1, True),
                          (22, 302, 100, 2, False), (21, 300, 256, 1, False), (23, 301, 200, 1, True)])
def test_selective_scan_step_four_rows_per_block(KI, dev, dtype, rows, channels, states, groups, views):
    """Rows enough for four to a block, their number no multiple of four; padding inside a group and at the end."""
    import torch

    c, state, slots, _ = _scan_case(rows + states, rows, rows, channels, states, groups, dtype, dev)
    if views:
        _as_views(c, channels, dev)
    for r in (1, 6, 8, 9, 10, 11, rows - 1):
        slots[r] = -1 - r
    live = [r for r in range(rows) if slots[r] >= 0]
    want, err, last, lasterr = ref.scan(ref.f64(c["u"]), ref.f64(c["delta"]), ref.f64(c["A"]), ref.f64(c["B"]),
                                        ref.f64(c["C"]), ref.f64(c["D"]), ref.f64(c["z"]), ref.f64(c["delta_bias"]), True,
                                        [(r, r + 1) for r in live], [ref.f64(state[int(slots[r])]) for r in live])
    before = state.clone()
    out = torch.full(c["u"].shape, 3.0, dtype=c["u"].dtype, device=dev)
    got = KI.selective_scan_step(**c, state=state, slots=slots.to(dev), out=out)
    KI.context(0).check()
    _within(got[live], want[live], err[live], out.dtype)
    _within(state[slots[live].long().to(dev)], np.stack(last), np.stack(lasterr), torch.float32)
    named = set(slots[live].tolist())
    rest = [s for s in range(state.shape[0]) if s not in named]
    assert torch.equal(state[rest], before[rest])
    assert (got[[r for r in range(rows) if r not in live]] == 3.0).all()


@pytest.mark.parametrize("dtype,channels,width,tokens",
                         [("bfloat16", 516, 2, 18945), ("bfloat16", 516, 4, 18945), ("bfloat16", 516, 8, 18945),  # runs of 64
                          ("float32", 258, 3, 18945), ("float16", 129, 4, 18945),
                          ("bfloat16", 516, 4, 9473), ("float32", 258, 6, 9473), ("float32", 129, 7, 9473),        # of 32
                          ("float16", 516, 5, 5001)])                                                             # of 16
def test_causal_conv_long_runs(KI, dev, dtype, channels, width, tokens):
    """Runs of tokens in which every ring slot is filled many times; sequences that begin a token before, at and after the
    places where runs begin, short and empty ones among them, continued from their slots."""
    starts = {64 * i + i % 3 - 1 for i in range(1, 60)} | {16 * i + 1 for i in range(250, 262)} | {32 * i for i in range(140, 150)}
    offsets = [0, 0] + sorted(starts | {700, 701, 703, 704 + width}) + [tokens - 9, tokens - 9, tokens - 2]
    x, w, bias, state, slots, initial, off = _conv_case(width, offsets, channels, width, dtype, dev, more=2)
    slots[5] = -1
    _conv_check(KI, dev, x, w, bias, state, slots, initial, off, "silu", dtype)


@pytest.mark.parametrize("M,N,K", [(3850, 3900, 144), (4609, 4700, 16), (2100, 12800, 48)])
def test_int8_gemm_of_many_tiles(KI, dev, M, N, K):
    """Three to seven tiles of 256 x 256 for each CTA pair, so that accumulators and scales are used again, with so few K
    blocks that the MMAs run ahead of the epilogue; every element."""
    import torch

    a, w, sa, sw, bias = _operands(M + N + K, M, N, K, dev)
    s = (a.double() @ w.double().t()) * sa.double()[:, None] * sw.double()  # (the integer sums are exact)
    for dtype, b in ((torch.float32, None), (torch.bfloat16, bias), (torch.float16, bias)):
        want = s if b is None else s + b.double()
        err = 4 * ref.U * s.abs() + (0 if b is None else ref.U * want.abs())
        bound = err + ref.HALF_STEP[dtype] * (want.abs() + err) + ref.TINY[dtype]
        big = torch.full((M + 2, N + 3), 5.0, dtype=dtype, device=dev)
        out = KI.int8_gemm(a, w, sa, sw, bias=b, out=big[1:-1, 1:1 + N])
        KI.context(0).check()
        assert torch.isfinite(out).all() and ((out.double() - want).abs() <= bound).all()
        big[1:-1, 1:1 + N] = 5.0
        assert (big == 5.0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", [None, "silu"])
@pytest.mark.parametrize("channels,width", [(16, 4), (17, 3), (24, 8)])
def test_causal_conv_of_infinities(KI, dev, dtype, act, channels, width):
    """Infinities, NaN and values of the type's size in inputs and states stay in the outputs that they reach."""
    import torch

    T = 30
    x, w, bias, state, *_ = _conv_case(channels, [0, T], channels, width, dtype, dev, more=0)
    inf, top = float("inf"), torch.finfo(x.dtype).max
    w[:, :] = w.abs().clamp(0.1, 0.9)
    x[5, 0], x[6, 1], x[9, 2] = inf, -inf, float("nan")
    x[12, 3], x[13, 4] = top, -top
    x[14, 5], x[15, 5] = inf, -inf
    state[0, 0, 6], state[0, width - 2, 7] = inf, float("nan")
    with np.errstate(all="ignore"):
        want, err, last = ref.conv(ref.f64(x), ref.f64(w), ref.f64(bias), [(0, T)], [ref.f64(state[0])], act == "silu")
    held, token = state.clone(), state.clone()
    _as_defined(KI.causal_conv(x, w, bias, state=held, activation=act), want, err, x.dtype)
    steps = [KI.causal_conv_step(x[t:t + 1], w, bias, state=token, activation=act) for t in range(T)]
    _as_defined(torch.cat(steps), want, err, x.dtype)
    assert np.array_equal(ref.f64(held[0]), last[0], equal_nan=True) and torch.equal(held, token)
    KI.context(0).check()


@pytest.mark.parametrize("N", [1153, 1920, 1921, 2304])
@pytest.mark.parametrize("M,K", [(1, 1040), (1, 1031), (48, 1040), (33, 1031), (128, 1040), (100, 1031)])
def test_int8_gemm_in_clusters(KI, dev, M, N, K):
    """10 to 18 tiles, whose K blocks are shared by four or eight CTAs."""
    import torch

    a, w, sa, sw, bias = _operands(M + N + K, M, N, K, dev)
    for dtype, b in ((torch.float32, None), (torch.bfloat16, bias)):
        out = KI.int8_gemm(a, w, sa, sw, bias=b, dtype=dtype)
        KI.context(0).check()
        _check_product(out, a, w, sa, sw, b, dtype)
