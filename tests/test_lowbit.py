"""Narrow block formats of the Linear layers (apn_amd.lowbit): the 8-bit activation checkpoint with
the products that write and read it, and microscaled 4-bit rows with their product, against plain
implementations in 64 bits written from the formats' definition.

Tolerances. Codes and read-back values are compared for equality: every step of the definition is
exact in float32 (powers of two, one rounding). Float outputs are sums of n products p_i: summed in
float32 in any order their error is at most (n + 16) u S, S = sum |p_i|, with u = 2^-23 (one unit in
the last place per addition, so truncating adders are covered; 16 covers the bias, the activation and
the joins of split sums). Products of float32 factors are taken as six bf16 products of three-way cut
factors; what is left out is at most 2^-21 |p_i| (mid lo + lo mid + lo lo, with mid < 2^-7 and
lo < 2^-15 of the factor). A 16-bit output adds half a step of its type.
"""
import math

import pytest
import torch

gpu = pytest.mark.gpu
autograd = pytest.mark.autograd
BLOCK = 32
U = 2.0 ** -23
CUT = 2.0 ** -21


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need an MI355X"
    return torch.device("cuda")


# --- the formats from their definition, in 64 bits, on the CPU ---------------------------------------

def _blocks(x):
    M, K = x.shape
    B = -(-K // BLOCK)
    b = torch.zeros(M, B * BLOCK, dtype=torch.float64)
    b[:, :K] = x.double().cpu()
    return b.reshape(M, B, BLOCK)


def _floor_log2(a):
    m, e = torch.frexp(a)
    return torch.where(a > 0, e - 1, torch.full_like(e, -2000)), 2 * m


def ref_q8(x):
    """(codes [M, 32 B] int64, scale bytes [M, B], values [M, K] float64)."""
    b = _blocks(x)
    fine = torch.isfinite(b).all(-1)
    top = torch.where(fine, b.abs().amax(-1), torch.zeros(()).double())
    e, m = _floor_log2(top)
    s = (e - 6 + (m >= 127.5 / 64).int()).clamp(-127, 121)
    q = torch.round(torch.where(fine[..., None], b.abs(), torch.zeros(()).double()) * 2.0 ** (-s[..., None]).double())
    q = q.clamp(max=127)
    neg = ~(b > 0)
    v = torch.where(neg, -q, q) * 2.0 ** s[..., None].double()
    v = torch.where(fine[..., None], v, torch.full_like(v, math.nan))
    byte = torch.where(fine, s + 127, torch.full_like(s, 255))
    codes = q.long() | (neg.long() << 7)
    return codes.reshape(len(x), -1), byte.long(), v.reshape(len(x), -1)[:, :x.shape[1]]


def ref_mx4(x):
    """(nibbles [M, 32 B] int64, scale bytes [M, B], values [M, K] float64)."""
    b = _blocks(x)
    fine = torch.isfinite(b).all(-1)
    top = torch.where(fine, b.abs().amax(-1), torch.zeros(()).double())
    s = (_floor_log2(top)[0] - 2).clamp(min=-127)
    a = torch.where(fine[..., None], b.abs(), torch.zeros(()).double()) * 2.0 ** (-s[..., None]).double()
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
    hi = torch.bucketize(a.clamp(max=6), grid).clamp(max=7)     # grid[hi - 1] < a <= grid[hi]
    lo = (hi - 1).clamp(min=0)
    up, down = grid[hi] - a, a - grid[lo]
    code = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    code = torch.where(a >= 6, torch.full_like(code, 7), code)
    neg = torch.signbit(b)
    v = torch.where(neg, -grid[code], grid[code]) * 2.0 ** s[..., None].double()
    v = torch.where(fine[..., None], v, torch.full_like(v, math.nan))
    byte = torch.where(fine, s + 127, torch.full_like(s, 255))
    return (code | (neg.long() << 3)).reshape(len(x), -1), byte.long(), v.reshape(len(x), -1)[:, :x.shape[1]]


def _awkward(M, K, seed, dtype=torch.float32):
    """Rows over the whole exponent range, with zeros, ties, subnormals, the largest values, all
    negative blocks, and non-finite values in some blocks."""
    g = torch.Generator().manual_seed(seed)
    span = 20.0 if dtype != torch.float16 else 3.0
    x = torch.randn(M, K, generator=g) * torch.exp(torch.randn(M, 1, generator=g) * span)
    big = torch.finfo(dtype).max
    tiny = torch.finfo(dtype).tiny
    rows = [torch.zeros(K), torch.full((K,), big), torch.full((K,), -big), torch.full((K,), tiny / 4),
            torch.arange(K) * 0.25, torch.arange(K) * 0.5 + 0.25, -torch.rand(K, generator=g),
            torch.full((K,), 127.5), torch.full((K,), 127.49), torch.linspace(-7.9, 7.9, K), torch.full((K,), -0.0)]
    for i, r in enumerate(rows[:M]):
        x[i] = r
    x = x.clamp(-big, big)
    if M > 20:
        x[15, K // 2], x[16, K - 1], x[17, 0] = math.inf, math.nan, -math.inf
    return x.to(dtype)


def _same(a, b):
    """Equal values, NaN where NaN."""
    a, b = a.double().cpu(), b.double().cpu()
    return a.shape == b.shape and bool(((a == b) | (torch.isnan(a) & torch.isnan(b))).all())


def _nibbles(codes):
    c = codes.cpu().long()
    return torch.stack([c & 15, c >> 4], -1).reshape(len(c), -1)


SHAPES = [(1, 1), (3, 31), (64, 32), (65, 33), (40, 191), (130, 257), (5, 4096), (2, 1000)]


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,K", SHAPES)
def test_q8_pack_equals_definition(dev, M, K, dtype):
    from apn_amd import lowbit as lb
    x = _awkward(M, K, M * 1000 + K, dtype)
    r = lb.q8_pack(x.to(dev))
    codes, byte, values = ref_q8(x)
    nb = -(-K // BLOCK)
    assert torch.equal(r.scales[:, :nb].long().cpu(), byte)
    assert not r.scales[:, nb:].any()
    fine = (byte < 255).repeat_interleave(BLOCK, 1)
    assert torch.equal(r.codes.long().cpu()[fine], codes[fine])
    assert torch.equal(r.codes.long().cpu() >> 7, codes >> 7)      # signs also where the block is not finite
    assert _same(r.dequantize(), values)
    assert _same(r.dequantize(torch.bfloat16), values)
    if dtype == torch.float32:
        half = values.float().half()
        assert _same(r.dequantize(torch.float16), half)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,K", SHAPES)
def test_mx4_quantize_equals_definition(dev, M, K, dtype):
    from apn_amd import lowbit as lb
    x = _awkward(M, K, M * 1000 + K + 1, dtype)
    r = lb.mx4_quantize(x.to(dev))
    codes, byte, values = ref_mx4(x)
    nb = -(-K // BLOCK)
    assert torch.equal(r.scales[:, :nb].long().cpu(), byte)
    assert not r.scales[:, nb:].any()
    fine = (byte < 255).repeat_interleave(BLOCK, 1)
    assert torch.equal(_nibbles(r.codes)[fine], codes[fine])
    assert _same(r.dequantize(), values)
    assert _same(r.dequantize(torch.bfloat16), values)
    assert _same(r.dequantize(torch.float16), values.float().half())


@gpu
@pytest.mark.parametrize("kind", ["q8_pack", "mx4_quantize"])
def test_pack_of_strided_rows(dev, kind):
    """Padded rows, rows that start off a 16-byte boundary, columns behind one another (a transpose),
    repeated rows, leading dimensions and no rows at all equal the packed copy of the same values."""
    from apn_amd import lowbit as lb
    pack = getattr(lb, kind)
    g = torch.Generator(device=dev).manual_seed(3)
    buf = torch.randn(70, 200, device=dev, generator=g)
    for x in (buf[:, :191], buf[:, 1:130], buf[3:, 5:6], buf.t(), buf[:1].expand(9, 200), buf[::3, :64],
              buf.reshape(7, 10, 200)[:, :, :77], buf[0]):
        a, b = pack(x), pack(x.reshape(-1, x.shape[-1]).clone())
        assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
    none = pack(buf[:0])
    assert none.shape == (0, 200) and none.dequantize().shape == (0, 200)


# --- products of the training step -------------------------------------------------------------------

CASES = [(1, 1, 1), (1, 256, 256), (2, 17, 33), (37, 33, 17), (64, 128, 128), (65, 191, 128), (300, 129, 97),
         (1000, 5, 513), (257, 640, 200), (129, 192, 64), (4097, 128, 128)]


def _rand(M, N, K, seed, dev):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn(M, K, device=dev, generator=g)
    w = torch.randn(N, K, device=dev, generator=g) / K ** 0.5
    b = torch.randn(N, device=dev, generator=g)
    dy = torch.randn(M, N, device=dev, generator=g)
    return x, w, b, dy


def _act64(v, slope):
    return v if slope is None else torch.where(v > 0, v, v * slope)


def _bound(n, S):
    return ((n + 16) * U + CUT) * S


def _within(a, ref, bound):
    over = (a.double() - ref).abs() - bound
    assert float(over.max()) <= 0, (float(over.max()), float((a.double() - ref).abs().max()))


@gpu
@pytest.mark.parametrize("slope", [None, 0.0, 0.01, -0.5, 2.0])
@pytest.mark.parametrize("M,K,N", CASES)
def test_linear_q8_vs_float64(dev, M, K, N, slope):
    from apn_amd import lowbit as lb
    x, w, b, _ = _rand(M, N, K, M + K + N, dev)
    y, kept = lb.linear_q8(x, w, b, slope)
    pre = x.double() @ w.double().t() + b.double()
    S = x.double().abs() @ w.double().abs().t() + b.double().abs()
    amp = 1.0 if slope is None else max(1.0, abs(slope))
    _within(y, _act64(pre, slope), amp * _bound(K, S))     # |act'| <= amp on both sides of the kink
    again = lb.q8_pack(y)      # the checkpoint is the packed output, bit for bit
    assert torch.equal(kept.codes, again.codes) and torch.equal(kept.scales, again.scales)
    y2, _ = lb.linear_q8(x, w, None, slope)
    _within(y2, _act64(pre - b.double(), slope), amp * _bound(K, S))


@gpu
@pytest.mark.parametrize("slope", [None, 0.0, 0.01])
@pytest.mark.parametrize("M,K,N", CASES)
def test_linear_q8_backward_vs_float64(dev, M, K, N, slope):
    """All three gradients against the formula in 64 bits on the checkpoints' values and signs (the
    reference reads the codes through the CPU definition, not through the kernels)."""
    from apn_amd import lowbit as lb
    x, w, b, dy = _rand(M, N, K, 7 * M + K + N, dev)
    x[:, ::7] *= 1e-3          # columns of another size within a block
    y = _act64(x.double() @ w.double().t() + b.double(), slope).float()
    xk, yk = lb.q8_pack(x), lb.q8_pack(y)
    dx, dw, db = lb.linear_q8_backward(dy, w, xk, yk if slope is not None else None, slope)
    xv = ref_q8(x)[2].to(dev)
    g = dy.double()
    if slope is not None:
        g = torch.where(y > 0, g, g * slope)
    _within(dx, g @ w.double(), _bound(N, g.abs() @ w.double().abs()))
    _within(dw, (xv.t() @ g).t(), _bound(M, (xv.abs().t() @ g.abs()).t()))
    _within(db, g.sum(0), _bound(M, g.abs().sum(0)))
    # each alone is what they are together, and twice the same bits
    for i in range(3):
        need = tuple(j == i for j in range(3))
        one = lb.linear_q8_backward(dy, w, xk, yk, slope, need) if slope is not None else \
            lb.linear_q8_backward(dy, w, xk, None, None, need)
        assert torch.equal(one[i], (dx, dw, db)[i]) and all(one[j] is None for j in range(3) if j != i)


# sizes around the kernels' limits: 16 | 17 rows, 192 | 193 columns of the reduction, 128-row and
# 128-column tiles, chunks of 32 columns, many tiles
EDGES = [(4, 300, 31), (5, 65, 100), (15, 4, 130), (16, 513, 63), (16, 7, 1), (17, 193, 193), (18, 1, 300), (128, 224, 128),
         (129, 225, 129), (700, 400, 260), (3000, 193, 1), (2500, 193, 700), (49200, 64, 33)]


@gpu
@pytest.mark.parametrize("slope", [None, 0.01])
@pytest.mark.parametrize("M,K,N", EDGES)
def test_linear_q8_kernel_edges(dev, M, K, N, slope):
    test_linear_q8_vs_float64(dev, M, K, N, slope)
    test_linear_q8_backward_vs_float64(dev, M, K, N, slope)


@gpu
@pytest.mark.parametrize("M", [3, 16, 40])
@pytest.mark.parametrize("K", [30, 250])
def test_linear_q8_masked_and_short_rows(dev, M, K):
    """Small and general row kernels: padded rows whose padding is NaN, gradients that are not finite
    where slope 0 masks them, one row that holds an infinity beside finite ones."""
    from apn_amd import lowbit as lb
    N = 70
    x, w, b, dy = _rand(M, N, K, M + K, dev)
    wide = torch.full((M, K + 3), math.nan, device=dev)
    wide[:, :K] = x
    y, kept = lb.linear_q8(wide[:, :K], w, b, 0.0)
    y1, kept1 = lb.linear_q8(x, w, b, 0.0)
    assert torch.equal(y, y1) and torch.equal(kept.codes, kept1.codes) and torch.equal(kept.scales, kept1.scales)
    x2 = x.clone()
    x2[1, K - 1] = math.inf
    y2, _ = lb.linear_q8(x2, w, b, None)
    y3, _ = lb.linear_q8(x, w, b, None)
    rest = torch.arange(M, device=dev) != 1
    assert torch.equal(y2[rest], y3[rest]) and not torch.isfinite(y2[1]).any()
    xk = lb.q8_pack(x)
    bad = torch.where(y > 0, dy, torch.full_like(dy, math.nan))
    for a, r in zip(lb.linear_q8_backward(bad, w, xk, kept, 0.0),
                    lb.linear_q8_backward(torch.where(y > 0, dy, torch.zeros_like(dy)), w, xk, kept, 0.0)):
        assert torch.equal(a, r)


@gpu
def test_linear_q8_large_rows_split_sums(dev):
    """A training step's row count: the weight gradient's split sums against 64 bits."""
    from apn_amd import lowbit as lb
    M, K, N = 203_008 + 37, 191, 128
    x, w, b, dy = _rand(M, N, K, 5, dev)
    y, yk = lb.linear_q8(x, w, b, 0.01)
    xk = lb.q8_pack(x)
    dx, dw, db = lb.linear_q8_backward(dy, w, xk, yk, 0.01)
    g = torch.where(y > 0, dy.double(), dy.double() * 0.01)
    xv = xk.dequantize().double()
    _within(dx, g @ w.double(), _bound(N, g.abs() @ w.double().abs()))
    # split sums: at most M / 64 chunks of 4 matrix steps of 3 products, then the splits
    _within(dw, (xv.t() @ g).t(), (4 * 3 * (M // 64 + 1) * U) * (xv.abs().t() @ g.abs()).t())
    _within(db, g.sum(0), M * U * g.abs().sum(0))
    rel = lambda a, r: float((a.double() - r).norm() / r.norm())  # noqa: E731
    assert rel(dw, (xv.t() @ g).t()) < 2e-6 and rel(db, g.sum(0)) < 2e-6   # sqrt-like, not worst case


@gpu
def test_linear_q8_signs_of_tiny_outputs(dev):
    """An output that rounds to code 0 still takes its own side of the kink in the backward pass, and
    an output of exactly 0 the slope's."""
    from apn_amd import lowbit as lb
    x = torch.zeros(4, 32, device=dev)
    x[:, 0] = torch.tensor([1e-9, -1e-9, 0.0, 3.0])
    w = torch.zeros(32, 32, device=dev)
    w[:, 0] = 1.0
    w[0, 0] = 1e6            # the block's scale: the others round to 0
    y, kept = lb.linear_q8(x, w, None, 0.25)
    assert float(kept.dequantize()[0, 1]) == 0.0 and float(y[0, 1]) > 0
    dy = torch.ones(4, 32, device=dev)
    _, _, db = lb.linear_q8_backward(dy[:1], w, None, lb.Q8Rows(kept.codes[:1], kept.scales[:1], 32), 0.25,
                                     (False, False, True))
    assert torch.equal(db, torch.ones(32, device=dev))
    for row in (1, 2):
        k = lb.Q8Rows(kept.codes[row:row + 1].clone(), kept.scales[row:row + 1].clone(), 32)
        _, _, db = lb.linear_q8_backward(dy[:1], w, None, k, 0.25, (False, False, True))
        assert torch.equal(db, torch.full((32,), 0.25, device=dev))


@gpu
def test_linear_q8_non_finite(dev):
    """Non-finite inputs reach every output that they reach in float32, and no other row; a gradient
    that slope 0 masks is dropped even where it is not finite; a checkpoint block that is not finite
    makes its columns of dw NaN and no others."""
    from apn_amd import lowbit as lb
    x, w, b, dy = _rand(100, 64, 96, 9, dev)
    x[5, 3], x[70, 40], x[71, 90] = math.nan, math.inf, -math.inf
    y, kept = lb.linear_q8(x, w, b, 0.01)
    bad = torch.zeros(100, dtype=torch.bool, device=dev)
    bad[[5, 70, 71]] = True
    assert not torch.isfinite(y[bad]).any() and torch.isfinite(y[~bad]).all()
    assert torch.isnan(kept.dequantize()[bad]).all() and torch.isfinite(kept.dequantize()[~bad]).all()
    x2, w, b, dy = _rand(100, 64, 96, 10, dev)
    y2 = x2 @ w.t()
    yk = lb.q8_pack(y2)
    dy[y2 <= 0] = math.nan
    dx, dw, db = lb.linear_q8_backward(dy, w, lb.q8_pack(x2), yk, 0.0)
    assert torch.isfinite(dx).all() and torch.isfinite(dw).all() and torch.isfinite(db).all()
    x2[9, 40] = math.inf
    dy = torch.nan_to_num(dy)
    _, dw, _ = lb.linear_q8_backward(dy, w, lb.q8_pack(x2), yk, 0.0)
    live = (y2[9] > 0)
    assert torch.isnan(dw[live][:, 32:64]).all() and torch.isfinite(dw[:, :32]).all() and torch.isfinite(dw[:, 64:]).all()


@gpu
def test_linear_q8_range_ends(dev):
    """Factors at both ends of the float32 range: exact powers of two stay exact."""
    from apn_amd import lowbit as lb
    x = torch.zeros(3, 40, device=dev)
    x[0, 0], x[1, 1], x[2, 39] = 2.0 ** 120, 2.0 ** -100, -(2.0 ** -60)
    w = torch.zeros(33, 40, device=dev)
    w[:, 0], w[:, 1], w[:, 39] = 2.0 ** 7, 2.0 ** -20, 2.0 ** -40
    y, kept = lb.linear_q8(x, w)
    want = torch.tensor([2.0 ** 127, 2.0 ** -120, -(2.0 ** -100)], dtype=torch.float64).to(dev)
    assert torch.equal(y.double(), want[:, None].expand(3, 33))
    assert torch.equal(kept.dequantize().double(), y.double())


@gpu
def test_linear_q8_strides(dev):
    """Padded, offset, transposed and repeated operands equal their copies bit for bit."""
    from apn_amd import lowbit as lb
    g = torch.Generator(device=dev).manual_seed(1)
    buf = torch.randn(150, 200, device=dev, generator=g)
    wb = torch.randn(200, 130, device=dev, generator=g)
    for x, w in ((buf[:, :191], wb.t()[:, :191]), (buf[:, 3:67], wb[:70, 1:65]), (buf[1:, 1:2], wb[:, :1]),
                 (buf[:1].expand(33, 200), wb.t()), (buf.reshape(3, 50, 200), wb.t())):
        b = torch.randn(w.shape[0], device=dev, generator=g)
        y, k = lb.linear_q8(x, w, b, 0.1)
        y1, k1 = lb.linear_q8(x.reshape(-1, x.shape[-1]).clone(), w.contiguous().clone(), b, 0.1)
        assert torch.equal(y, y1) and torch.equal(k.codes, k1.codes) and torch.equal(k.scales, k1.scales)
        xk = lb.q8_pack(x)
        dyb = torch.randn(y.shape[0], y.shape[1] + 3, device=dev, generator=g)
        for dy in (dyb[:, :-3], dyb[:, 2:-1], dyb[:1, :-3].expand(y.shape)):
            got = lb.linear_q8_backward(dy, w, xk, k, 0.1)
            want = lb.linear_q8_backward(dy.clone(), w.contiguous().clone(), xk, k, 0.1)
            assert all(torch.equal(a, c) for a, c in zip(got, want))


@gpu
def test_linear_q8_no_rows(dev):
    from apn_amd import lowbit as lb
    w = torch.randn(7, 33, device=dev)
    y, k = lb.linear_q8(torch.empty(0, 33, device=dev), w, None, 0.0)
    assert y.shape == (0, 7) and k.shape == (0, 7)
    dx, dw, db = lb.linear_q8_backward(torch.empty(0, 7, device=dev), w, lb.q8_pack(torch.empty(0, 33, device=dev)), k, 0.0)
    assert dx.shape == (0, 33) and not dw.any() and dw.shape == (7, 33) and not db.any()


# --- the autograd stack ------------------------------------------------------------------------------

def _stack(dev, sizes, slopes, seed):
    torch.manual_seed(seed)
    mods = []
    for (i, o), s in zip(zip(sizes[:-1], sizes[1:]), slopes):
        mods.append(torch.nn.Linear(i, o))
        if s is not None:
            mods.append(torch.nn.ReLU() if s == 0 else torch.nn.LeakyReLU(s))
    return torch.nn.Sequential(*mods).to(dev)


def _chain_gradients(net_pairs, x, dy, kepts):
    """The chain's gradients in 64 bits with every saved row replaced by its checkpoint's value."""
    g = dy.double()
    out = []
    for (layer, slope), xin, y in zip(reversed(net_pairs), reversed(kepts[:-1]), reversed(kepts[1:])):
        if slope is not None:
            g = torch.where(y > 0, g, g * slope)
        out.append((g.t() @ ref_q8(xin)[2].to(g.device), g.sum(0)))
        g = g @ layer.weight.detach().double()
    return g, out[::-1]


@gpu
@autograd
def test_sequential_q8_gradients(dev):
    """linear.sequential(checkpoint="q8") under autograd: the output is that of the layers, and every
    gradient is the chain rule's on the checkpoints' values."""
    from apn_amd import linear as LIN, lowbit as lb
    net = _stack(dev, [191, 128, 96, 33], [0.01, 0.0, None], 2)
    g = torch.Generator(device=dev).manual_seed(4)
    buf = torch.randn(777, 192, device=dev, generator=g)
    x = buf[:, :191].requires_grad_(True)
    dy = torch.randn(777, 33, device=dev, generator=g)
    y = LIN.sequential(net, x, checkpoint="q8")
    y.backward(dy)
    pairs = LIN.layer_pairs(net)
    rows, h = [x.detach()], x.detach()
    for layer, slope in pairs:
        h = lb.linear_q8(h, layer.weight, layer.bias, slope)[0]
        rows.append(h)
    assert torch.equal(h, y)
    gx, gp = _chain_gradients(pairs, x, dy, rows)
    rel = lambda a, r: float((a.double() - r).norm() / r.norm())  # noqa: E731
    # three chained float32 products: 3 x the relative error of one, ~1e-6 for these widths
    assert rel(x.grad, gx) < 1e-5
    for (layer, _), (gw, gb) in zip(pairs, gp):
        assert rel(layer.weight.grad, gw) < 1e-5 and rel(layer.bias.grad, gb) < 1e-5


@gpu
@autograd
def test_sequential_q8_vs_differences(dev):
    """The gradient of a smooth stack (no activation: the forward is exact in the parameters) against
    central differences in 64 bits of the same loss with the rows as the checkpoints hold them."""
    from apn_amd import linear as LIN, lowbit as lb
    net = _stack(dev, [24, 16, 8], [None, None], 6)
    g = torch.Generator(device=dev).manual_seed(7)
    x0 = lb.q8_pack(torch.randn(40, 24, device=dev, generator=g)).dequantize()   # its own checkpoint
    x = x0.clone().requires_grad_(True)
    dy = torch.randn(40, 8, device=dev, generator=g)
    LIN.sequential(net, x, checkpoint="q8").backward(dy)
    w1, w2 = net[0].weight.detach().double(), net[1].weight.detach().double()

    def loss(w1_, x_):
        h = x_ @ w1_.t() + net[0].bias.detach().double()
        return ((h @ w2.t() + net[1].bias.detach().double()) * dy.double()).sum()

    eps = 1e-4
    for i, j in ((0, 0), (3, 7), (15, 23)):
        d = torch.zeros_like(w1)
        d[i, j] = eps
        fd = (loss(w1 + d, x0.double()) - loss(w1 - d, x0.double())) / (2 * eps)
        assert abs(float(net[0].weight.grad[i, j].double() - fd)) <= 1e-5 * float(dy.abs().sum())
        d = torch.zeros(40, 24, dtype=torch.float64, device=dev)
        d[i, j] = eps
        fd = (loss(w1, x0.double() + d) - loss(w1, x0.double() - d)) / (2 * eps)
        assert abs(float(x.grad[i, j].double() - fd)) <= 1e-5 * float(dy.abs().sum())


@gpu
@autograd
def test_sequential_q8_frozen_parts_and_columns(dev):
    """Frozen layers, an input without gradient, a shared layer used twice, a layer without bias, and
    the first layer's column map give the gradients of the plain stack to the checkpoints' accuracy
    (2^-7 of a block's largest magnitude per kept value) and None where none is wanted."""
    from apn_amd import linear as LIN
    g = torch.Generator(device=dev).manual_seed(8)
    x = torch.randn(500, 70, device=dev, generator=g)
    cols = torch.arange(64, device=dev) + 4
    net = _stack(dev, [64, 64, 64], [0.01, 0.01], 9)
    shared = torch.nn.Sequential(net[0], net[1], net[0], torch.nn.Linear(64, 5, bias=False).to(dev))
    frozen = _stack(dev, [64, 32, 32, 4], [0.0, 0.0, None], 10)
    frozen[2].requires_grad_(False)
    frozen[4].weight.requires_grad_(False)
    for m, want_x in ((net, True), (shared, True), (frozen, False)):
        grads = []
        for ck in (None, "q8"):
            m.zero_grad(set_to_none=True)
            xi = x.clone().requires_grad_(want_x)
            y = LIN.sequential(m, xi, col_pos=cols, checkpoint=ck)
            (y * y).sum().backward()
            grads.append([xi.grad] + [p.grad for p in m.parameters()])
        for a, b in zip(*grads):
            assert (a is None) == (b is None)
            if a is not None:
                assert float((a - b).norm() / a.norm()) < 2.0 ** -6
    with pytest.raises(RuntimeError, match="modified by an inplace"):   # a weight changed before its backward
        y = LIN.sequential(net, x[:, :64].clone().requires_grad_(True), checkpoint="q8")
        with torch.no_grad():
            net[2].weight.mul_(2.0)
        y.sum().backward()


@gpu
@autograd
def test_sequential_q8_keeps_less(dev):
    """Between forward and backward the stack holds at most 0.3 of the float32 rows' bytes."""
    from apn_amd import linear as LIN
    net = _stack(dev, [128] * 5, [0.01] * 4, 11)
    x = torch.randn(65536, 128, device=dev).requires_grad_(True)
    held = []
    for ck in (None, "q8"):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = LIN.sequential(net, x, checkpoint=ck)
        held.append(torch.cuda.memory_allocated() - before - y.numel() * 4)
        del y
    assert held[1] < 0.45 * held[0], held   # the plain stack's input and output are the caller's: 3 rows of 4 bytes


@gpu
@autograd
@pytest.mark.parametrize("S,C", [(1, 1), (3, 33), (1000, 128), (257, 200)])
def test_idw_sum_q8_backward(dev, S, C):
    from apn_amd import lowbit as lb
    from apn_amd.train import IdwSum, IdwSumQ8
    g = torch.Generator(device=dev).manual_seed(S + C)
    out = torch.randn(8 * S, C, device=dev, generator=g).requires_grad_(True)
    w = torch.rand(S, 8, device=dev, generator=g).requires_grad_(True)
    dh = torch.randn(S, C, device=dev, generator=g)
    kept = lb.q8_pack(out)
    h = IdwSumQ8.apply(w, out, kept)
    assert torch.equal(h, IdwSum.apply(w, out))
    h.backward(dh)
    v = ref_q8(out.detach())[2].to(dev).reshape(S, 8, C)
    prod = v * dh.double()[:, None]
    _within(w.grad, prod.sum(-1), (C + 16) * U * prod.abs().sum(-1))
    assert torch.equal(out.grad, (w.detach()[:, :, None] * dh[:, None]).reshape(8 * S, C))


# --- 4-bit products ----------------------------------------------------------------------------------

MX = [(1, 1, 1), (1, 256, 256), (1, 4096, 64), (3, 32, 33), (16, 96, 17), (33, 100, 65), (128, 128, 64),
      (130, 191, 128), (200, 1000, 129), (257, 2048, 300), (1000, 64, 31)]


@gpu
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,K,N", MX)
def test_mx4_linear_vs_float64(dev, M, K, N, out_dtype):
    """From float rows and from quantized ones, every output type and activation."""
    from apn_amd import lowbit as lb
    x, w, b, _ = _rand(M, N, K, M + K + N, dev)
    x *= torch.exp2(torch.randint(-6, 7, (M, 1), device=dev).float())
    wq = lb.mx4_quantize(w)
    xv, wv = ref_mx4(x)[2].to(dev), ref_mx4(w)[2].to(dev)
    pre = xv @ wv.t()
    S = xv.abs() @ wv.abs().t() + b.double().abs()
    for bias, slope in ((None, None), (b, 0.01), (b, 0.0)):
        y = lb.mx4_linear(x, wq, bias, slope, out_dtype)
        assert y.dtype == out_dtype
        ref = _act64(pre if bias is None else pre + b.double(), slope)
        half = 0.0 if out_dtype == torch.float32 else torch.finfo(out_dtype).eps / 2
        _within(y, ref, (K + 16) * U * S * (1 + half) + half * ref.abs() + (6e-8 if out_dtype == torch.float16 else 0))
    assert torch.equal(lb.mx4_linear(lb.mx4_quantize(x), wq, b, 0.01, out_dtype), lb.mx4_linear(x, wq, b, 0.01, out_dtype))
    xb = x.bfloat16()
    assert torch.equal(lb.mx4_linear(xb, wq, b, None, out_dtype), lb.mx4_linear(xb.float(), wq, b, None, out_dtype))


@gpu
@pytest.mark.parametrize("M,K,N", [(3500, 33, 3600), (3300, 100, 3800), (3500, 700, 3700), (3841, 1000, 3585),
                                   (2048, 4096, 1536), (33000, 96, 100), (1500, 520, 1600)])
def test_mx4_linear_many_tiles_vs_float64(dev, M, K, N):
    """Enough tiles for every tile shape, K with whole and partial steps, scale rows of whole and
    partial 16-byte pieces; padding bytes of the scales that are not zero are not read."""
    from apn_amd import lowbit as lb
    x, w, b, _ = _rand(M, N, K, M + K + N, dev)
    xq, wq = lb.mx4_quantize(x), lb.mx4_quantize(w)
    xv, wv = xq.dequantize().double(), wq.dequantize().double()   # (equal to the definition: above)
    ref = xv @ wv.t() + b.double()
    S = xv.abs() @ wv.abs().t() + b.double().abs()
    y = lb.mx4_linear(xq, wq, b)
    _within(y, ref, (K + 16) * U * S)
    nb = -(-K // BLOCK)
    for r in (xq, wq):
        r.scales[:, nb:] = 255
    assert torch.equal(lb.mx4_linear(xq, wq, b), y)
    assert torch.equal(lb.mx4_linear(xq, wq, b, 0.01, torch.bfloat16), _act64(y, 0.01).to(torch.bfloat16))


@gpu
def test_mx4_linear_non_finite_and_empty(dev):
    from apn_amd import lowbit as lb
    x, w, b, _ = _rand(70, 40, 96, 3, dev)
    x[4, 50], x[66, 0] = math.inf, math.nan
    y = lb.mx4_linear(x, lb.mx4_quantize(w), b)
    bad = torch.zeros(70, dtype=torch.bool, device=dev)
    bad[[4, 66]] = True
    assert torch.isnan(y[bad]).all() and torch.isfinite(y[~bad]).all()
    w[7, 3] = math.inf
    y = lb.mx4_linear(x[:4], lb.mx4_quantize(w), b)
    assert torch.isnan(y[:, 7]).all() and torch.isfinite(y[:, :7]).all() and torch.isfinite(y[:, 8:]).all()
    assert lb.mx4_linear(x[:0], lb.mx4_quantize(w), b).shape == (0, 40)
    zero = lb.mx4_linear(torch.zeros(5, 96, device=dev), lb.mx4_quantize(torch.zeros(40, 96, device=dev)), b)
    assert torch.equal(zero, b.expand(5, 40))


def _ref_chain(layers, x):
    h = x.double()
    for w, b, slope in layers:
        h = _act64(ref_mx4(h)[2].to(x.device) @ ref_mx4(w)[2].to(x.device).t() + b.double(), slope)
    return h


@gpu
@pytest.mark.parametrize("M,sizes", [(1, [33, 32]), (1, [17, 256, 64]), (100, [191, 128, 128, 128, 128]), (65, [64, 40, 200, 7]),
                                     (3000, [191, 128, 128]), (257, [300, 288, 128])])
def test_mx4_sequential_vs_float64(dev, M, sizes):
    """A stack with 4-bit rows in between. Where float32 and float64 sums fall on two sides of a
    rounding border of an inner row, that code differs by one step (a third of a value at most, of one
    of n inputs); such flips are at most a few in a million, so the 2-norm stays within 1e-3."""
    from apn_amd import lowbit as lb
    g = torch.Generator(device=dev).manual_seed(M)
    layers = []
    for i, (k, n) in enumerate(zip(sizes[:-1], sizes[1:])):
        layers.append((torch.randn(n, k, device=dev, generator=g) / k ** 0.5, torch.randn(n, device=dev, generator=g),
                       0.01 if i < len(sizes) - 2 else None))
    x = torch.randn(M, sizes[0], device=dev, generator=g)
    packed = [lb.MX4Layer(lb.mx4_quantize(w), b, s) for w, b, s in layers]
    y = lb.mx4_sequential(packed, x)
    ref = _ref_chain(layers, x)
    assert float((y.double() - ref).norm() / ref.norm()) < 1e-3
    yb = lb.mx4_sequential(packed, x, out_dtype=torch.bfloat16)
    assert torch.equal(yb, y.to(torch.bfloat16))
    # the same stack one layer at a time
    h = x
    for p in packed:
        h = lb.mx4_linear(h, p.weight, p.bias, p.slope)
    assert float((y - h).norm() / h.norm()) < 1e-3


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,sizes,slope", [(1, [1, 1], 0.0), (17, [31, 33, 5], 0.01), (5000, [192, 128, 128], 0.0),
                                           (333, [256, 256, 256, 256, 256], 0.01), (100, [129, 130, 1, 7], -0.5),
                                           (40, [8] * 9, None), (65, [191, 64, 255, 30], None)])
def test_mx4_stack_in_one_launch(dev, M, sizes, slope, dtype, out_dtype):
    """A stack that fits one launch (several layers, widths up to 256) equals the same layers one by one
    up to flips of inner codes (see above), for every type, padded rows and short blocks; a row that is
    not finite stays its own."""
    from apn_amd import lowbit as lb
    g = torch.Generator(device=dev).manual_seed(sum(sizes) + M)
    packed = [lb.MX4Layer(lb.mx4_quantize(torch.randn(n, k, device=dev, generator=g) / k ** 0.5),
                          torch.randn(n, device=dev, generator=g) if i != 1 else None, slope)
              for i, (k, n) in enumerate(zip(sizes[:-1], sizes[1:]))]
    x = torch.randn(M, sizes[0] + 3, device=dev, generator=g).to(dtype)[:, 1:sizes[0] + 1]
    y = lb.mx4_sequential(packed, x, out_dtype)
    h = x
    for p in packed[:-1]:
        h = lb.mx4_linear(h, p.weight, p.bias, p.slope)
    h = lb.mx4_linear(h, packed[-1].weight, packed[-1].bias, packed[-1].slope)
    # one flip in a few rows is a larger share of a small output: 1e-3 of many rows, 0.1 of few
    half = 0.0 if out_dtype == torch.float32 else torch.finfo(out_dtype).eps / 2
    assert y.dtype == out_dtype
    bound = (1e-3 if M * sizes[-1] > 1000 else 0.1) + half
    assert float((y.double() - h.double()).norm()) <= bound * float(h.double().norm())
    assert torch.equal(y, lb.mx4_sequential(packed, x.clone(), out_dtype))
    if M > 20:
        x = x.clone()
        x[3, 0], x[19, -1] = math.inf, math.nan
        bad = torch.zeros(M, dtype=torch.bool, device=dev)
        bad[[3, 19]] = True
        z = lb.mx4_sequential(packed, x, out_dtype)
        assert torch.isnan(z[bad]).all() and torch.equal(z[~bad], y[~bad])
    assert lb.mx4_sequential(packed, x[:0], out_dtype).shape == (0, sizes[-1])


# --- streams, graphs, the model ------------------------------------------------------------------------

def _functional_step(lb, x, w, b, dy, packed):
    y, k = lb.linear_q8(x, w, b, 0.01)
    grads = lb.linear_q8_backward(dy, w, lb.q8_pack(x), k, 0.01)
    square = lb.mx4_quantize(w[:, :1].expand(-1, w.shape[0]).contiguous())
    return (y, *grads, lb.mx4_linear(x, packed, b, 0.01), lb.mx4_linear(x[:3], packed, b, 0.01),
            lb.mx4_sequential([lb.MX4Layer(packed, b, 0.0), lb.MX4Layer(square, b)], x))


@gpu
def test_mx4_layer_is_frozen(dev):
    """A layer built from a module holds what the module held then: neither an in-place change of the
    module's parameters nor new storage for them reaches it."""
    from apn_amd import lowbit as lb
    from apn_amd.linear import layer_pairs
    torch.manual_seed(0)
    net = torch.nn.Sequential(torch.nn.Linear(33, 64), torch.nn.ReLU(), torch.nn.Linear(64, 20)).to(dev)
    x = torch.randn(50, 33, device=dev)
    layers = lb.mx4_layers(layer_pairs(net))
    y = lb.mx4_sequential(layers, x)
    with torch.no_grad():
        for p in net.parameters():
            p.fill_(math.nan)
            p.data = torch.full_like(p, 7.0)
    fill = [torch.full((64,), math.nan, device=dev) for _ in range(64)]   # takes freed storage, if any
    assert torch.equal(lb.mx4_sequential(layers, x), y) and len(fill) == 64


@gpu
def test_captured_and_replayed_beside_eager_work(dev):
    """Two captures of the functional forms share nothing: replayed in turn with eager calls and new
    inputs between them, every replay equals the eager result."""
    from apn_amd import lowbit as lb
    steps = []
    for seed, (M, K, N) in enumerate(((515, 191, 128), (4100, 96, 200))):
        x, w, b, dy = _rand(M, N, K, seed, dev)
        packed = lb.mx4_quantize(w)
        _functional_step(lb, x, w, b, dy, packed)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _functional_step(lb, x, w, b, dy, packed)
        steps.append((graph, x, w, b, dy, packed, out))
    for rep in range(4):
        for graph, x, w, b, dy, packed, out in steps:
            g = torch.Generator(device=dev).manual_seed(100 + rep)
            x.copy_(torch.randn(x.shape, device=dev, generator=g))
            dy.copy_(torch.randn(dy.shape, device=dev, generator=g))
            graph.replay()
            want = _functional_step(lb, x, w, b, dy, packed)
            torch.cuda.synchronize()
            for a, c in zip(out, want):
                assert torch.equal(a, c), rep


@gpu
def test_two_streams_at_once(dev):
    """The same calls on two streams at the same time give the results of one after the other."""
    from apn_amd import lowbit as lb
    args = []
    for seed in range(2):
        x, w, b, dy = _rand(20000, 128, 191, 20 + seed, dev)
        args.append((x, w, b, dy, lb.mx4_quantize(w)))
    want = [_functional_step(lb, *a) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(dev) for _ in args]
    got = []
    for _ in range(3):
        for s, a in zip(streams, args):
            with torch.cuda.stream(s):
                got.append(_functional_step(lb, *a))
    torch.cuda.synchronize()
    for i, r in enumerate(got):
        for a, c in zip(r, want[i % 2]):
            assert torch.equal(a, c)


@gpu
@autograd
def test_autograd_stack_refuses_capture(dev):
    from apn_amd import linear as LIN
    net = _stack(dev, [32, 32], [0.01], 1)
    x = torch.randn(64, 32, device=dev)
    LIN.sequential(net, x, checkpoint="q8").sum().backward()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    said = None
    with torch.cuda.graph(graph):
        z = x + 1.0
        try:
            LIN.sequential(net, z, checkpoint="q8")
        except RuntimeError as e:
            said = str(e)
    assert said is not None and "captured" in said


@gpu
@autograd
def test_autograd_stack_refuses_captured_backward(dev, monkeypatch):
    """The backward pass of an eager forward (the capture is pretended: a real one would end in it)."""
    from apn_amd import linear as LIN
    net = _stack(dev, [32, 32], [0.01], 1)
    y = LIN.sequential(net, torch.randn(64, 32, device=dev), checkpoint="q8").sum()
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="captured"):
        y.backward()
    monkeypatch.undo()
    assert all(p.grad is None for p in net.parameters())


@gpu
@autograd
def test_training_step_with_checkpoints_then_preview(dev):
    """The operators together as a user has them: a training step of the model with its rows kept in
    8 bits (the output is the plain step's to float32 rounding, the gradients the plain step's to
    the checkpoints' accuracy), then a frame of it with feat_net in 4 bits."""
    from apn_amd import harness, synthetic as S
    scene = S.make_scene("C1")
    model = harness.build_model(scene, dev)
    rk = scene.render_kwargs(dev)
    t = torch.tensor([scene.cfg.t], device=dev)
    with torch.no_grad():
        target = model(t + 0.1, render_kwargs=rk)["rgb_marched"].clone()
    runs = []
    for ck in (None, "q8"):
        model.activation_checkpoint = ck
        model.zero_grad(set_to_none=True)
        out = model(t, render_kwargs=rk)
        torch.nn.functional.mse_loss(out["rgb_marched"], target).backward()
        runs.append((out["rgb_marched"].detach(), {k: p.grad.clone() for k, p in model.named_parameters()
                                                   if p.grad is not None}))
    (a, ga), (b, gb) = runs
    assert float((a - b).abs().max()) < 1e-5      # two f32 sums of four layers of up to 191 terms
    assert set(ga) == set(gb) and any(k.startswith("feat_net") for k in ga)
    for k in ga:
        n = float(ga[k].norm())
        # every kept value is within 2^-7 of its block's largest, the errors of a sum's terms of either sign
        assert float((ga[k] - gb[k]).norm()) <= 0.03 * n + 1e-12, k
    model.activation_checkpoint = "q4"
    with pytest.raises(ValueError, match="activation_checkpoint"):
        model(t, render_kwargs=rk)
    model.activation_checkpoint = None
    with torch.no_grad():
        full = model(t, render_kwargs=rk)["rgb_marched"].clone()
        model.feat_format = "mx4"
        low = model(t, render_kwargs=rk)["rgb_marched"].clone()
        with pytest.raises(NotImplementedError):
            model.capture_frame(t, rk)
        model.feat_format = "mx3"
        with pytest.raises(ValueError, match="feat_format"):
            model(t, render_kwargs=rk)
        model.feat_format = None
        assert torch.equal(model(t, render_kwargs=rk)["rgb_marched"], full)
    assert torch.isfinite(low).all() and not torch.equal(low, full)
    # 4-bit rows and weights: relative error of a product about 0.1 per layer; colours are sigmoids in (0, 1)
    assert float((low - full).square().mean()) < 0.05 ** 2


# --- refusals (CPU) ------------------------------------------------------------------------------------

def test_refusals_cpu():
    from apn_amd import linear as LIN, lowbit as lb
    f = torch.float32
    x, w = torch.zeros(4, 33), torch.zeros(5, 33)
    for call in (lambda: lb.q8_pack(x), lambda: lb.mx4_quantize(x), lambda: lb.linear_q8(x, w),
                 lambda: lb.Q8Rows(torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 4, dtype=torch.uint8), 33),
                 lambda: lb.sequential_q8([(torch.nn.Linear(33, 5), None)], x)):
        with pytest.raises(RuntimeError, match="device"):
            call()
    u = lambda *s: torch.zeros(*s, dtype=torch.uint8)  # noqa: E731
    with pytest.raises(ValueError, match="codes"):
        lb.Q8Rows(u(4, 33), u(4, 4), 33)
    with pytest.raises(ValueError, match="codes"):
        lb.MX4Rows(u(4, 32), u(3, 4), 33)
    with pytest.raises(ValueError, match="codes"):
        lb.MX4Rows(u(4, 32), u(4, 2), 33)
    with pytest.raises(TypeError, match="uint8"):
        lb.Q8Rows(torch.zeros(4, 64), u(4, 4), 33)
    with pytest.raises(ValueError, match="columns"):
        lb.Q8Rows(u(4, 0), u(4, 0), 0)
    with pytest.raises(ValueError, match="contiguous"):
        lb.Q8Rows(u(64, 4).t(), u(4, 4), 33)
    with pytest.raises(TypeError, match="MX4Rows"):
        lb.mx4_linear(x, w)
    with pytest.raises(TypeError, match="MX4Rows"):
        lb.MX4Layer(w)
    with pytest.raises(ValueError, match="no layers"):
        lb.mx4_sequential([], x)
    with pytest.raises(ValueError, match="no layers"):
        lb.sequential_q8([], x)
    with pytest.raises(ValueError, match="checkpoint"):
        LIN.sequential(torch.nn.Linear(33, 5), x, checkpoint="q4")
    with pytest.raises(ValueError, match="Tanh"):
        LIN.layer_pairs(torch.nn.Sequential(torch.nn.Linear(3, 3), torch.nn.Tanh()))
    with pytest.raises(TypeError, match="Q8Rows"):
        lb.linear_q8_backward(x, w, x)
    # a CPU stack runs as torch does, with or without a checkpoint asked for
    net = torch.nn.Sequential(torch.nn.Linear(33, 5), torch.nn.LeakyReLU())
    assert torch.equal(LIN.sequential(net, x + 1, checkpoint="q8"), net(x + 1))
    assert f is torch.float32


def test_c_entries_refuse_without_gpu():
    """Invalid arguments come back as a status before anything is launched."""
    from apn_amd import _lib
    lib = _lib.load()
    p = 4096    # a pointer that is never followed
    assert lib.apn_q8_pack(p, 3, 4, 32, 32, p, p, None) == 1          # type
    assert lib.apn_q8_pack(p, 0, 4, 32, 31, p, p, None) == 1          # rows overlap
    assert lib.apn_q8_pack(p, 0, -1, 32, 32, p, p, None) == 1
    assert lib.apn_q8_pack(None, 0, 4, 32, 32, p, p, None) == 1
    assert lib.apn_q8_pack(p, 0, 4, 0, 32, p, p, None) == 1
    assert lib.apn_q8_pack(p, 0, 4, (1 << 20) + 1, 1 << 21, p, p, None) == 1
    assert lib.apn_q8_pack(p, 0, 4, 32, 32, p + 4, p, None) == 1      # codes off 16 bytes
    assert lib.apn_q8_pack(None, 0, 0, 32, 32, None, None, None) == 0   # no rows: nothing to do
    assert lib.apn_q8_unpack(p, p, 4, 32, p, 9, 32, None) == 1
    assert lib.apn_q8_linear_fwd(p, 16, p, 32, None, 4, 8, 32, 0, 0.0, p, 8, p, p, None) == 1
    assert lib.apn_q8_linear_fwd(p, 32, p, 32, None, 4, 8, 32, 0, 0.0, p, 7, p, p, None) == 1
    assert lib.apn_q8_linear_bwd_dx(p, 8, p + 8, 0.0, p, 32, 4, 8, 32, p, 32, None) == 1
    assert lib.apn_q8_linear_bwd_dw(p, 8, p, 0.0, None, None, 4, 8, 32, p, p, p, None) == 1
    assert lib.apn_q8_linear_bwd_dw(p, 8, p, 0.0, p, p, 4, 8, 32, p, p, None, None) == 1
    assert lib.apn_q8_linear_bwd_dw(p, 8, p, 0.0, p, p, 4, 8, 32, None, None, None, None) == 0   # nothing asked for
    for M in (0, 1, 63, 64, 65, 1000, 100000, 1 << 40):
        for N, K in ((1, 1), (128, 128), (128, 191), (1 << 20, 1), (513, 4096)):
            assert lib.apn_q8_linear_bwd_dw_workspace_bytes(M, N, K) >= N * (K + 1) * 4
    assert lib.apn_q8_idw_sum_bwd(4, 0, p, p, p, p, p, p, None) == 1
    assert lib.apn_mx4_quantize(p, 5, 4, 32, 32, p, p, None) == 1
    assert lib.apn_mx4_dequantize(p, p, 4, 32, p, 0, 16, None) == 1
    assert lib.apn_mx4_linear(p, p, p, p, None, 4, 0, 32, 0, 0.0, p, 0, 32, None) == 1
    assert lib.apn_mx4_linear(p, p, p + 1, p, None, 4, 8, 32, 0, 0.0, p, 0, 32, None) == 1
    assert lib.apn_mx4_linear(p, p, p, p, None, 4, 8, 32, 0, 0.0, p, 4, 32, None) == 1
    assert lib.apn_mx4_linear(p, p + 2, p, p, None, 4, 8, 32, 0, 0.0, p, 0, 32, None) == 1
    assert lib.apn_mx4_linear_few(p, 0, 32, p, p, None, 17, 8, 32, 0, 0.0, p, 0, 8, None) == 1
    assert lib.apn_mx4_linear_few(p, 0, 31, p, p, None, 4, 8, 32, 0, 0.0, p, 0, 8, None) == 1
    arg = _lib.MX4LayerArg
    two = (arg * 2)(arg(p, p, None, 64, 32, 0, 0.0), arg(p, p, None, 64, 64, 1, 0.5))
    assert lib.apn_mx4_network_lds_bytes(2, two) > 2 * 64 * 16
    assert lib.apn_mx4_network(p, 0, 31, 4, 2, two, p, 0, 64, None) == 1
    assert lib.apn_mx4_network(p, 0, 32, 4, 9, two, p, 0, 64, None) == 1
    two[1].K = 32
    assert lib.apn_mx4_network_lds_bytes(2, two) == 0 and lib.apn_mx4_network(p, 0, 32, 4, 2, two, p, 0, 64, None) == 1
    wide = (arg * 1)(arg(p, p, None, 257, 32, 0, 0.0))
    assert lib.apn_mx4_network_lds_bytes(1, wide) == 0 and lib.apn_mx4_network_lds_bytes(0, None) == 0


@gpu
def test_refusals_gpu(dev):
    from apn_amd import lowbit as lb
    x, w = torch.zeros(4, 33, device=dev), torch.zeros(5, 33, device=dev)
    with pytest.raises(TypeError, match="float"):
        lb.q8_pack(x.double())
    with pytest.raises(TypeError, match="float32 only"):
        lb.linear_q8(x.half(), w)
    with pytest.raises(ValueError, match="width"):
        lb.linear_q8(x, w[:, :32])
    with pytest.raises(ValueError, match="bias"):
        lb.linear_q8(x, w, torch.zeros(4, device=dev))
    with pytest.raises(TypeError, match="bias"):
        lb.linear_q8(x, w, torch.zeros(5, device=dev, dtype=torch.float64))
    with pytest.raises(ValueError, match="slope"):
        lb.linear_q8(x, w, None, math.nan)
    with pytest.raises(ValueError, match="at least one column"):
        lb.q8_pack(x[:, :0])
    with pytest.raises(ValueError, match="without rows"):
        lb.linear_q8(x, w[:0])
    with pytest.raises(RuntimeError, match="device"):
        lb.linear_q8(x, w.cpu())
    xk, yk = lb.q8_pack(x), lb.q8_pack(torch.zeros(4, 5, device=dev))
    dy = torch.zeros(4, 5, device=dev)
    with pytest.raises(ValueError, match="needs y_kept"):
        lb.linear_q8_backward(dy, w, xk, None, 0.0)
    with pytest.raises(ValueError, match="x_kept is"):
        lb.linear_q8_backward(dy, w, yk, yk, 0.0)
    with pytest.raises(ValueError, match="y_kept is"):
        lb.linear_q8_backward(dy, w, xk, xk, 0.0)
    with pytest.raises(ValueError, match="dw needs"):
        lb.linear_q8_backward(dy, w, None, yk, 0.0)
    with pytest.raises(ValueError, match="gradient width"):
        lb.linear_q8_backward(dy[:, :4], w, xk, yk, 0.0)
    with pytest.raises(ValueError, match="input width"):
        lb.mx4_linear(x[:, :32], lb.mx4_quantize(w))
    with pytest.raises(TypeError, match="float"):
        lb.mx4_linear(x, lb.mx4_quantize(w), out_dtype=torch.float64)
    with pytest.raises(TypeError, match="MX4Rows"):
        lb.mx4_linear(x, xk)
    layer = lb.MX4Layer(lb.mx4_quantize(w))
    with pytest.raises(ValueError, match="behind 5 outputs"):
        lb.mx4_sequential([layer, layer], x)
    with pytest.raises(ValueError, match="input width"):
        lb.mx4_sequential([layer], x[:, :32])
    with pytest.raises(TypeError, match="MX4Layer"):
        lb.mx4_sequential([w], x)
    with pytest.raises(TypeError, match="float"):
        lb.mx4_sequential([layer], x.double())


@gpu
@pytest.mark.parametrize("M,K,N", [(5, 2304, 40), (16, 4100, 70), (8, 130, 33), (9, 2080, 16), (1, 2049, 1)])
def test_mx4_linear_few_rows_vs_float64(dev, M, K, N):
    test_mx4_linear_vs_float64(dev, M, K, N, torch.float32)


@gpu
@pytest.mark.parametrize("slopes", [[2.0, None, 2.0], [0.01, 1.0, 1.5], [-2.0, 1.0, 0.0]])
def test_mx4_sequential_other_slopes(dev, slopes):
    """Slopes of 1, above and below: the stack equals its layers one after the other (the one-launch
    form takes slopes up to 1, others go layer by layer)."""
    from apn_amd import lowbit as lb
    g = torch.Generator(device=dev).manual_seed(7)
    layers, k = [], 100
    for n, slope in zip((64, 96, 33), slopes):
        w = torch.randint(-3, 4, (n, k), device=dev, generator=g).float()   # exact sums in any order
        layers.append(lb.MX4Layer(lb.mx4_quantize(w), torch.randint(-2, 3, (n,), device=dev, generator=g).float(), slope))
        k = n
    h = torch.randint(-6, 7, (130, 100), device=dev, generator=g).float()
    y = lb.mx4_sequential(layers, h)
    for layer in layers:
        h = lb.mx4_linear(h, layer.weight, layer.bias, layer.slope)
    assert torch.equal(y, h)


@gpu
def test_mx4_sequential_overflow(dev):
    """Sums that leave float32's range: ReLU takes -inf to 0 and +inf to NaN (its block's scale), the
    other rows are untouched."""
    from apn_amd import lowbit as lb
    big = torch.full((32, 32), 3e38, device=dev)
    x = torch.zeros(20, 32, device=dev)
    x[3], x[5] = -4.0, 4.0
    first = lb.MX4Layer(lb.mx4_quantize(big), None, 0.0)
    second = lb.MX4Layer(lb.mx4_quantize(torch.ones(16, 32, device=dev)), torch.ones(16, device=dev), None)
    y = lb.mx4_sequential([first, second], x)
    want = torch.ones(20, 16, device=dev)
    want[5] = math.nan
    assert torch.equal(torch.nan_to_num(y, nan=7.0), torch.nan_to_num(want, nan=7.0))


# --- the activation's side, from the output's sign ------------------------------------------------------

def test_negative_slopes_have_no_backward_cpu():
    """With a slope below 0 every output of the activation is positive, so the checkpoint's sign does
    not say on which side of the kink its input was: such a backward is refused, before anything runs."""
    from apn_amd import _lib, linear as LIN, lowbit as lb
    x, w = torch.zeros(4, 33), torch.zeros(5, 33)
    with pytest.raises(ValueError, match="slope"):
        lb.linear_q8_backward(torch.zeros(4, 5), w, None, None, -0.5, (True, False, False))
    with pytest.raises(ValueError, match="slope"):
        lb.sequential_q8([(torch.nn.Linear(33, 5), 0.01), (torch.nn.Linear(5, 5), -0.5)], x)
    # the CPU form of a stack runs torch's own modules, whatever its slopes
    net = torch.nn.Sequential(torch.nn.Linear(33, 5), torch.nn.LeakyReLU(-0.5))
    assert torch.equal(LIN.sequential(net, x + 1, checkpoint="q8"), net(x + 1))
    lib, p = _lib.load(), 4096    # a pointer that is never followed
    for slope in (-0.5, math.nan):
        assert lib.apn_q8_linear_bwd_dx(p, 8, p, slope, p, 32, 4, 8, 32, p, 32, None) == 1
        assert lib.apn_q8_linear_bwd_dw(p, 8, p, slope, p, p, 4, 8, 32, p, p, p, None) == 1


@gpu
@autograd
def test_negative_slopes_are_refused_under_autograd(dev):
    from apn_amd import linear as LIN, lowbit as lb
    x, w, b, dy = _rand(40, 24, 33, 12, dev)
    y, kept = lb.linear_q8(x, w, b, -0.5)
    with pytest.raises(ValueError, match="slope"):
        lb.linear_q8_backward(dy, w, lb.q8_pack(x), kept, -0.5)
    net = _stack(dev, [33, 24, 8], [-0.5, 0.01], 13)
    with pytest.raises(ValueError, match="slope"):
        LIN.sequential(net, x, checkpoint="q8")
    assert lb.linear_q8_backward(dy, w, lb.q8_pack(x), kept, -0.0)[0].shape == x.shape   # -0 is ReLU's


@gpu
@pytest.mark.parametrize("slope", [0.0, 1e-30, 0.01, 1.0, 2.0])
@pytest.mark.parametrize("M,K,N", [(3, 40, 33), (70, 70, 34), (500, 250, 66)])
def test_linear_q8_backward_gates_on_the_input_of_the_activation(dev, M, K, N, slope):
    """The derivative belongs to the activation's input v, not to its output: the gradients from
    ``linear_q8``'s own checkpoint against the formula in 64 bits with v from the same product without
    its activation (the same sums, so the same sign), an exact 0 among them."""
    from apn_amd import lowbit as lb
    x, w, b, dy = _rand(M, N, K, M + N, dev)
    x[1], b[::5] = 0.0, 0.0          # v = 0 in every fifth column of row 1
    v, _ = lb.linear_q8(x, w, b, None)
    _, kept = lb.linear_q8(x, w, b, slope)
    xk = lb.q8_pack(x)
    dx, dw, db = lb.linear_q8_backward(dy, w, xk, kept, slope)
    g = torch.where(v > 0, dy.double(), dy.double() * slope)
    xv = ref_q8(x)[2].to(dev)
    # (below 2^-110 a factor of a product is cut at bf16's smallest step: each is off by at most 2^-133)
    tiny = 2.0 ** -133
    _within(dx, g @ w.double(), _bound(N, g.abs() @ w.double().abs()) + tiny * N * float(w.abs().max()) + tiny)
    _within(dw, (xv.t() @ g).t(), _bound(M, (xv.abs().t() @ g.abs()).t()) + tiny * M * float(xv.abs().max()) + tiny)
    _within(db, g.sum(0), _bound(M, g.abs().sum(0)) + tiny * M)


# --- forms that no case above reaches, or does not show to be reached -----------------------------------

def _entries(monkeypatch, lb):
    """The list that the entry points launched from now on are put into."""
    seen = []
    launch = lb._launch
    monkeypatch.setattr(lb, "_launch", lambda dev, entry, *args: (seen.append(entry), launch(dev, entry, *args))[1])
    return seen


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,sizes,slope", [(1, [1, 1, 1], 0.0), (17, [31, 33, 5], 0.5), (5000, [192, 128, 128], 0.0),
                                           (333, [256, 256, 256, 256, 256], 0.5), (100, [129, 130, 1, 7], -0.5),
                                           (40, [8] * 9, None), (65, [191, 64, 255, 30], None), (1000, [256, 128, 128, 128, 128], 0.5)])
def test_mx4_stack_takes_one_launch(dev, monkeypatch, M, sizes, slope, dtype):
    """Stacks up to the one-launch form's limits run in it, and their results are those of the layers one
    by one, bit for bit, because every sum is exact in any order: inputs are whole numbers up to 6, a
    weight row has at most four entries of 1 or -1, biases are up to 2, and quantising (to at most 5/4 of
    the block's largest) keeps multiples of a power of two. A layer's sums are thus at most 5 times its
    inputs and 2: below 2^22 after 8 layers (slope None), below 2^13 and multiples of 2^-4 after 4 (slopes
    of 1/2)."""
    from apn_amd import lowbit as lb
    g = torch.Generator(device=dev).manual_seed(sum(sizes) + M)
    ints = lambda top, *shape: torch.randint(-top, top + 1, shape, device=dev, generator=g).float()  # noqa: E731

    def weight(n, k):
        w = torch.zeros(n, k, device=dev)
        return w.scatter_(1, torch.randint(0, k, (n, min(k, 4)), device=dev, generator=g), ints(1, n, min(k, 4)))
    packed = [lb.MX4Layer(lb.mx4_quantize(weight(n, k)), ints(2, n) if i != 1 else None, slope)
              for i, (k, n) in enumerate(zip(sizes[:-1], sizes[1:]))]
    x = ints(6, M, sizes[0] + 3).to(dtype)[:, 1:sizes[0] + 1]
    h = x
    for p in packed:
        h = lb.mx4_linear(h, p.weight, p.bias, p.slope)
    seen = _entries(monkeypatch, lb)
    for out_dtype in (torch.float32, torch.bfloat16, torch.float16):
        y = lb.mx4_sequential(packed, x, out_dtype)
        assert torch.equal(y, h.to(out_dtype))
    assert seen == ["apn_mx4_network"] * 3


@gpu
@pytest.mark.parametrize("x_dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,K,N", [(1, 8193, 17), (8, 16500, 33), (9, 33, 20), (12, 8200, 16), (16, 130, 40), (16, 20000, 31)])
def test_mx4_few_float_rows_entry_vs_float64(dev, M, K, N, x_dtype):
    """``apn_mx4_linear_few`` itself over all its row counts (the Python call takes it up to 8 rows), and
    over reductions of more than one panel of 8192 columns; more rows are refused."""
    from apn_amd import _lib, lowbit as lb
    x, w, b, _ = _rand(M, N, K, M + K + N, dev)
    x = x.to(x_dtype)
    wq = lb.mx4_quantize(w)
    out = torch.full((M + 1, N + 2), 7.0, device=dev)
    lb._launch(dev.index or 0, "apn_mx4_linear_few", x.data_ptr(), lb._TYPES[x_dtype], K, *wq._at, b.data_ptr(), M, N, K,
               1, 0.01, out.data_ptr(), 0, N + 2)
    xv, wv = ref_mx4(x.float())[2].to(dev), ref_mx4(w)[2].to(dev)
    S = xv.abs() @ wv.abs().t() + b.double().abs()
    _within(out[:M, :N], _act64(xv @ wv.t() + b.double(), 0.01), (K + 16) * U * S)
    assert (out[M] == 7.0).all() and (out[:, N:] == 7.0).all()      # nothing behind the rows and columns
    with pytest.raises(_lib.APNError):
        lb._launch(dev.index or 0, "apn_mx4_linear_few", x.data_ptr(), 0, K, *wq._at, None, 17, N, K, 0, 0.0,
                   out.data_ptr(), 0, N + 2)


@gpu
@pytest.mark.parametrize("M,K,N", [(1, 8193, 40), (16, 16500, 33)])
def test_mx4_few_coded_rows_of_several_panels(dev, M, K, N):
    from apn_amd import lowbit as lb
    x, w, b, _ = _rand(M, N, K, M + K + N, dev)
    xq, wq = lb.mx4_quantize(x), lb.mx4_quantize(w)
    xv, wv = ref_mx4(x)[2].to(dev), ref_mx4(w)[2].to(dev)
    _within(lb.mx4_linear(xq, wq, b), xv @ wv.t() + b.double(), (K + 16) * U * (xv.abs() @ wv.abs().t() + b.double().abs()))


@gpu
@pytest.mark.parametrize("slope", [None, 0.0, 0.01])
@pytest.mark.parametrize("M,K,N", [(49200, 100, 150), (49200, 150, 100), (49155, 191, 192), (49200, 256, 128)])
def test_linear_q8_many_rows_every_form(dev, M, K, N, slope):
    """Row counts past the fine column split, so that each wide form of the rows kernels runs (reductions
    up to 128 and 192 columns and above, outputs up to 128 and 192), forward and dX with and without
    signs. A factor whose parts were cut or kept wrong is off by 2^-8 of itself."""
    test_linear_q8_vs_float64(dev, M, K, N, slope)
    from apn_amd import lowbit as lb
    _, w, _, dy = _rand(M, N, K, 3, dev)
    y = torch.randn(M, N, device=dev, generator=torch.Generator(device=dev).manual_seed(4))
    dx = lb.linear_q8_backward(dy, w, None, lb.q8_pack(y), slope, (True, False, False))[0]
    g = dy.double() if slope is None else torch.where(y > 0, dy.double(), dy.double() * slope)
    _within(dx, g @ w.double(), _bound(N, g.abs() @ w.double().abs()))


@gpu
@autograd
def test_pose_embedding_scene_with_checkpoints_then_preview(dev, monkeypatch):
    """A model with a pose embedding, whose first feat_net layer is 256 columns wide (the general rows
    kernel, the wide form of the one-launch stack): a training step with 8-bit checkpoints against the
    plain step, then a frame with feat_net in 4 bits, each through the operators. A kept value is within
    2^-7 of its block's largest magnitude, about 3 of the block's root mean square: 0.03 of a gradient
    whose terms do not cancel (feat_net's own), several times that of those reached through the blend
    weights alone, where they partly do."""
    from apn_amd import harness, lowbit as lb, synthetic as S
    scene = S.make_scene("G2")
    model = harness.build_model(scene, dev)
    rk = scene.render_kwargs(dev)
    t = torch.tensor([scene.cfg.t], device=dev)
    with torch.no_grad():
        target = model(t + 0.1, render_kwargs=rk)["rgb_marched"].clone()
    seen = _entries(monkeypatch, lb)
    runs = []
    for ck in (None, "q8"):
        model.activation_checkpoint = ck
        model.zero_grad(set_to_none=True)
        out = model(t, render_kwargs=rk)
        torch.nn.functional.mse_loss(out["rgb_marched"], target).backward()
        runs.append((out["rgb_marched"].detach(), {k: p.grad.clone() for k, p in model.named_parameters()
                                                   if p.grad is not None}))
        assert bool(seen) == (ck == "q8")
    assert {"apn_q8_pack", "apn_q8_linear_fwd", "apn_q8_linear_bwd_dw", "apn_q8_linear_bwd_dx"} == set(seen)
    assert model.feat_net[0].weight.shape[1] + 1 == 256     # and one column of padding behind the 63 of the position
    (a, ga), (b, gb) = runs
    assert float((a - b).abs().max()) < 1e-5
    assert set(ga) == set(gb) and any(k.startswith("pose_embedding_net") for k in ga)
    for k in ga:
        bound = 0.03 if k.startswith("feat_net") else 0.1
        assert float((ga[k] - gb[k]).norm()) <= bound * float(ga[k].norm()) + 1e-12, k
    model.activation_checkpoint = None
    del seen[:]
    with torch.no_grad():
        full = model(t, render_kwargs=rk)["rgb_marched"].clone()
        model.feat_format = "mx4"
        low = model(t, render_kwargs=rk)["rgb_marched"].clone()
    assert set(seen) == {"apn_mx4_quantize", "apn_mx4_network"}
    assert torch.isfinite(low).all() and not torch.equal(low, full)
    assert float((low - full).square().mean()) < 0.05 ** 2
