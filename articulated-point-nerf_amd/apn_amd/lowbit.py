"""Narrow block formats for the Linear layers (apn_q8.hip, apn_mx4.hip).

* q8: the 8-bit activation checkpoint. A training step of the neighbour MLP keeps every layer's
  rows (8 per kept sample) for its backward pass; ``linear_q8`` writes a layer's f32 output and its
  8-bit checkpoint in one pass, ``linear_q8_backward`` computes all three gradients from the
  checkpoints, and ``sequential_q8`` is the autograd form for a stack of layers
  (``linear.sequential(net, x, checkpoint="q8")``; ``TemporalPoints.activation_checkpoint``).
  A kept row takes 33/128 of its f32 bytes.
* mx4: microscaled 4-bit rows (E2M1 elements, one power-of-two scale per 32). ``mx4_linear`` is a
  Linear layer with both operands in 4 bits, ``mx4_sequential`` a stack of them with the rows
  between the layers in 4 bits (``TemporalPoints.feat_format``: preview renders).

Both formats store a row of K values in blocks of 32 consecutive columns (include/apn_hip.h has the
layout). A block that holds an infinity or NaN reads back as NaN, whole; an infinite operand of
``linear_q8`` makes the results it reaches infinite or NaN.

Device tensors only. Rows are the last dimension; leading dimensions are flattened. Every call runs
on the current stream of its tensors' device and allocates only through torch, so the functional
forms (not the autograd one) can be captured into a graph. The functional forms are outside
autograd: their results carry no gradient.
"""
from __future__ import annotations

import math

import torch

from . import _lib as L

__all__ = ["Q8Rows", "q8_pack", "linear_q8", "linear_q8_backward", "sequential_q8", "MX4Rows", "mx4_quantize",
           "mx4_linear", "MX4Layer", "mx4_layers", "mx4_sequential"]

BLOCK = 32
MAX_COLS = 1 << 20
MAX_LD = 1 << 24     # rows further apart are copied
FEW_ROWS = 8         # mx4_linear of so many float rows quantizes them inside the product (8 x 4096 x 4096:
                     # 10.5 us, in two launches 8.7 + 3; 16 rows 14.5 and 9.9 + 3)
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _blocks(k: int) -> int:
    return -(-k // BLOCK)


def _scale_bytes(k: int) -> int:
    return -(-_blocks(k) // 4) * 4


def _type(dtype, what):
    t = _TYPES.get(dtype)
    if t is None:
        raise TypeError(f"{what}: float32, bfloat16 or float16, got {dtype}")
    return t


def _device(what, first, *others):
    """The index of the one device that all tensors (None: left out) are on."""
    dev = first.get_device()
    same = dev >= 0
    for t in others:
        if t is not None and t.get_device() != dev:
            same = False
    if not same:
        L.require_cuda(first, *others, what=what)
        devs = {str(t.device) for t in (first, *others) if t is not None}
        raise RuntimeError(f"{what}: tensors on different devices: {', '.join(sorted(devs))}")
    return dev


def _launch(dev, entry, *args):
    """``entry(*args, stream)`` on device ``dev`` and its current stream. The smallest calls cost
    what their host side costs, so addresses go in as plain integers, the stream as its raw handle,
    and the device is switched only if it is not the current one."""
    fn = getattr(L.load(), entry)
    if dev == torch.cuda.current_device():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev))
    if rc != 0:
        raise L.APNError(f"{entry} failed: {L._STATUS.get(rc, rc)}")


def _addr(t):
    return None if t is None else t.data_ptr()


def _rows(x, what):
    """x [..., K] as a 2-D tensor with unit column stride and rows that do not overlap, M, K and the
    row stride."""
    shape = x.shape
    if not shape or shape[-1] == 0:
        raise ValueError(f"{what}: expected rows of at least one column, got shape {tuple(shape)}")
    K = shape[-1]
    if K > MAX_COLS:
        raise ValueError(f"{what}: at most {MAX_COLS} columns, got {K}")
    if len(shape) != 2:
        x = x.detach().reshape(-1, K)
    M, (ld, unit) = x.shape[0], x.stride()
    if (unit != 1 and K > 1) or (M > 1 and (ld < K or ld >= MAX_LD)):
        return x.detach().contiguous(), M, K, K
    return x, M, K, ld if M > 1 else K


def _weight_rows(w, K, what):
    if w.dim() != 2 or w.shape[1] != K:
        raise ValueError(f"{what}: input width {K} vs weight {tuple(w.shape)}")
    if w.shape[0] == 0:
        raise ValueError(f"{what}: weight without rows {tuple(w.shape)}")
    return _rows(w, what)


def _bias(b, N, what):
    if b is None:
        return None
    if b.dim() != 1 or b.shape[0] != N:
        raise ValueError(f"{what}: bias {tuple(b.shape)} for {N} outputs")
    if b.dtype != torch.float32:
        raise TypeError(f"{what}: float32 bias, got {b.dtype}")
    return b if b.is_contiguous() else b.detach().contiguous()


def _act(slope, what):
    if slope is None:
        return 0, 0.0
    slope = float(slope)
    if not -math.inf < slope < math.inf:
        raise ValueError(f"{what}: slope must be finite, got {slope}")
    return 1, slope


def _act_backward(slope, what):
    """The slope of an activation whose derivative is taken from the sign of its output. Below 0 an
    output is never negative: its sign does not tell the two sides apart."""
    act, sl = _act(slope, what)
    if act and sl < 0.0:
        raise ValueError(f"{what}: no backward pass through a negative slope ({sl}): the kept sign is the output's")
    return sl


class _BlockRows:
    """Codes and scales of [rows, cols] values; ``codes`` uint8 [rows, _BYTES ceil(cols / 32)],
    ``scales`` uint8 [rows, 4 ceil(ceil(cols / 32) / 4)], both contiguous; codes behind column cols
    are zeros (q8: 0x80)."""

    _BYTES = 0

    def __init__(self, codes, scales, cols):
        cols = int(cols)
        what = type(self).__name__
        if not 1 <= cols <= MAX_COLS:
            raise ValueError(f"{what}: 1 to {MAX_COLS} columns, got {cols}")
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise TypeError(f"{what}: uint8 codes and scales, got {codes.dtype} and {scales.dtype}")
        want = (self._BYTES * _blocks(cols), _scale_bytes(cols))
        if codes.dim() != 2 or scales.dim() != 2 or codes.shape[0] != scales.shape[0] or \
                (codes.shape[1], scales.shape[1]) != want:
            raise ValueError(f"{what}: codes [M, {want[0]}] and scales [M, {want[1]}] for {cols} columns, got "
                             f"{tuple(codes.shape)} and {tuple(scales.shape)}")
        if not (codes.is_contiguous() and scales.is_contiguous()) or codes.data_ptr() % 16 or scales.data_ptr() % 4:
            raise ValueError(f"{what}: contiguous codes (16-byte aligned) and scales (4-byte aligned)")
        _device(what, codes, scales)
        self._buf, self._codes, self._scales = None, codes, scales
        self.rows, self.cols, self.device = codes.shape[0], cols, codes.device

    @classmethod
    def _empty(cls, rows, cols, device):
        """Rows for a kernel to fill: one allocation, their layout needs no check."""
        self = cls.__new__(cls)
        n = rows * cls._BYTES * _blocks(cols)
        self._buf = torch.empty(n + rows * _scale_bytes(cols), dtype=torch.uint8, device=device)
        self._codes = self._scales = None
        self.rows, self.cols, self.device = rows, cols, device
        return self

    @property
    def _at(self):
        """The addresses of codes and scales."""
        if self._buf is None:
            return self._codes.data_ptr(), self._scales.data_ptr()
        p = self._buf.data_ptr()
        return p, p + self.rows * self._BYTES * _blocks(self.cols)

    @property
    def codes(self) -> torch.Tensor:
        if self._codes is None:
            w = self._BYTES * _blocks(self.cols)
            self._codes = self._buf[:self.rows * w].view(self.rows, w)
        return self._codes

    @property
    def scales(self) -> torch.Tensor:
        if self._scales is None:
            w = _scale_bytes(self.cols)
            self._scales = self._buf[self._buf.numel() - self.rows * w:].view(self.rows, w)
        return self._scales

    @property
    def shape(self):
        return self.rows, self.cols

    @property
    def nbytes(self):
        return self.rows * (self._BYTES * _blocks(self.cols) + _scale_bytes(self.cols))

    def _index(self, what, dev):
        """Checks that these rows are on device index ``dev``."""
        if self.device.index != dev:
            raise RuntimeError(f"{what}: tensors on different devices: {self.device} and cuda:{dev}")

    def _read(self, entry, dtype):
        t = _type(dtype, f"{type(self).__name__}.dequantize")
        out = torch.empty((self.rows, self.cols), dtype=dtype, device=self.device)
        _launch(out.get_device(), entry, *self._at, self.rows, self.cols, out.data_ptr(), t, self.cols)
        return out


class Q8Rows(_BlockRows):
    """An 8-bit checkpoint of [rows, cols] values (``q8_pack``, ``linear_q8``)."""

    _BYTES = 32

    def dequantize(self, dtype=torch.float32) -> torch.Tensor:
        """The values the codes stand for, [rows, cols] (exact in float32 and bfloat16)."""
        return self._read("apn_q8_unpack", dtype)


class MX4Rows(_BlockRows):
    """Microscaled 4-bit rows (``mx4_quantize``)."""

    _BYTES = 16

    def dequantize(self, dtype=torch.float32) -> torch.Tensor:
        """The values the codes stand for, [rows, cols] (exact in float32 and bfloat16)."""
        return self._read("apn_mx4_dequantize", dtype)


def _pack(cls, entry, x, what):
    t = _type(x.dtype, what)
    x, M, K, ld = _rows(x, what)
    dev = _device(what, x)
    out = cls._empty(M, K, x.device)
    _launch(dev, entry, x.data_ptr(), t, M, K, ld, *out._at)
    return out


def q8_pack(x: torch.Tensor) -> Q8Rows:
    """The 8-bit checkpoint of x [..., K] (float32, bfloat16 or float16). Off by at most 2^-7 of the
    largest magnitude of the value's block."""
    return _pack(Q8Rows, "apn_q8_pack", x, "q8_pack")


def linear_q8(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, slope: float | None = None):
    """(y, kept): y [M, N] = act(x weight^T + bias) in float32 and its 8-bit checkpoint, in one pass.
    x [..., K] and weight [N, K] float32; ``slope``: None (no activation), 0 (ReLU) or the LeakyReLU
    negative slope (a slope below 0 has no backward pass: ``linear_q8_backward``). The products are
    f32-accurate."""
    what = "linear_q8"
    if x.dtype != torch.float32 or weight.dtype != torch.float32:
        raise TypeError(f"{what}: float32 only, got {x.dtype} and {weight.dtype}")
    x, M, K, ldx = _rows(x, what)
    w, N, _, ldw = _weight_rows(weight, K, what)
    b = _bias(bias, N, what)
    act, sl = _act(slope, what)
    dev = _device(what, x, w, b)
    y = torch.empty((M, N), dtype=torch.float32, device=x.device)
    kept = Q8Rows._empty(M, N, x.device)
    _launch(dev, "apn_q8_linear_fwd", x.data_ptr(), ldx, w.data_ptr(), ldw, _addr(b), M, N, K, act, sl, y.data_ptr(), N,
            *kept._at)
    return y, kept


def linear_q8_backward(dy: torch.Tensor, weight: torch.Tensor, x_kept: Q8Rows | None, y_kept: Q8Rows | None = None,
                       slope: float | None = None, need=(True, True, True)):
    """(dx, dw, db) of ``linear_q8`` from the checkpoints of its input and (with an activation) its
    output: g = dy * (y > 0 ? 1 : slope), dx = g weight, dw = g^T x', db = sum g, with x' the
    values of ``x_kept``. ``need``: which of the three are computed (None for the others; x_kept
    may be None without dw). A gradient masked by slope 0 is 0 whatever dy holds there. Sums over
    the rows are taken in a fixed order. ``slope`` is at least 0 (else ValueError): the derivative comes
    from the sign bit of y's codes, which is that of the activation's input only then."""
    what = "linear_q8_backward"
    want_x, want_w, want_b = need
    for kept, name in ((x_kept, "x_kept"), (y_kept, "y_kept")):
        if kept is not None and not isinstance(kept, Q8Rows):
            raise TypeError(f"{what}: {name} must be Q8Rows, got {type(kept).__name__}")
    if dy.dtype != torch.float32 or weight.dtype != torch.float32:
        raise TypeError(f"{what}: float32 only, got {dy.dtype} and {weight.dtype}")
    dy, M, N, ld_dy = _rows(dy, what)
    if weight.dim() != 2 or weight.shape[0] != N:
        raise ValueError(f"{what}: gradient width {N} vs weight {tuple(weight.shape)}")
    w, _, K, ldw = _rows(weight, what)
    if want_w and x_kept is None:
        raise ValueError(f"{what}: dw needs x_kept")
    if x_kept is not None and x_kept.shape != (M, K):
        raise ValueError(f"{what}: x_kept is {x_kept.shape}, expected {(M, K)}")
    if y_kept is not None and y_kept.shape != (M, N):
        raise ValueError(f"{what}: y_kept is {y_kept.shape}, expected {(M, N)}")
    sl = _act_backward(slope, what)
    if slope is not None and y_kept is None:
        raise ValueError(f"{what}: an activation needs y_kept")
    dev = _device(what, dy, w)
    for kept in (x_kept, y_kept):
        if kept is not None:
            kept._index(what, dev)
    mask = y_kept._at[0] if slope is not None else None
    xc, xs = x_kept._at if want_w else (None, None)
    empty = lambda *shape: torch.empty(shape, dtype=torch.float32, device=dy.device)  # noqa: E731
    dx = dw = db = None
    # (dx last: dy is then in the 256 MB cache for it, and dx for the layer below: 99 -> 96 us, 203008 x 128 x 128)
    if want_w or want_b:
        dw = empty(N, K) if want_w else None
        db = empty(N) if want_b else None
        ws = empty(max(int(L.load().apn_q8_linear_bwd_dw_workspace_bytes(M, N, K)) // 4, 1))
        _launch(dev, "apn_q8_linear_bwd_dw", dy.data_ptr(), ld_dy, mask, sl, xc, xs, M, N, K,
                _addr(dw), _addr(db), ws.data_ptr())
    if want_x:
        Kp = -(-K // 4) * 4   # rows of whole 16-byte pieces, as linear's: odd rows written 1.5 x as slowly
        dx = empty(M, Kp)
        _launch(dev, "apn_q8_linear_bwd_dx", dy.data_ptr(), ld_dy, mask, sl, w.data_ptr(), ldw, M, N, K,
                dx.data_ptr(), Kp)
        if Kp != K:
            dx = dx[:, :K]
    return dx, dw, db


def _not_captured(what):
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{what}: autograd steps cannot be captured; capture linear_q8 / linear_q8_backward")


class _Q8Stack(torch.autograd.Function):
    """A stack of Linear layers: f32 forward, everything the backward needs kept in 8 bits (the
    stack's input and each layer's output, once)."""

    @staticmethod
    def forward(ctx, x, slopes, col_pos, holder, *params):
        weights, biases = params[0::2], params[1::2]
        lead = x.shape[:-1]
        h = x.reshape(-1, x.shape[-1])
        x0 = q8_pack(h) if weights[0].requires_grad else None
        ws, kept = [], []
        for i, (w, b, slope) in enumerate(zip(weights, biases, slopes)):
            w = w.detach()
            if i == 0 and col_pos is not None:   # x holds weight column j at column col_pos[j]
                wide = torch.zeros(w.shape[0], -(-h.shape[1] // 4) * 4, device=w.device, dtype=w.dtype)
                wide[:, col_pos] = w
                w = wide[:, :h.shape[1]]
            h, k = linear_q8(h, w, b, slope)
            ws.append(w)
            kept.append(k)
        ctx.slopes, ctx.col_pos, ctx.in_shape, ctx.cols = slopes, col_pos, x.shape, [k.cols for k in kept]
        flat = [t for k in kept for t in (k.codes, k.scales)]
        ctx.save_for_backward(*(p for p in weights), *ws, *(() if x0 is None else (x0.codes, x0.scales)), *flat)
        ctx.has_x0 = x0 is not None
        if holder is not None:
            holder.append(kept[-1])
        return h.reshape(*lead, h.shape[-1])

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        _not_captured("sequential_q8")
        n = len(ctx.slopes)
        saved = ctx.saved_tensors
        ws, rest = saved[n:2 * n], saved[2 * n:]
        x0 = None
        if ctx.has_x0:
            x0, rest = Q8Rows(rest[0], rest[1], ctx.in_shape[-1]), rest[2:]
        kept = [Q8Rows(rest[2 * i], rest[2 * i + 1], ctx.cols[i]) for i in range(n)]
        need = ctx.needs_input_grad
        grads = [None] * (2 * n)
        g = dy.reshape(-1, dy.shape[-1])
        dx = None
        for i in reversed(range(n)):
            below = need[0] if i == 0 else need[0] or any(need[4:4 + 2 * i])
            nw, nb = need[4 + 2 * i], need[5 + 2 * i]
            dx, dw, db = linear_q8_backward(g, ws[i], x0 if i == 0 else kept[i - 1], kept[i], ctx.slopes[i],
                                            (below, nw, nb))
            if i == 0 and ctx.col_pos is not None and dw is not None:
                dw = dw[:, ctx.col_pos]
            grads[2 * i], grads[2 * i + 1] = dw, db
            if not below:
                break
            g = dx
        return (dx.reshape(ctx.in_shape) if need[0] else None, None, None, None, *grads)


def sequential_q8(layers, x: torch.Tensor, col_pos=None, keep_output=False):
    """A stack of (torch.nn.Linear, slope) pairs under autograd with 8-bit activation checkpoints:
    between forward and backward no float row of the stack is kept, only the 8-bit checkpoint of x
    and of each layer's output. ``col_pos``: linear.linear's. With ``keep_output`` returns
    (y, Q8Rows of y). Slopes are at least 0 (linear_q8_backward).

    Not under graph capture: a captured backward reaches the parameters' gradient accumulators, and
    one that an eager step created earlier on another stream ends the capture and with it the
    process; capture linear_q8 / linear_q8_backward instead."""
    what = "sequential_q8"
    layers = list(layers)
    if not layers:
        raise ValueError(f"{what}: no layers")
    for _, slope in layers:
        _act_backward(slope, what)
    L.require_cuda(x, what=what)
    _not_captured(what)
    params = [p for layer, _ in layers for p in (layer.weight, layer.bias)]
    holder = [] if keep_output else None
    y = _Q8Stack.apply(x, tuple(s for _, s in layers), col_pos, holder, *params)
    return (y, holder[0]) if keep_output else y


# --- 4-bit rows -----------------------------------------------------------------------------------

def mx4_quantize(x: torch.Tensor) -> MX4Rows:
    """x [..., K] (float32, bfloat16 or float16) as microscaled 4-bit rows."""
    return _pack(MX4Rows, "apn_mx4_quantize", x, "mx4_quantize")


def mx4_linear(x, weight: MX4Rows, bias: torch.Tensor | None = None, slope: float | None = None,
               out_dtype=torch.float32) -> torch.Tensor:
    """act(mx4(x) weight^T + bias) as [M, N] of ``out_dtype`` (float32, bfloat16, float16): exact
    4-bit products, float32 sums. x: MX4Rows, or a float tensor [..., K] that is quantized first."""
    what = "mx4_linear"
    if not isinstance(weight, MX4Rows):
        raise TypeError(f"{what}: weight must be MX4Rows, got {type(weight).__name__}")
    t = _type(out_dtype, what)
    N, K = weight.rows, weight.cols
    own = isinstance(x, MX4Rows)
    width = x.cols if own else x.shape[-1] if x.dim() else 0
    if width != K:
        raise ValueError(f"{what}: input width {width} vs weight {weight.shape}")
    if N == 0:
        raise ValueError(f"{what}: weight without rows {weight.shape}")
    b = _bias(bias, N, what)
    act, sl = _act(slope, what)
    if not own:
        xt = _type(x.dtype, what)
        rows, M, _, ldx = _rows(x, what)
        dev = _device(what, rows)
        weight._index(what, dev)
        if b is not None:
            _device(what, rows, b)
        if M <= FEW_ROWS:   # quantized on the way
            out = torch.empty((M, N), dtype=out_dtype, device=weight.device)
            _launch(dev, "apn_mx4_linear_few", rows.data_ptr(), xt, ldx, *weight._at, _addr(b), M, N, K, act, sl,
                    out.data_ptr(), t, N)
            return out
        x = mx4_quantize(rows)
    else:
        dev = x.device.index
        weight._index(what, dev)
        if b is not None and b.get_device() != dev:
            _device(what, x.codes, b)
    M = x.rows
    out = torch.empty((M, N), dtype=out_dtype, device=weight.device)
    _launch(dev, "apn_mx4_linear", *x._at, *weight._at, _addr(b), M, N, K, act, sl, out.data_ptr(), t, N)
    return out


class MX4Layer:
    """A frozen Linear layer: 4-bit weight rows, float32 bias, activation slope (None: none)."""

    def __init__(self, weight: MX4Rows, bias: torch.Tensor | None = None, slope: float | None = None):
        if not isinstance(weight, MX4Rows):
            raise TypeError(f"MX4Layer: weight must be MX4Rows, got {type(weight).__name__}")
        if bias is not None:
            _device("MX4Layer", weight.codes, bias)
        bias = _bias(bias, weight.shape[0], "MX4Layer")
        self.weight, self.slope = weight, slope
        self.bias = None if bias is None else bias.detach().clone()   # (a parameter's storage may be replaced)
        self._act = _act(slope, "MX4Layer")

    def _arg(self):
        return L.MX4LayerArg(*self.weight._at, _addr(self.bias), *self.weight.shape, *self._act)


def mx4_layers(layers, col_pos=None, width=None):
    """(torch.nn.Linear, slope) pairs as MX4Layers, their weights quantized once. ``col_pos``
    (int64 [in_features]) with ``width``: the stack's input rows are ``width`` wide and hold input j
    at column col_pos[j] (linear.linear's)."""
    out = []
    for i, (layer, slope) in enumerate(layers):
        w = layer.weight.detach()
        if i == 0 and col_pos is not None:
            wide = torch.zeros(w.shape[0], int(width), device=w.device, dtype=w.dtype)
            wide[:, col_pos] = w
            w = wide
        out.append(MX4Layer(mx4_quantize(w), layer.bias, slope))
    return out


def mx4_sequential(layers, x: torch.Tensor, out_dtype=torch.float32) -> torch.Tensor:
    """A stack of MX4Layers on x [..., K] (float32, bfloat16, float16); the rows between the layers are
    4-bit. Returns [M, N] of ``out_dtype``. Stacks whose weights fit one CU's LDS (depth <= 8, widths
    <= 256: feat_net) run in one launch, others layer by layer."""
    what = "mx4_sequential"
    layers = list(layers)
    if not layers:
        raise ValueError(f"{what}: no layers")
    if any(not isinstance(y, MX4Layer) for y in layers):
        raise TypeError(f"{what}: MX4Layer expected")
    for a, b in zip(layers, layers[1:]):
        if b.weight.cols != a.weight.shape[0]:
            raise ValueError(f"{what}: a layer of width {b.weight.cols} behind {a.weight.shape[0]} outputs")
    t, xt = _type(out_dtype, what), _type(x.dtype, what)
    rows, M, K, ldx = _rows(x, what)
    if K != layers[0].weight.cols:
        raise ValueError(f"{what}: input width {K} vs weight {layers[0].weight.shape}")
    dev = _device(what, rows)
    for y in layers:
        y.weight._index(what, dev)
    args = (L.MX4LayerArg * len(layers))(*(y._arg() for y in layers))
    if len(layers) > 1 and L.load().apn_mx4_network_lds_bytes(len(layers), args):
        out = torch.empty((M, layers[-1].weight.shape[0]), dtype=out_dtype, device=rows.device)
        _launch(dev, "apn_mx4_network", rows.data_ptr(), xt, ldx, M, len(layers), args, out.data_ptr(), t, out.shape[1])
        return out
    h = rows
    for y in layers[:-1]:
        h = mx4_linear(h, y.weight, y.bias, y.slope)
    return mx4_linear(h, layers[-1].weight, layers[-1].bias, layers[-1].slope, out_dtype=out_dtype)
