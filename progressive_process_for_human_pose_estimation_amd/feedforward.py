"""A gated feed-forward block over the channels of a feature map on HIP kernels (csrc/hgk_ffn.hip,
hgk_dropout.hip, hgk_linear_i8.hip), for training and, in 8-bit integers, for serving.

    gated_linear(x, w_gate, w_up, activation)             act(x w_gate^T) * (x w_up^T)
    linear_dropout_add(x, w, residual, p, seed, offset)   residual + dropout(x w^T)
    dropout_add(x, residual, p, seed, offset)             residual + dropout(x)
    quantize_rows(x)                                      int8 rows and a scale for each
    linear_i8(x, w, w_scale, bias, residual)              the product in 8-bit integers
    gated_linear_i8(x, wg, sg, wu, su, activation)        the gated product in 8-bit integers
    Dropout, GatedFeedForward, GatedFeedForwardI8         the modules made of them

Activations are channels-last: [..., C] fp32 or bf16 on the GPU (an NCHW map in channels_last
memory is `x.permute(0, 2, 3, 1)`, without a copy). Weights are [out, in] in the activations' type;
gradients have the type of what they belong to. Sums are fp32 (int32 in the 8-bit products) and results
are rounded once; the gated product's backward rounds the gradients of its two inner products to the
operands' type on the way. Other strides, and views that do not start on a 16-byte border, are copied
first.

Dropout's mask is a function of (seed, offset, element) and never stored: the backward draws it
again. An element is dropped with probability p to the nearest 2^-16 and the rest is scaled by the
inverse of the probability that is kept. The same (seed, offset) gives the same mask: pass another
offset for each use. `step`, an int64 GPU tensor of one element, is added to the offset on the
device, so that a captured graph draws other masks at each replay; it must not change between a
forward and its backward. Everything here can be captured (a backward together with its forward, on
leaves of which no eager graph is alive) and traced by torch.jit.trace; forward mode, make_fx and a
second derivative are refused. There is no CPU fallback.
"""
import math

import torch
import torch.nn as nn
from torch.autograd import forward_ad

from . import hgk as H

ACTIVATIONS = {"silu": 0, "gelu": 1, "relu": 2, "sigmoid": 3}
_DTYPES = {torch.float32: H.F32, torch.bfloat16: H.BF16}
_U64 = 1 << 64
_PROXY = torch._C._TorchDispatchModeKey.PROXY
_dispatch_mode, _tracing = torch._C._get_dispatch_mode, torch._C._is_tracing


def _code(what, x):
    dt = _DTYPES.get(x.dtype)
    if dt is None:
        raise H.HgkError(f"{what}: unsupported dtype {x.dtype} (float32 or bfloat16)")
    return dt


def _act(activation):
    a = ACTIVATIONS.get(activation)
    if a is None:
        raise H.HgkError(f"unknown activation {activation!r}: expected one of {sorted(ACTIVATIONS)}")
    return a


def _dense(t):
    """t as the kernels read it: dense, on a 16-byte border"""
    if not t.is_contiguous():
        t = t.contiguous()
    return t.clone() if t.data_ptr() & 15 else t


def _check(what, x, k, *others):
    """x [..., k] and the other operands: on one device, each of its type"""
    if _dispatch_mode(_PROXY) is not None:
        raise H.HgkError(f"{what}: make_fx cannot record it (torch.jit.trace can)")
    shape = x.shape
    if not shape or shape[-1] != k:
        raise H.HgkError(f"{what}: expected rows of {k} channels, got shape {tuple(shape)}")
    device = x.device
    for t, dtype in others:
        if t is not None and (t.dtype is not dtype or t.device != device):
            if t.device != device:
                raise H.HgkError(f"{what}: operands on {device} and {t.device}")
            raise H.HgkError(f"{what}: expected {dtype}, got {t.dtype}")


def _gpu(what, x):
    if not x.is_cuda:
        raise H.HgkError(f"{what}: tensors must live on the GPU")


def _weight_type(x, masters):
    """The type that weights have to be of: x's, or fp32 for a module's masters, which are rounded to x's type
    for the products and have fp32 gradients"""
    return torch.float32 if masters and x.dtype is torch.bfloat16 else x.dtype


def _check_weights(what, w, v=None):
    shape = w.shape
    if len(shape) != 2 or 0 in shape or (v is not None and v.shape != shape):
        raise H.HgkError(f"{what}: weights are [out, in], got {[tuple(t.shape) for t in (w, v) if t is not None]}")
    return shape


def _check_dropout(p, seed, offset, step, device):
    if not 0.0 <= p <= 1.0:
        raise H.HgkError(f"dropout: p = {p} is no probability")
    if not (isinstance(seed, int) and isinstance(offset, int) and 0 <= seed < _U64 and 0 <= offset < _U64):
        raise H.HgkError("dropout: seed and offset are whole numbers of 64 bits")
    if step is not None and (step.dtype != torch.int64 or step.numel() != 1 or step.device != device):
        raise H.HgkError(f"dropout: step is an int64 tensor of one element on {device}")


def _by_function(*operands):
    """Whether a call goes through its autograd function: where a gradient is wanted, under torch.jit.trace
    (which records functions; of a bare launch it would record the allocation of the result) and in forward
    mode (where a function refuses the tangent that a bare launch would lose)"""
    if _tracing() or forward_ad._current_level >= 0:
        return True
    if torch.is_grad_enabled():
        for t in operands:
            if t is not None and t.requires_grad:
                return True
    return False


def _launch(x, fn, *args):
    """fn(stream, *args) on x's device and that device's current stream"""
    dev = x.get_device()
    if dev == torch._C._cuda_getDevice():
        rc = fn(torch._C._cuda_getCurrentRawStream(dev), *args)
    else:
        with torch.cuda.device(dev):
            rc = fn(torch._C._cuda_getCurrentRawStream(dev), *args)
    if rc:
        H.check(rc)


def _workspace(n, x):
    """(pointer, bytes, owner) of a scratch buffer of the call's stream"""
    if not n:
        return None, 0, None
    ws = torch.empty(n, dtype=torch.uint8, device=x.device)
    return ws.data_ptr(), n, ws


def _wanted(dx, dw):
    """HGK_BWD_*: all, the input's or the weights' gradients"""
    return 1 if dx and dw else 2 if dx else 3


def _once(backward):
    """once_differentiable, whose bookkeeping is spared where no second derivative can be asked for"""
    checked = torch.autograd.function.once_differentiable(backward)

    def call(ctx, grad):
        return checked(ctx, grad) if torch.is_grad_enabled() else backward(ctx, grad)
    return call


# The operands are checked where they are launched, not before the autograd function: a traced graph calls
# the function by itself, with other operands.

# ---- the gated product ----
def _gated_operands(x, w_gate, w_up, activation, masters):
    """(x, w_gate, w_up, activation) as the kernels take them, or HgkError"""
    C = _check_weights("gated_linear", w_gate, w_up)[1]
    of = _weight_type(x, masters) if masters else x.dtype
    _check("gated_linear", x, C, (w_gate, of), (w_up, of))
    _code("gated_linear", x)
    act = _act(activation)
    _gpu("gated_linear", x)
    if of is not x.dtype:
        w_gate, w_up = w_gate.to(x.dtype), w_up.to(x.dtype)
    return _dense(x), _dense(w_gate), _dense(w_up), act


def _gated_fwd(x, wg, wu, act):
    F, C = wg.shape
    M, dt, lib = x.numel() // C, _DTYPES[x.dtype], H.lib()
    h = x.new_empty((*x.shape[:-1], F))
    wp, n, own = _workspace(lib.hgk_gated_workspace(dt, M, C, F, 0), x)
    _launch(x, lib.hgk_gated_fwd, dt, x.data_ptr(), wg.data_ptr(), wu.data_ptr(), h.data_ptr(), M, C, F,
            act, wp, n)
    return h


class _Gated(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, wg, wu, activation, masters):
        ctx.wtype = _weight_type(x, masters)
        x, wg, wu, act = _gated_operands(x, wg, wu, activation, masters)
        ctx.save_for_backward(x, wg, wu)
        ctx.act = act
        return _gated_fwd(x, wg, wu, act)

    @staticmethod
    @_once
    def backward(ctx, dh):
        x, wg, wu = ctx.saved_tensors
        F, C = wg.shape
        M, dt, lib = x.numel() // C, _DTYPES[x.dtype], H.lib()
        dh = _dense(dh)
        dx = torch.empty_like(x) if ctx.needs_input_grad[0] else None
        dw = ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        dwg, dwu = (torch.empty_like(v, dtype=ctx.wtype) for v in (wg, wu)) if dw else (None, None)
        wp, n, own = _workspace(lib.hgk_gated_workspace(dt, M, C, F, _wanted(dx is not None, dw)), x)
        if ctx.wtype is not x.dtype:
            dt |= H.F32_WGRAD
        _launch(x, lib.hgk_gated_bwd, dt, x.data_ptr(), wg.data_ptr(), wu.data_ptr(), dh.data_ptr(),
                H.ptr(dx), H.ptr(dwg), H.ptr(dwu), M, C, F, ctx.act, wp, n)
        return dx, dwg, dwu, None, None


def _gated(x, w_gate, w_up, activation, masters=False):
    if _by_function(x, w_gate, w_up):
        return _Gated.apply(x, w_gate, w_up, activation, masters)
    return _gated_fwd(*_gated_operands(x, w_gate, w_up, activation, masters))


def gated_linear(x, w_gate, w_up, activation="silu"):
    """act(x w_gate^T) * (x w_up^T): x [..., C], w_gate and w_up [F, C] -> [..., F]. Both products, the
    activation and the product of the two in one kernel; the backward computes them again and keeps
    nothing but the inputs. activation: silu, gelu (erf), relu, sigmoid."""
    return _gated(x, w_gate, w_up, activation)


# ---- product, dropout and residual ----
def _linear_operands(x, w, residual, p, seed, offset, step, masters):
    N, K = _check_weights("linear_dropout_add", w)
    of = _weight_type(x, masters) if masters else x.dtype
    _check("linear_dropout_add", x, K, (w, of), (residual, x.dtype))
    _code("linear_dropout_add", x)
    if residual is not None and residual.shape != (*x.shape[:-1], N):
        raise H.HgkError(f"linear_dropout_add: residual of shape {tuple(residual.shape)}")
    _check_dropout(p, seed, offset, step, x.device)
    _gpu("linear_dropout_add", x)
    if of is not x.dtype:
        w = w.to(x.dtype)
    return _dense(x), _dense(w), None if residual is None else _dense(residual)


def _linear_fwd(x, w, res, p, seed, offset, step):
    N, K = w.shape
    M, dt, lib = x.numel() // K, _DTYPES[x.dtype], H.lib()
    y = x.new_empty((*x.shape[:-1], N))
    wp, n, own = _workspace(lib.hgk_linear_workspace(dt, M, K, N, p > 0, 0), x)
    _launch(x, lib.hgk_linear_fwd, dt, x.data_ptr(), w.data_ptr(), H.ptr(res), y.data_ptr(), M, K, N, p,
            seed, offset, H.ptr(step), wp, n)
    return y


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, res, p, seed, offset, step, masters):
        ctx.wtype = _weight_type(x, masters)
        x, w, res = _linear_operands(x, w, res, p, seed, offset, step, masters)
        ctx.save_for_backward(x, w, step)
        ctx.drop = (p, seed, offset)
        return _linear_fwd(x, w, res, p, seed, offset, step)

    @staticmethod
    @_once
    def backward(ctx, dy):
        x, w, step = ctx.saved_tensors
        p, seed, offset = ctx.drop
        N, K = w.shape
        M, dt, lib = x.numel() // K, _DTYPES[x.dtype], H.lib()
        dx = dw = None
        if ctx.needs_input_grad[0] or ctx.needs_input_grad[1]:
            g = _dense(dy)
            dx = torch.empty_like(x) if ctx.needs_input_grad[0] else None
            dw = torch.empty_like(w, dtype=ctx.wtype) if ctx.needs_input_grad[1] else None
            drops = int(p * 65536 + 0.5) > 0
            wp, n, own = _workspace(lib.hgk_linear_workspace(dt, M, K, N, drops, _wanted(dx is not None, dw is not None)), x)
            if ctx.wtype is not x.dtype:
                dt |= H.F32_WGRAD
            _launch(x, lib.hgk_linear_bwd, dt, x.data_ptr(), w.data_ptr(), g.data_ptr(), H.ptr(dx),
                    H.ptr(dw), M, K, N, p, seed, offset, H.ptr(step), wp, n)
        return dx, dw, dy if ctx.needs_input_grad[2] else None, None, None, None, None, None


def _linear(x, w, residual, p=0.0, seed=0, offset=0, step=None, masters=False):
    if _by_function(x, w, residual):
        return _Linear.apply(x, w, residual, p, seed, offset, step, masters)
    return _linear_fwd(*_linear_operands(x, w, residual, p, seed, offset, step, masters), p, seed, offset, step)


def linear_dropout_add(x, w, residual=None, p=0.0, seed=0, offset=0, step=None):
    """residual + dropout(x w^T): x [..., K], w [N, K], residual [..., N] or None -> [..., N]; dropout
    and residual in the product's epilogue. The mask is dropout_add's over the output."""
    return _linear(x, w, residual, p, seed, offset, step)


# ---- dropout ----
def _dropout_operands(x, residual, rows_per_mask, p, seed, offset, step):
    if x.dim() < 1:
        raise H.HgkError("dropout_add: expected [..., C]")
    _check("dropout_add", x, x.shape[-1], (residual, x.dtype))
    _code("dropout_add", x)
    if residual is not None and residual.shape != x.shape:
        raise H.HgkError(f"dropout_add: residual of shape {tuple(residual.shape)} to {tuple(x.shape)}")
    if rows_per_mask is None:
        if x.dim() < 3:
            raise H.HgkError(f"dropout_add: rows_per_mask = None takes [N, ..., C], got shape {tuple(x.shape)}")
        rows_per_mask = max(1, int(math.prod(x.shape[1:-1])))
    if not (isinstance(rows_per_mask, int) and 1 <= rows_per_mask < _U64 >> 1):
        raise H.HgkError(f"dropout_add: rows_per_mask = {rows_per_mask}")
    _check_dropout(p, seed, offset, step, x.device)
    _gpu("dropout_add", x)
    return _dense(x), None if residual is None else _dense(residual), rows_per_mask


def _dropout(x, res, rows_per_mask, p, seed, offset, step):
    C = x.shape[-1]
    y = torch.empty_like(x)
    n = x.numel()
    if n:
        _launch(x, H.lib().hgk_dropout_add, _DTYPES[x.dtype], x.data_ptr(), H.ptr(res), y.data_ptr(), n // C,
                C, rows_per_mask, p, seed, offset, H.ptr(step))
    return y


class _DropoutAdd(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, res, rows_per_mask, p, seed, offset, step):
        x, res, rows_per_mask = _dropout_operands(x, res, rows_per_mask, p, seed, offset, step)
        if step is not None:
            ctx.save_for_backward(step)
        ctx.args = (rows_per_mask, p, seed, offset, step is not None)
        return _dropout(x, res, rows_per_mask, p, seed, offset, step)

    @staticmethod
    @_once
    def backward(ctx, dy):
        rows_per_mask, p, seed, offset, has_step = ctx.args
        step = ctx.saved_tensors[0] if has_step else None
        of_x, of_res = ctx.needs_input_grad[:2]
        dx = _dropout(_dense(dy), None, rows_per_mask, p, seed, offset, step) if of_x else None
        return dx, dy if of_res else None, None, None, None, None, None


def dropout_add(x, residual=None, p=0.5, seed=0, offset=0, step=None, rows_per_mask=1):
    """residual + dropout(x) over [..., C]. rows_per_mask: that many consecutive rows share a mask row
    (H * W of an NHWC map, or None, drops whole channels of each image); what is dropped is selected
    away, so an infinity or NaN there does not reach the result."""
    if _by_function(x, residual):
        return _DropoutAdd.apply(x, residual, rows_per_mask, p, seed, offset, step)
    return _dropout(*_dropout_operands(x, residual, rows_per_mask, p, seed, offset, step), p, seed, offset, step)


# ---- 8-bit integers ----
def _no_gradient(ctx, *grads):
    raise H.HgkError("the 8-bit operators have no gradient: call them under torch.no_grad() or on detached operands")


class _QuantizeRows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        q, s = _quantize_rows(x)
        ctx.mark_non_differentiable(q, s)
        return q, s

    backward = staticmethod(_no_gradient)


def _quantize_rows(x):
    _check("quantize_rows", x, x.shape[-1] if x.dim() else 0)
    _code("quantize_rows", x)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise H.HgkError("quantize_rows: expected [..., K]")
    _gpu("quantize_rows", x)
    x = _dense(x)
    q = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    s = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    _launch(x, H.lib().hgk_quantize_rows_i8, _DTYPES[x.dtype], x.data_ptr(), q.data_ptr(), s.data_ptr(), s.numel(),
            x.shape[-1])
    return q, s


def quantize_rows(x):
    """(q int8 [..., K], scale fp32 [...]): scale = max |row| / 127, q = rint(row / scale). A row of
    zeros has scale 0; a row that holds an infinity or a NaN has scale NaN. No gradient."""
    return _QuantizeRows.apply(x) if _by_function(x) else _quantize_rows(x)


def _check_scale(what, s, n):
    if s is None:
        raise H.HgkError(f"{what}: weights without their scales")
    if tuple(s.shape) != (n,):
        raise H.HgkError(f"{what}: expected {n} values, got shape {tuple(s.shape)}")


def _linear_i8(x, w, w_scale, bias, residual):
    N, K = _check_weights("linear_i8", w)
    _check("linear_i8", x, K, (w, torch.int8), (w_scale, torch.float32), (bias, torch.float32),
           (residual, x.dtype))
    _code("linear_i8", x)
    if residual is not None and residual.shape != (*x.shape[:-1], N):
        raise H.HgkError(f"linear_i8: residual of shape {tuple(residual.shape)}")
    _check_scale("linear_i8", w_scale, N)
    if bias is not None:
        _check_scale("linear_i8", bias, N)
    _gpu("linear_i8", x)
    x, w, w_scale = _dense(x), _dense(w), _dense(w_scale)
    bias = None if bias is None else _dense(bias)
    residual = None if residual is None else _dense(residual)
    M, lib = x.numel() // K, H.lib()
    y = x.new_empty((*x.shape[:-1], N))
    wp, n, own = _workspace(lib.hgk_linear_i8_workspace(M, K, N, 0), x)
    _launch(x, lib.hgk_linear_i8, _DTYPES[x.dtype], x.data_ptr(), w.data_ptr(), w_scale.data_ptr(), H.ptr(bias),
            H.ptr(residual), y.data_ptr(), M, K, N, wp, n)
    return y


class _LinearI8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, *operands):
        return _linear_i8(*operands)

    backward = staticmethod(_no_gradient)


def linear_i8(x, w, w_scale, bias=None, residual=None):
    """x w^T (+ bias + residual) in 8-bit integers: x [..., K] fp32 / bf16 is quantised row by row
    (quantize_rows), w is int8 [N, K] with w_scale fp32 [N] (quantize_rows of the weights), bias fp32
    [N], residual [..., N] in x's type, which is the result's. The integer sums are exact (K <=
    131072). No gradient: a backward that reaches the result is refused."""
    call = _LinearI8.apply if _by_function(x, w_scale, bias, residual) else _linear_i8
    return call(x, w, w_scale, bias, residual)


def _gated_i8(x, wg, sg, wu, su, activation):
    F, C = _check_weights("gated_linear_i8", wg, wu)
    _check("gated_linear_i8", x, C, (wg, torch.int8), (wu, torch.int8), (sg, torch.float32), (su, torch.float32))
    _code("gated_linear_i8", x)
    act = _act(activation)
    _check_scale("gated_linear_i8", sg, F)
    _check_scale("gated_linear_i8", su, F)
    _gpu("gated_linear_i8", x)
    x, wg, sg, wu, su = _dense(x), _dense(wg), _dense(sg), _dense(wu), _dense(su)
    M, lib = x.numel() // C, H.lib()
    h = x.new_empty((*x.shape[:-1], F))
    wp, n, own = _workspace(lib.hgk_linear_i8_workspace(M, C, F, 1), x)
    _launch(x, lib.hgk_gated_i8, _DTYPES[x.dtype], x.data_ptr(), wg.data_ptr(), sg.data_ptr(), wu.data_ptr(),
            su.data_ptr(), h.data_ptr(), M, C, F, act, wp, n)
    return h


class _GatedI8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, *operands):
        return _gated_i8(*operands)

    backward = staticmethod(_no_gradient)


def gated_linear_i8(x, w_gate, gate_scale, w_up, up_scale, activation="silu"):
    """gated_linear with both products in 8-bit integers (see linear_i8): w_gate and w_up int8 [F, C]
    with a scale for each row. No gradient: a backward that reaches the result is refused."""
    call = _GatedI8.apply if _by_function(x, gate_scale, up_scale) else _gated_i8
    return call(x, w_gate, gate_scale, w_up, up_scale, activation)


# ---- modules ----
class _Masks(nn.Module):
    """The (seed, offset, step) of a module's dropout. The seed is drawn from torch's CPU generator at
    construction and the offset in every training call, so that torch.manual_seed governs the masks and
    torch.utils.checkpoint, which puts the generator back, draws the same ones again. `offset` keeps
    the last one. Under graph capture and in a trace the host's offset is frozen, so a device counter moves
    on at each replay and each use keeps the value that it saw, for its backward and for a checkpoint's recompute."""

    def __init__(self, p):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise H.HgkError(f"dropout: p = {p} is no probability")
        self.p = p
        self.seed, self.offset = self._draw(), 0
        self.register_buffer("step", torch.zeros(1, dtype=torch.int64), persistent=False)
        self._uses = (0, {})  # the last capture, and the counter's value in each of its uses by their offset

    @staticmethod
    def _draw():
        return int(torch.randint(0, 1 << 62, (1,), device="cpu").item())

    def next_mask(self, x):
        """keyword arguments of the next use, on x's device"""
        if not self.training or self.p == 0.0:
            return {"p": 0.0}
        tracing = _tracing()
        self.offset = 0 if tracing else self._draw()  # a trace is compared with another one: no number of its own
        return {"p": self.p, "seed": self.seed, "offset": self.offset, "step": self._recorded_step(x, tracing)}

    def _recorded_step(self, x, tracing):
        """The device counter's value for this use, None where neither a graph nor a trace records it"""
        if not tracing and not (x.is_cuda and torch.cuda.is_current_stream_capturing()):
            return None
        if self.step.device != x.device:
            raise H.HgkError(f"dropout: move the module to {x.device} before capturing or tracing it")
        if tracing:
            self.step.add_(1 << 32)
            return self.step.clone()
        # a forward within a backward is a recompute. It may be captured apart from its forward
        capture, recompute = H.capture_id(x.device), torch._C._current_graph_task_id() != -1
        if capture != self._uses[0] and not recompute:
            self._uses = (capture, {})
        uses = self._uses[1]
        if self.offset not in uses:
            if recompute:
                raise H.HgkError("dropout: a recompute under capture that does not draw its forward's mask: checkpoint "
                                 "with preserve_rng_state=True, and recompute before the module is captured anew")
            self.step.add_(1 << 32)
            uses[self.offset] = self.step.clone()
        return uses[self.offset]


class Dropout(_Masks):
    """nn.Dropout over channels-last [..., C] with the skip added in the same pass: forward(x,
    residual=None). channels=True drops whole channels of each image of an NHWC map (nn.Dropout2d)."""

    def __init__(self, p=0.5, channels=False):
        super().__init__(p)
        self.channels = channels

    def forward(self, x, residual=None):
        kw = self.next_mask(x)
        if kw["p"] == 0.0 and residual is None:
            return x
        if self.channels and x.dim() < 3:
            raise H.HgkError("Dropout(channels=True): expected an NHWC map")
        return dropout_add(x, residual, rows_per_mask=None if self.channels else 1, **kw)


class GatedFeedForward(_Masks):
    """x + dropout(w_down (act(w_gate x) * (w_up x))) over channels-last [..., channels]. Parameters
    are fp32 [out, in] with nn.Linear's initialisation; beside bf16 maps they are masters, rounded in each
    call, whose gradients stay fp32. quantized() gives the block in 8-bit integers for serving."""

    def __init__(self, channels, hidden, activation="silu", p=0.0, residual=True):
        super().__init__(p)
        _act(activation)
        self.activation, self.residual = activation, residual
        self.w_gate = nn.Parameter(torch.empty(hidden, channels))
        self.w_up = nn.Parameter(torch.empty(hidden, channels))
        self.w_down = nn.Parameter(torch.empty(channels, hidden))
        for w in (self.w_gate, self.w_up, self.w_down):
            nn.init.kaiming_uniform_(w, a=math.sqrt(5))

    def forward(self, x):
        ws = (self.w_gate, self.w_up, self.w_down)
        masters = all(w.dtype is torch.float32 for w in ws)
        wg, wu, wd = (w.to(_weight_type(x, masters)) for w in ws)
        h = _gated(x, wg, wu, self.activation, masters)
        return _linear(h, wd, x if self.residual else None, masters=masters, **self.next_mask(x))

    def quantized(self):
        return GatedFeedForwardI8(self)


class GatedFeedForwardI8(nn.Module):
    """A GatedFeedForward served in 8-bit integers: weights quantised once, with a scale for each
    output channel; activations row by row in each call. No dropout; a backward through it is refused."""

    def __init__(self, block):
        super().__init__()
        self.activation, self.residual = block.activation, block.residual
        for name in ("gate", "up", "down"):
            q, s = quantize_rows(getattr(block, "w_" + name).detach())
            self.register_buffer("w_" + name, q)
            self.register_buffer(name + "_scale", s)

    def _apply(self, fn, *args, **kwargs):
        # .to(dtype), .bfloat16() and the like: the scales stay fp32, whatever they are moved to
        scales = {n: getattr(self, n) for n in ("gate_scale", "up_scale", "down_scale")}
        super()._apply(fn, *args, **kwargs)
        for n, s in scales.items():
            if getattr(self, n).dtype is not s.dtype:
                setattr(self, n, s.to(getattr(self, n).device))
        return self

    def forward(self, x):
        h = gated_linear_i8(x, self.w_gate, self.gate_scale, self.w_up, self.up_scale, self.activation)
        return linear_i8(h, self.w_down, self.down_scale, residual=x if self.residual else None)
