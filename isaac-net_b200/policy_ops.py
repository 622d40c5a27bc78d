"""Operators of the policy that reads NetModule.obs() and answers with a TrafficRequest, as CUDA kernels.

    y, n = block_norm(x, w, h, post_weight=, gate=, scale=)   norms before and after a residual block, gate, scale
    y    = gated_ffn(x, w_gate, w_up, w_down, act=)           the block itself: act(x Wg^T) * (x Wu^T), times Wd^T
    y    = counter_dropout(x, p, s0, env_id, episode, ctr)    dropout keyed by global env id, mask never stored
    token, logp = sample_logits(logits, u, ...)               temperature, top-k, top-p, min-p from given uniforms

The first three are differentiable (torch.autograd).  As everywhere in this package there is no CPU path and no fallback:
tensors live on one CUDA device, unsupported settings raise B200Unsupported before anything is launched, and the work
is queued on the current stream of the tensors' device.  The operators have no counterpart in isaac-net, whose
policies are its user's.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _native as nat
from .engine import B200Unsupported

_TYPES = {torch.bfloat16: nat.BF16, torch.float16: nat.F16, torch.float32: nat.F32}
_TYPES_16 = {torch.bfloat16: nat.BF16, torch.float16: nat.F16}
_M32 = 0xFFFFFFFF


# ---------------------------------------------------------------------------------------------------- plumbing
# A serving call is a few microseconds of device time, so the checks on the way are plain comparisons; messages are only
# put together once one fails.
_raw_stream, _current_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice


def _fits(t, dev, dtype):
    """Whether `t` is a tensor of `dtype` on CUDA device `dev` (an index)."""
    return isinstance(t, torch.Tensor) and t.dtype is dtype and t.get_device() == dev


def _refuse(t, name, like=None, dtype=None):
    """Raises what is wrong with an argument that does not fit."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise B200Unsupported(f"{name} is on {t.device}: the policy operators run on CUDA tensors only")
    if like is not None:
        if t.device != like.device:
            raise ValueError(f"{name} is on {t.device}, the first tensor on {like.device}")
        raise TypeError(f"{name} is {t.dtype}, expected {dtype or like.dtype}")
    raise B200Unsupported(f"{name} is {t.dtype}: not a type this operator takes")


def _first(t, name, types=_TYPES):
    """Checks an operator's first tensor [..., D]; its type code and device index."""
    code = types.get(t.dtype) if isinstance(t, torch.Tensor) else None
    if code is None or not t.is_cuda:
        _refuse(t, name)
    if t.dim() < 1 or t.shape[-1] < 1:
        raise ValueError(f"{name} must be [..., D] with D >= 1, got shape {tuple(t.shape)}")
    return code, t.get_device()


def _rows(t, d):
    """`t` [..., D] as rows: (tensor to read, row stride in elements), a copy where its rows have no one stride or its
    elements are not contiguous."""
    if t.is_contiguous():
        return t, d
    if t.stride(-1) == 1 or d == 1:
        if t.dim() == 2:
            return t, t.stride(0)
        try:
            v = t.view(-1, d)
            return v, v.stride(0)
        except RuntimeError:
            pass
    return t.contiguous(), d


def _ptr(t):
    return None if t is None else t.data_ptr()


def _call(name, args, dev):
    """Queue one call of the library on the current stream of device index `dev`."""
    fn = getattr(_lib or _load(), name)
    if _current_device() == dev:
        rc = fn(ctypes.byref(args), _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(ctypes.byref(args), _raw_stream(dev))
    if rc != 0:
        nat.check(rc, name)


_lib = None


def _load():
    global _lib
    _lib = nat.lib()
    return _lib


def _grad_on(*ts):
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                return True
    return False


# ---------------------------------------------------------------------------------------------------- block_norm
def _norm_rows(t, d):
    r, ld = _rows(t, d)
    return (r, ld) if ld <= nat.MAX_NORM_LD else (t.contiguous(), d)


def _norm_args(x, w, h, post, gate, gate_rows, scale, eps):
    """The argument block of one call on [N, D] rows, and the tensors that it points into."""
    d = x.shape[-1]
    xr, ldx = _norm_rows(x, d)
    hr, ldh = _norm_rows(h, d) if h is not None else (None, 0)
    a = nat.InbNormArgs(_TYPES[x.dtype], d, x.numel() // d, ldx, ldh, gate_rows, scale, eps, xr.data_ptr(), _ptr(hr),
                        w.data_ptr(), _ptr(post), _ptr(gate))
    return a, (xr, hr, w, post, gate)


def _norm_forward(x, w, h, post, gate, gate_rows, scale, eps, stats):
    a, keep = _norm_args(x, w, h, post, gate, gate_rows, scale, eps)
    n = x.new_empty(x.shape)
    y = x.new_empty(x.shape) if h is not None else None
    a.y, a.n, a.stats = _ptr(y), n.data_ptr(), _ptr(stats)
    if x.numel():
        _call("inb_block_norm_fwd", a, x.get_device())
    return y, n


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, h, post, gate, gate_rows, scale, eps):
        stats = torch.empty(x.numel() // x.shape[-1], 2, device=x.device)
        y, n = _norm_forward(x, w, h, post, gate, gate_rows, scale, eps, stats)
        ctx.save_for_backward(x, w, h, post, gate, stats)
        ctx.settings = gate_rows, scale, eps
        ctx.set_materialize_grads(False)
        return (y, n) if h is not None else n

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        gy, gn = grads if len(grads) == 2 else (None, grads[0])
        x, w, h, post, gate, stats = ctx.saved_tensors
        d = x.shape[-1]
        new = lambda t: None if t is None else torch.empty(t.shape, dtype=t.dtype, device=t.device)
        outs = gx, gw, gh, gpost, ggate = [new(t) for t in (x, w, h, post, gate)]
        if (gy is None and gn is None) or x.numel() == 0:
            for t in outs:
                if t is not None:
                    t.zero_()
            return (*outs, None, None, None)
        a, keep = _norm_args(x, w, h, post, gate, *ctx.settings)
        yr, a.ldgy = _norm_rows(gy, d) if gy is not None else (None, 0)
        nr, a.ldgn = _norm_rows(gn, d) if gn is not None else (None, 0)
        a.gy, a.gn, a.stats = _ptr(yr), _ptr(nr), stats.data_ptr()
        a.gx, a.gw, a.gh, a.gpost, a.ggate = gx.data_ptr(), gw.data_ptr(), _ptr(gh), _ptr(gpost), _ptr(ggate)
        size = nat.i64()
        nat.check(nat.lib().inb_block_norm_work(ctypes.byref(a), ctypes.byref(size)), "inb_block_norm_work")
        work = torch.empty(size.value, device=x.device)
        a.work, a.work_elems = work.data_ptr(), size.value
        _call("inb_block_norm_bwd", a, x.get_device())
        return (*outs, None, None, None)


def _gate_rows(gate, x):
    """How many consecutive rows of x [..., D] one gate of `gate` [g..., D] scales: gate's leading dims equal x's up to
    some axis and are 1 from there on (missing leading dims count as 1)."""
    full = tuple(x.shape)
    shape = (1,) * (len(full) - gate.dim()) + tuple(gate.shape)
    rows, axis = 1, len(full) - 2
    if len(shape) == len(full) and shape[-1] == full[-1]:
        while axis >= 0 and shape[axis] == 1:
            rows *= full[axis]
            axis -= 1
        if shape[:axis + 1] == full[:axis + 1]:
            return rows
    raise ValueError(f"gate of shape {tuple(gate.shape)} does not fit x of shape {full}: [..., D] with x's leading sizes, "
                     "then ones")


def block_norm(x, weight, h=None, *, post_weight=None, gate=None, scale=1.0, eps=1e-6):
    """The norms before and after a residual block, with its gate and residual scale, in one pass.

        y = x + scale * gate * (post_weight * h / rms(h));   n = weight * y / rms(y);   rms(v) = sqrt(mean(v^2) + eps)

    x, h [..., D] (bf16, fp16 or fp32; statistics in fp32), weight [D] the next block's pre-norm, post_weight [D] or None
    (h is added as it is), gate [..., D] or None: leading sizes those of x, then ones ([D]: one gate; [E, 1, D]: one per
    env; [E, R, D]: one per robot).  Returns (y, n); without h just n, the pre-norm of x.  Differentiable in every
    tensor.  D up to 8192."""
    dev = _first(x, "x")[1]
    d, dt = x.shape[-1], x.dtype
    if d > nat.MAX_NORM_D:
        raise B200Unsupported(f"block_norm: D = {d} is above {nat.MAX_NORM_D}")
    if x.numel() // d > 0x7FFFFFFF:
        raise B200Unsupported("block_norm: more than 2^31 - 1 rows")
    if not _fits(weight, dev, dt):
        _refuse(weight, "weight", x)
    if weight.shape != (d,):
        raise ValueError(f"weight must have shape ({d},), got {tuple(weight.shape)}")
    rows = 0
    if h is None:
        if post_weight is not None or gate is not None:
            raise ValueError("post_weight and gate need h")
    else:
        if not _fits(h, dev, dt):
            _refuse(h, "h", x)
        if h.shape != x.shape:
            raise ValueError(f"h of shape {tuple(h.shape)} does not match x of shape {tuple(x.shape)}")
        if post_weight is not None:
            if not _fits(post_weight, dev, dt):
                _refuse(post_weight, "post_weight", x)
            if post_weight.shape != (d,):
                raise ValueError(f"post_weight must have shape ({d},), got {tuple(post_weight.shape)}")
            post_weight = post_weight.contiguous()
        if gate is not None:
            if not _fits(gate, dev, dt):
                _refuse(gate, "gate", x)
            rows = _gate_rows(gate, x)
            gate = gate.contiguous()
    weight = weight.contiguous()
    scale, eps = float(scale), float(eps)
    if _grad_on(x, weight, h, post_weight, gate):
        return _BlockNorm.apply(x, weight, h, post_weight, gate, rows, scale, eps)
    y, n = _norm_forward(x, weight, h, post_weight, gate, rows, scale, eps, None)
    return (y, n) if h is not None else n


# ---------------------------------------------------------------------------------------------------- gated_ffn
_status = {}


def status(device="cuda"):
    """The device status word of the operators' kernels on `device` (0 = no wait inside a kernel ever ran out); reading it
    synchronizes."""
    i = torch.device(device).index
    w = _status.get(torch.cuda.current_device() if i is None else i)
    return 0 if w is None else int(w.item())


def _status_word(dev):
    w = _status.get(dev)
    if w is None:
        w = _status[dev] = torch.zeros(1, dtype=torch.int32, device=f"cuda:{dev}")
    return w


def _ffn_args(x, wg, wu, wd, act, h, g, u):
    """The argument block of one call on [N, D] rows, and the tensors that it points into."""
    d, f = x.shape[-1], wg.shape[0]
    (xr, ldx), (gr, ldg), (ur, ldu), (dr, ldd) = _rows(x, d), _rows(wg, d), _rows(wu, d), _rows(wd, f)
    a = nat.InbFfnArgs(_TYPES[x.dtype], act, d, f, x.numel() // d, ldx, ldg, ldu, ldd, h.shape[-1], 0, xr.data_ptr(),
                       gr.data_ptr(), ur.data_ptr(), dr.data_ptr(), None, h.data_ptr(), _ptr(g), _ptr(u))
    a.status = _status_word(x.get_device()).data_ptr()
    return a, (xr, gr, ur, dr)


def _ffn_work(a, backward, dev):
    size = nat.i64()
    nat.check(nat.lib().inb_gated_ffn_work(ctypes.byref(a), backward, ctypes.byref(size)), "inb_gated_ffn_work")
    if size.value == 0:
        return None
    work = torch.empty(size.value, dtype=torch.uint8, device=dev)
    a.work, a.work_bytes = work.data_ptr(), size.value
    return work


def _ffn_forward(x, wg, wu, wd, act, keep):
    """(y, h, g, u): g, u None unless `keep`."""
    n, ldh = x.numel() // x.shape[-1], (wg.shape[0] + 7) // 8 * 8
    few = not keep and n <= nat.FFN_ROWS
    y, h = x.new_empty(x.shape), x.new_empty(2 * n if few else n, ldh)
    g, u = (torch.empty(-(-n // 128) * 128, ldh, device=x.device) if keep else None for _ in range(2))
    if n:
        a, held = _ffn_args(x, wg, wu, wd, act, h, g, u)
        a.y = y.data_ptr()
        work = None if few else _ffn_work(a, 0, x.device)
        _call("inb_gated_ffn_fwd", a, x.get_device())
    return y, h, g, u


class _GatedFfn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, wg, wu, wd, act):
        y, h, g, u = _ffn_forward(x, wg, wu, wd, act, True)
        ctx.save_for_backward(x, wg, wu, wd, h, g, u)
        ctx.act = act
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, wg, wu, wd, h, g, u = ctx.saved_tensors
        need = ctx.needs_input_grad
        new = lambda t, on: torch.empty(t.shape, dtype=t.dtype, device=t.device) if on else None
        dx, dwg, dwu, dwd = (new(x, need[0]), new(wg, need[1] or need[2]), new(wu, need[1] or need[2]), new(wd, need[3]))
        if x.numel() == 0:
            for t in (dwg, dwu, dwd):
                if t is not None:
                    t.zero_()
            return dx, dwg, dwu, dwd, None
        a, held = _ffn_args(x, wg, wu, wd, ctx.act, h, g, u)
        dyr, a.lddy = _rows(dy, x.shape[-1])
        a.dy, a.dx, a.dwg, a.dwu, a.dwd = dyr.data_ptr(), _ptr(dx), _ptr(dwg), _ptr(dwu), _ptr(dwd)
        if dx is not None or dwg is not None:
            dg, du = torch.empty_like(h), torch.empty_like(h)
            a.dg, a.du = dg.data_ptr(), du.data_ptr()
        work = _ffn_work(a, 1, x.device)
        _call("inb_gated_ffn_bwd", a, x.get_device())
        return dx, dwg if need[1] else None, dwu if need[2] else None, dwd, None


def gated_ffn(x, w_gate, w_up, w_down, *, act="silu"):
    """The gated feed-forward block y = (act(x w_gate^T) * (x w_up^T)) w_down^T.

    x [..., D], w_gate and w_up [F, D], w_down [D, F] (torch.nn.Linear's layout), all bf16 or all fp16; act "silu" or
    "gelu" (the erf form).  Products accumulate in fp32; the hidden activations and, in the backward pass, the gradients of
    the two projections are rounded to the inputs' type.  Differentiable in every tensor: a call that autograd records
    keeps the projections, 10 bytes for each of the N x F hidden elements.  Rows of x and of the weights may be strided;
    where they are not 16-byte aligned a padded copy is made in the call."""
    dev = _first(x, "x", _TYPES_16)[1]
    if act not in nat.ACTS:
        raise ValueError(f"act must be one of {tuple(nat.ACTS)}, got {act!r}")
    d, dt = x.shape[-1], x.dtype
    for t, name in ((w_gate, "w_gate"), (w_up, "w_up"), (w_down, "w_down")):
        if not _fits(t, dev, dt):
            _refuse(t, name, x)
    f = w_gate.shape[0] if w_gate.dim() == 2 else 0
    if f < 1 or w_gate.shape != (f, d) or w_up.shape != (f, d) or w_down.shape != (d, f):
        raise ValueError(f"w_gate and w_up must be [F, {d}] and w_down [{d}, F], got {tuple(w_gate.shape)}, "
                         f"{tuple(w_up.shape)}, {tuple(w_down.shape)}")
    if max(d, f, x.numel() // d) > nat.MAX_FFN:
        raise B200Unsupported(f"gated_ffn: sizes above {nat.MAX_FFN}")
    if _grad_on(x, w_gate, w_up, w_down):
        return _GatedFfn.apply(x, w_gate, w_up, w_down, nat.ACTS[act])
    return _ffn_forward(x, w_gate, w_up, w_down, nat.ACTS[act], False)[0]


# ---------------------------------------------------------------------------------------------------- counter_dropout
def _dropout_run(x, threshold, s0, stream, env_id, episode, ctr, keys_in, keys_out):
    x = x.contiguous()
    y = torch.empty_like(x)
    e = x.shape[0]
    if x.numel():
        a = nat.InbDropoutArgs(_TYPES[x.dtype], threshold, e, x.numel() // e, s0, stream, _ptr(env_id), _ptr(episode),
                               _ptr(ctr), _ptr(keys_in), _ptr(keys_out), x.data_ptr(), y.data_ptr())
        _call("inb_dropout", a, x.get_device())
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, threshold, s0, stream, env_id, episode, ctr):
        keys = torch.empty(x.shape[0], dtype=torch.int32, device=x.device)
        ctx.save_for_backward(keys)
        ctx.threshold = threshold
        return _dropout_run(x, threshold, s0, stream, env_id, episode, ctr, None, keys)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gy):
        keys, = ctx.saved_tensors
        return _dropout_run(gy, ctx.threshold, 0, 0, None, None, None, keys, None), None, None, None, None, None, None


def counter_dropout(x, p, s0, env_id, episode=None, ctr=None, *, stream=0):
    """Dropout of x [E, ...] drawn from the engine's counter RNG; the mask is recomputed, never stored.

    Element i of env e's row is dropped with probability p (held to a multiple of 2^-16) by a hash of (s0, env_id[e],
    episode[e], ctr[e], stream, i); what is kept is scaled by 1 / (1 - p).  s0 is the engine's key (NRB200Engine.s0, or
    engine.seed_key(seed)), env_id / episode / ctr [E] int64 its id, episode and step tensors (None: 0), stream tells
    the layers of one step apart.  The draw follows the global env id: shards of a batch drop what the whole batch
    drops.  A backward call uses the keys of its forward call, whatever has become of the counters since.  With
    inference, do not call it."""
    if not isinstance(x, torch.Tensor) or x.dtype not in _TYPES or not x.is_cuda:
        _refuse(x, "x")
    if x.dim() < 1:
        raise ValueError("x must be [E, ...]")
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"p must be in [0, 1], got {p}")
    if not (0 <= s0 <= _M32 and 0 <= stream <= _M32):
        raise ValueError("s0 and stream are 32-bit words")
    e, dev = x.shape[0], x.get_device()
    for t, name in ((env_id, "env_id"), (episode, "episode"), (ctr, "ctr")):
        if t is None and name != "env_id":
            continue
        if not _fits(t, dev, torch.int64):
            _refuse(t, name, x, torch.int64)
        if t.shape != (e,):
            raise ValueError(f"{name} must have shape ({e},), got {tuple(t.shape)}")
    n = x.numel() // e if e else 0
    if n > nat.MAX_DROPOUT_N or e * max(1, -(-n // 4096)) > 0x7FFFFFFF:
        raise B200Unsupported(f"counter_dropout: {e} envs of {n} elements are more than one call can draw")
    env_id = env_id.contiguous()
    episode = None if episode is None else episode.contiguous()
    ctr = None if ctr is None else ctr.contiguous()
    threshold = round(p * 65536)
    if _grad_on(x):
        return _Dropout.apply(x, threshold, int(s0), int(stream), env_id, episode, ctr)
    return _dropout_run(x, threshold, int(s0), int(stream), env_id, episode, ctr, None, None)


# ---------------------------------------------------------------------------------------------------- sample_logits
def sample_logits(logits, u, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, mask=None):
    """One token a row: (token int64 [...], logp fp32 [...]) of logits [..., V] (bf16, fp16 or fp32) and uniforms u [...]
    fp32 in [0, 1) (the engine's counter RNG, or any other).

    In this order: divide by temperature (<= 0: take the largest logit), keep the top_k largest (0: all), of those the
    smallest prefix whose mass reaches top_p (>= 1: all), of those the ones of at least min_p times the largest
    probability, then draw by inverse CDF in index order.  Ties go to the lowest index.  logp is the token's
    log-probability after the filters, what a policy gradient needs of the behaviour.  Each setting is a number or a
    tensor [...] of one per row (fp32; top_k int32).  mask [..., V] or [V] bool, False = not allowed; NaN logits are not
    allowed either.  A row that allows nothing gives token -1 and logp -inf.

    The masses are summed in fixed point (2^-40 of the largest), so the token does not depend on how the sum is split;
    weights below 2^-40 of the largest are never drawn."""
    code, dev = _first(logits, "logits")
    v, lead = logits.shape[-1], logits.shape[:-1]
    n = logits.numel() // v
    if v > nat.MAX_SAMPLE_V or n > nat.MAX_SAMPLE_N:
        raise B200Unsupported(f"sample_logits: {n} rows of {v}: at most {nat.MAX_SAMPLE_N} rows of {nat.MAX_SAMPLE_V}")
    if not _fits(u, dev, torch.float32):
        _refuse(u, "u", logits, torch.float32)
    if u.shape != lead:
        raise ValueError(f"u must have shape {tuple(lead)}, got {tuple(u.shape)}")
    lr, ld = _rows(logits, v)
    keep, scalars, rows = [], [], []
    for value, name in ((temperature, "temperature"), (top_p, "top_p"), (min_p, "min_p"), (top_k, "top_k")):
        if isinstance(value, torch.Tensor):
            dt = torch.int32 if name == "top_k" else torch.float32
            if not _fits(value, dev, dt):
                _refuse(value, name, logits, dt)
            if value.shape != lead:
                raise ValueError(f"{name} must be a number or have shape {tuple(lead)}, got {tuple(value.shape)}")
            value = value.contiguous()
            keep.append(value)
            scalars.append(0)
            rows.append(value.data_ptr())
        else:
            if not value >= 0 or (name == "min_p" and value > 1.0) or (name == "top_k" and int(value) != value):
                raise ValueError(f"{name} = {value} is out of range")
            rows.append(None)
            scalars.append(min(int(value), 0x7FFFFFFF) if name == "top_k" else value)
    mr, ldm = None, 0
    if mask is not None:
        if not _fits(mask, dev, torch.bool):
            _refuse(mask, "mask", logits, torch.bool)
        if mask.shape != logits.shape and mask.shape != (v,):
            raise ValueError(f"mask must have shape {tuple(logits.shape)} or ({v},), got {tuple(mask.shape)}")
        mr, ldm = (mask.contiguous(), 0) if mask.dim() == 1 and logits.dim() > 1 else _rows(mask, v)
    u = u.contiguous()
    token, logp = u.new_empty(lead, dtype=torch.int64), u.new_empty(lead)
    if n:
        a = nat.InbSampleArgs(code, v, n, ld, ldm, lr.data_ptr(), _ptr(mr), u.data_ptr(), scalars[0],
                              scalars[1], scalars[2], scalars[3], rows[0], rows[1], rows[2], rows[3], token.data_ptr(),
                              logp.data_ptr())
        _call("inb_sample", a, dev)
    return token, logp


__all__ = ["block_norm", "gated_ffn", "counter_dropout", "sample_logits", "status"]
