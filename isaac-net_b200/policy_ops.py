"""Operators of the policy that reads NetModule.obs() and answers with a TrafficRequest, as CUDA kernels.

    y, n = block_norm(x, w, h, post_weight=, gate=, scale=)   norms before and after a residual block, gate, scale
    y    = gated_ffn(x, w_gate, w_up, w_down, act=)           the block itself: act(x Wg^T) * (x Wu^T), times Wd^T
    y    = counter_dropout(x, p, s0, env_id, episode, ctr)    dropout keyed by global env id, mask never stored
    token, logp = sample_logits(logits, u, ...)               temperature, top-k, top-p, min-p from given uniforms
    u    = uniforms(s0, n, env_id, episode, ctr)              such uniforms from the engine's counter RNG

The first three are differentiable (torch.autograd, once, in reverse mode; a tensor with a tangent is refused).  As everywhere in this package there is no CPU path and no
fallback: tensors live on one CUDA device, unsupported settings raise B200Unsupported, wrong shapes ValueError and wrong
types TypeError before anything is launched, and the work is queued on the current stream of the tensors' device.  The
calls may be captured in a CUDA graph.  The operators have no counterpart in isaac-net, whose policies are its user's.

The functions are csrc/policy_torch.cpp, on top of the C ABI (inb_block_norm_fwd and the others of
include/isaac_net_b200.h).
"""
from __future__ import annotations

import ctypes
import importlib.machinery
import importlib.util
import os

import torch

from . import _native as nat
from .engine import B200Unsupported


def _load():
    """The extension module, bound to the library that _native loaded (raises if either is missing)."""
    path = os.path.join(nat.LIB_DIR, nat.TORCH_LIB)
    if not os.path.exists(path):
        raise RuntimeError(f"{path} is missing: the policy operators have no fallback path. Build it with "
                           "`python -c 'import __graft_entry__ as g; g.build()'`.")
    name = nat.TORCH_LIB.split(".")[0]
    loader = importlib.machinery.ExtensionFileLoader(name, path)
    module = importlib.util.module_from_spec(importlib.util.spec_from_loader(name, loader))
    loader.exec_module(module)
    lib = nat.lib()
    names = [*nat.POLICY_EXPORTS, "inb_block_norm_work", "inb_gated_ffn_work"]
    module.bind({n: ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in names}, B200Unsupported)
    return module


_ext = _load()
_block_norm, _gated_ffn, _counter_dropout, _sample_logits = (_ext.block_norm, _ext.gated_ffn, _ext.counter_dropout,
                                                             _ext.sample_logits)


def block_norm(x, weight, h=None, *, post_weight=None, gate=None, scale=1.0, eps=1e-6):
    """The norms before and after a residual block, with its gate and residual scale, in one pass.

        y = x + scale * gate * (post_weight * h / rms(h));   n = weight * y / rms(y);   rms(v) = sqrt(mean(v^2) + eps)

    x, h [..., D] (bf16, fp16 or fp32; statistics in fp32), weight [D] the next block's pre-norm, post_weight [D] or None
    (h is added as it is), gate [..., D] or None: leading sizes those of x, then ones ([D]: one gate; [E, 1, D]: one per
    env; [E, R, D]: one per robot).  Returns (y, n); without h just n, the pre-norm of x.  Differentiable in every
    tensor.  D up to 8192."""
    return _block_norm(x, weight, h, post_weight, gate, scale, eps)


def gated_ffn(x, w_gate, w_up, w_down, *, act="silu"):
    """The gated feed-forward block y = (act(x w_gate^T) * (x w_up^T)) w_down^T.

    x [..., D], w_gate and w_up [F, D], w_down [D, F] (torch.nn.Linear's layout), all bf16 or all fp16; act "silu" or
    "gelu" (the erf form).  Products accumulate in fp32; the hidden activations (but for up to 8 rows without autograd)
    and, in the backward pass, the gradients of the two projections are rounded to the inputs' type (fp16: infinite above
    65504).  Differentiable in every tensor: a call that autograd records keeps the hidden activations and both projections
    rounded to 24 bits, 8 bytes for each of the N x F hidden elements.
    Rows of x and of the weights may be strided; where they are not 16-byte aligned a padded copy is made in the call.
    Waits inside the kernels have a limit; outputs of a call whose wait ran out are not valid, which status() tells."""
    code = nat.ACTS.get(act)
    if code is None:
        raise ValueError(f"act must be one of {tuple(nat.ACTS)}, got {act!r}")
    return _gated_ffn(x, w_gate, w_up, w_down, code)


def counter_dropout(x, p, s0, env_id, episode=None, ctr=None, *, stream=0):
    """Dropout of x [E, ...] drawn from the engine's counter RNG; the mask is recomputed, never stored.

    Element i of env e's row is dropped with probability p (held to a multiple of 2^-16) by a hash of (s0, env_id[e],
    episode[e], ctr[e], stream, i); what is kept is scaled by 1 / (1 - p).  s0 is the engine's key (NRB200Engine.s0, or
    engine.seed_key(seed)), env_id / episode / ctr [E] int64 its id, episode and step tensors (None: 0), stream tells
    the layers of one step apart.  The draw follows the global env id: shards of a batch drop what the whole batch
    drops.  A backward call uses the keys of its forward call, whatever has become of the counters since.  For
    inference, do not call it."""
    return _counter_dropout(x, p, s0, env_id, episode, ctr, stream)


def sample_logits(logits, u, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, mask=None):
    """One token a row: (token int64 [...], logp fp32 [...]) of logits [..., V] (bf16, fp16 or fp32) and uniforms u [...]
    fp32 in [0, 1) (the engine's counter RNG, or any other).

    In this order: divide by temperature (0: take the largest logit), keep the top_k largest (0: all), of those the
    smallest prefix whose mass reaches top_p (>= 1: all), of those the ones of at least min_p times the largest
    probability, then draw by inverse CDF in index order.  Ties go to the lowest index.  logp is the token's
    log-probability after the filters, what a policy gradient needs of the behaviour.  Each setting is a number or a
    tensor [...] of one per row (fp32; top_k int32).  A number out of its range raises ValueError; a row's entry, which only
    the device sees, counts as the nearest one in range, and NaN as 0.  mask [..., V] or [V] bool, False = not allowed; NaN logits are not
    allowed either.  A row that allows nothing gives token -1 and logp -inf.

    The masses are summed in fixed point (2^-40 of the largest), so the token does not depend on how the sum is split;
    weights below 2^-40 of the largest are never drawn."""
    return _sample_logits(logits, u, temperature, top_k, top_p, min_p, mask)


CH_SAMPLE = 0x53       # counter-RNG channel of uniforms()


def uniforms(s0, n, env_id, episode=None, ctr=None, *, stream=0):
    """[E, n] fp32 uniforms in [0, 1) of the engine's counter RNG (inb_rng_draw), keyed like counter_dropout's draws by
    (s0, env_id[e], episode[e], ctr[e], stream): the given random numbers of sample_logits."""
    if not isinstance(env_id, torch.Tensor):
        raise TypeError(f"env_id must be a tensor, got {type(env_id).__name__}")
    for name, t in (("env_id", env_id), ("episode", episode), ("ctr", ctr)):
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a tensor or None, got {type(t).__name__}")
        if not t.is_cuda:
            raise B200Unsupported(f"{name} is on {t.device}: the policy operators run on CUDA tensors only")
        if t.device != env_id.device:
            raise ValueError(f"{name} is on {t.device}, env_id on {env_id.device}")
        if t.dtype != torch.int64:
            raise TypeError(f"{name} is {t.dtype}, expected torch.int64")
        if t.dim() != 1 or t.shape != env_id.shape:
            raise ValueError(f"env_id, episode and ctr must have one shape [E], got {name} of {tuple(t.shape)}")
    if not (0 <= s0 <= 0xFFFFFFFF and 0 <= stream <= 0xFFFFFFFF):
        raise ValueError("s0 and stream are 32-bit words")
    e = env_id.shape[0]
    if n < 0 or e * n > 0x7FFFFFFF:
        raise B200Unsupported(f"uniforms: {e} x {n} draws are more than one call makes")
    episode = torch.zeros_like(env_id) if episode is None else episode
    env_id, episode, ctr = (t if t is None else t.contiguous() for t in (env_id, episode, ctr))
    out = torch.empty(e, n, device=env_id.device)
    with torch.cuda.device(env_id.device):
        rc = nat.lib().inb_rng_draw(e, n, s0, CH_SAMPLE, stream, env_id.data_ptr(), episode.data_ptr(),
                                    None if ctr is None else ctr.data_ptr(), 0, out.data_ptr(),
                                    torch.cuda.current_stream().cuda_stream)
    nat.check(rc, "inb_rng_draw")
    return out


def status(device="cuda"):
    """The device status word of the operators' kernels on `device` (0 = no wait inside a kernel ever ran out, in eager calls
    and in replays of graphs alike); reading it waits for all of the device's work."""
    i = torch.device(device).index
    return _ext.status(torch.cuda.current_device() if i is None else i)


__all__ = ["block_norm", "gated_ffn", "counter_dropout", "sample_logits", "uniforms", "status"]
