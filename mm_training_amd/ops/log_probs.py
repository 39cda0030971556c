"""Log probabilities of given categories with entropy, log-sum-exp and the likeliest alternatives, from logits, as HIP kernels with
their gradient (libmmt_hip.so, csrc/log_probs.hip): beside ``bev_geometry.depth_softmax`` what a depth distribution (or any other
categorical one, of any size) is asked for when it is a loss target, an uncertainty or a set of hypotheses.

Takes CUDA tensors, launches on the current stream, never falls back to torch ops."""
from collections import namedtuple

import torch
from torch.autograd import Function
from torch.autograd.forward_ad import unpack_dual

from .. import _lib

MAX_TOP = 64

LogProbs = namedtuple("LogProbs", ("log_prob", "entropy", "lse", "top_log_prob", "top_ids"))


def _rows(x):
    """(x with contiguous rows that are equally spaced in memory -- x itself where they are, else a copy --, rows, row stride)."""
    D = x.shape[-1]
    rows = x.numel() // D
    if D == 1 or x.stride(-1) == 1:
        R, span = None, None
        for n, s in zip(reversed(x.shape[:-1]), reversed(x.stride()[:-1])):
            if n == 1:
                continue
            if R is None:
                R, span = s, s * n
            elif s == span:
                span = s * n
            else:
                break
        else:
            if R is None or R >= D:
                return x, rows, D if R is None else R
    return x.contiguous(), rows, D


def _forward(x, ids, top, rows, R):
    D = x.shape[-1]
    lead, dev = x.shape[:-1], x.device
    bf16 = _lib.DTYPE_BF16 if x.dtype == torch.bfloat16 else _lib.DTYPE_F32
    entropy = torch.empty(lead, dtype=torch.float32, device=dev)
    lse = torch.empty(lead, dtype=torch.float32, device=dev)
    stats = torch.empty(lead + (4,), dtype=torch.float32, device=dev)
    log_prob = torch.empty(lead, dtype=torch.float32, device=dev) if ids is not None else None
    top_lp = torch.empty(lead + (top,), dtype=torch.float32, device=dev) if top else None
    top_ids = torch.empty(lead + (top,), dtype=torch.int64, device=dev) if top else None
    if rows:
        with _lib.on_device(dev):
            need = _lib.lib().mmt_log_probs_workspace_bytes(rows, D, top, bf16)
            ws = torch.empty(need, dtype=torch.uint8, device=dev) if need > 0 else None
            _lib.timed_call("log_probs", "mmt_log_probs_forward", rows, D, x.data_ptr(), R, bf16, ids.data_ptr() if ids is not None else 0,
                            ids.element_size() if ids is not None else 0, top, log_prob.data_ptr() if ids is not None else 0,
                            entropy.data_ptr(), lse.data_ptr(), stats.data_ptr(), top_lp.data_ptr() if top else 0,
                            top_ids.data_ptr() if top else 0, ws.data_ptr() if ws is not None else 0, max(need, 0), _lib.raw_stream(dev))
    return log_prob, entropy, lse, top_lp, top_ids, stats


def _backward(ctx, g_lp, g_h, g_lse, g_top, _):
    x, ids, stats, top_ids = ctx.saved_tensors
    top, rows, R = ctx.meta
    if g_lp is None and g_h is None and g_lse is None and g_top is None:
        return None, None, None
    D, dev = x.shape[-1], x.device
    grad = torch.empty(x.shape, dtype=x.dtype, device=dev)
    if rows:
        f32 = torch.float32
        g = [t if t is None or t.dtype is f32 and t.is_contiguous() else t.float().contiguous() for t in (g_lp, g_h, g_lse, g_top)]
        with _lib.on_device(dev):
            _lib.timed_call("log_probs_backward", "mmt_log_probs_backward", rows, D, x.data_ptr(), R, _lib.DTYPE_BF16 if x.dtype is torch.bfloat16 else _lib.DTYPE_F32,
                            ids.data_ptr() if ids is not None else 0, ids.element_size() if ids is not None else 0, top, stats.data_ptr(),
                            top_ids.data_ptr() if top else 0, *[0 if t is None else t.data_ptr() for t in g], grad.data_ptr(), D, _lib.raw_stream(dev))
    return grad, None, None


_backward_once = torch.autograd.function.once_differentiable(_backward)


class LogProbsFunction(Function):
    @staticmethod
    def forward(ctx, logits, ids, top):
        x, rows, R = _rows(logits)
        log_prob, entropy, lse, top_lp, top_ids, stats = _forward(x, ids, top, rows, R)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, ids, stats, top_ids)
        ctx.meta = (top, rows, R)
        if top:
            ctx.mark_non_differentiable(top_ids)
        return log_prob, entropy, lse, top_lp, top_ids

    @staticmethod
    def backward(ctx, *grads):
        # (grad mode is on in here under create_graph only: then a second differentiation has to raise)
        return (_backward_once if torch.is_grad_enabled() else _backward)(ctx, *grads)


def log_probs(logits, ids=None, top=0, dim=-1):
    """logits fp32 / bf16 with D categories along ``dim`` -> LogProbs of fp32 tensors (top_ids: int64), one value per row:

      log_prob      log softmax(logits)[ids]; None without ids.  An id outside 0 .. D - 1 (-1, -100, ..) names no category: log
                    probability 0 and no gradient
      entropy       -sum p log p          lse   log sum exp(logits)
      top_log_prob, top_ids   [..., top]: the ``top`` (<= 64) likeliest categories and their log probabilities, the lowest index first among
                    equal logits; None for top = 0

    All but top_ids carry gradients (first order, reverse mode; a forward-mode dual tensor is refused).  ``ids`` (int32 / int64) has
    the shape of ``logits`` without ``dim``; so have the results.  The rows may lie apart (a channel slice, ``dim=1`` of a
    channels_last [N, D, H, W] tensor): read in place where they are equally spaced with contiguous categories, else from one
    copy.  A row whose logits are all -inf has lse and log probabilities -inf,
    entropy 0 and gradient 0; NaN or +inf in a row makes its values NaN."""
    if not logits.is_cuda:
        raise RuntimeError("logits must be a CUDAtensor ")
    if logits.dtype not in (torch.float32, torch.bfloat16) or logits.dim() < 1:
        raise RuntimeError(f"logits must be a float32 / bfloat16 tensor of at least one dimension (found {logits.dtype}, {logits.dim()}-d)")
    if not -logits.dim() <= dim < logits.dim():
        raise RuntimeError(f"log_probs: dim {dim} of a {logits.dim()}-d tensor")
    x = logits if dim == -1 or dim == logits.dim() - 1 else logits.movedim(dim, -1)
    D = x.shape[-1]
    if D < 1 or D > 0x7FFFFFFF:
        raise RuntimeError(f"log_probs: {D} categories")
    top = int(top)
    if not 0 <= top <= min(MAX_TOP, D):
        raise RuntimeError(f"log_probs: top={top} is outside 0 .. min({MAX_TOP}, {D})")
    if ids is not None:
        if ids.dtype not in (torch.int32, torch.int64) or ids.device != logits.device or tuple(ids.shape) != tuple(x.shape[:-1]):
            raise RuntimeError(f"log_probs: ids must be an int32 / int64 tensor of shape {tuple(x.shape[:-1])} on {logits.device} "
                               f"(found {ids.dtype} {tuple(ids.shape)} on {ids.device})")
        ids = ids.contiguous()
    # (a dual tensor, which stays one under no_grad, takes the function too: that raises for want of a jvp; the kernel would drop the tangent)
    if (logits.requires_grad and torch.is_grad_enabled()) or unpack_dual(logits).tangent is not None:
        return LogProbs(*_lib.apply_function(LogProbsFunction, x, ids, top))
    x, rows, R = _rows(x)
    return LogProbs(*_forward(x, ids, top, rows, R)[:5])
