"""tensorplay_amd: MI355X (gfx950) backend for TensorPlay's P10 reduction + top-k path.

The Python surface mirrors the parts of TensorPlay this path touches:
``Tensor`` methods sum/mean/max/min/argmax/argmin/var/std (the overload set of
/root/reference/src/bindings/python/Tensor.cpp:1099-1224) plus ``topk``, and the
module functions of /root/reference/tensorplay/functional.py:401-432, plus
softmax / log_softmax / nll_loss (functional.py:313-317, 496-500) and their
gradients.  Tensors
live on ``"cpu"`` or ``"rocm[:N]"``; reductions run on ROCm devices only (the
CPU key has no kernels here -- that path stays TensorPlay's own).

The native library must be built (``python tensorplay_amd/build.py``); there is
no fallback.
"""
try:
    # One HIP runtime per process: torch ships its own libamdhip64 (same soname)
    # and its libraries load it by file name, so if this package's runtime were
    # loaded first the process would hold two.  Loading torch first makes both
    # resolve to torch's copy.
    import torch as _torch  # noqa: F401
except ImportError:
    pass
from . import _C  # noqa: E402

__version__ = "0.1.0"

Tensor = _C.TensorBase
DType = _C.DType
Device = _C.Device

uint8 = DType.uint8
int8 = DType.int8
int16 = DType.int16
int32 = DType.int32
int64 = DType.int64
uint16 = DType.uint16
uint32 = DType.uint32
uint64 = DType.uint64
float32 = DType.float32
float64 = DType.float64
bool_ = DType.bool
float16 = DType.float16    # half precision: the fine-tuning operators and copies between equal dtypes
bfloat16 = DType.bfloat16
undefined = DType.undefined


def device(spec):
    return Device(spec)


def tensor(data, dtype=None, device="cpu"):
    """Copy array-like `data` into a new tensor on `device` ("cpu" / "rocm[:N]")."""
    import numpy as np
    arr = np.asarray(data)
    if dtype is None and arr.dtype == np.float64 and not isinstance(data, np.ndarray):
        arr = arr.astype(np.float32)  # Python floats default to float32, as TensorPlay's tensor()
    return _C.tensor(arr, dtype, str(device))


def from_numpy(arr, device="cpu"):
    return _C.tensor(arr, None, str(device))


def empty(shape, dtype=float32, device="cpu"):
    return _C.empty(list(shape), dtype, str(device))


def from_torch(t):
    """Zero-copy view of a torch tensor that lives on an AMD GPU (keeps `t` alive)."""
    return _C._from_torch(t)


_from_dlpack = None


def to_torch(t):
    """Zero-copy torch view of a tensor (DLPack; keeps the tensor's memory alive).
    Its memory belongs to the stream that was current when it was allocated: mark
    the tensor with record_stream before another stream uses it."""
    global _from_dlpack
    if _from_dlpack is None:
        from torch.utils.dlpack import from_dlpack as _from_dlpack
    return _from_dlpack(_C._to_dlpack(t))


# ---- functional forms (tensorplay/functional.py:401-432 + topk) ----
def sum(input, dim=None, keepdim=False, dtype=None):
    return input.sum(dtype=dtype) if dim is None else input.sum(dim, keepdim, dtype=dtype)


def mean(input, dim=None, keepdim=False, dtype=None):
    return input.mean(dtype=dtype) if dim is None else input.mean(dim, keepdim, dtype=dtype)


def max(input, dim=None, keepdim=False):
    return input.max() if dim is None else input.max(dim, keepdim)


def min(input, dim=None, keepdim=False):
    return input.min() if dim is None else input.min(dim, keepdim)


def amax(input, dim=None, keepdim=False):
    return max(input, dim, keepdim)


def amin(input, dim=None, keepdim=False):
    return min(input, dim, keepdim)


def argmax(input, dim=None, keepdim=False):
    return input.argmax(dim, keepdim)


def argmin(input, dim=None, keepdim=False):
    return input.argmin(dim, keepdim)


def var(input, dim=None, correction=1, keepdim=False):
    return input.var(correction) if dim is None else input.var(dim, correction, keepdim)


def std(input, dim=None, correction=1, keepdim=False):
    return input.std(correction) if dim is None else input.std(dim, correction, keepdim)


def prod(input, dim=None, keepdim=False, dtype=None):
    return input.prod(dtype=dtype) if dim is None else input.prod(dim, keepdim, dtype=dtype)


def all(input, dim=None, keepdim=False):
    return input.all() if dim is None else input.all(dim, keepdim)


def any(input, dim=None, keepdim=False):
    return input.any() if dim is None else input.any(dim, keepdim)


def median(input):
    return input.median()


def norm(input, p=2.0, dim=None, keepdim=False):
    return input.norm(p) if dim is None else input.norm(dim, p, keepdim)


def topk(input, k, dim=-1, largest=True, sorted=True):
    return input.topk(k, dim, largest, sorted)


def softmax(input, dim, dtype=None):
    return input.softmax(dim, dtype)


def log_softmax(input, dim, dtype=None):
    return input.log_softmax(dim, dtype)


def nll_loss(input, target, weight=None, reduction=1, ignore_index=-100):
    """(output, total_weight), as tensorplay/functional.py:496-497."""
    return _C.nll_loss(input, target, weight, reduction, ignore_index)


def nll_loss_backward(grad_output, input, target, weight=None, reduction=1, ignore_index=-100,
                      total_weight=None):
    return _C.nll_loss_backward(grad_output, input, target, weight, reduction, ignore_index, total_weight)


def _softmax_backward_data(grad_output, output, dim):
    return _C._softmax_backward_data(grad_output, output, dim)


def _log_softmax_backward_data(grad_output, output, dim):
    return _C._log_softmax_backward_data(grad_output, output, dim)


def topk_topp_sample(input, uniforms, k=50, temperature=1.0, top_p=1.0):
    """One token id per row of the last dim: top-k, then the top-p nucleus, drawn with `uniforms`."""
    return _C.topk_topp_sample(input, uniforms, k, temperature, top_p)


def sum_backward(grad, input, dim=(), keepdim=False):
    return _C.sum_backward(grad, input, list(dim), keepdim)


def mean_backward(grad, input, dim=(), keepdim=False):
    return _C.mean_backward(grad, input, list(dim), keepdim)


def var_backward(grad, input, dim=(), correction=1, keepdim=False):
    return _C.var_backward(grad, input, list(dim), correction, keepdim)


def std_backward(grad, input, result, dim=(), correction=1, keepdim=False):
    return _C.std_backward(grad, input, result, list(dim), correction, keepdim)


# ---- operators of a fine-tuning step -------------------------------------------
# Logits are [..., vocab] of float32, float16 or bfloat16, targets int64 [...].  A target
# equal to ignore_index is skipped: its row is not read, its log-probability and
# gradient are 0.  Any other target outside the vocabulary makes the row NaN.
def token_logprob(input, target, temperature=1.0, ignore_index=-100):
    """(logp, lse): log of softmax(input / temperature) at each row's target, and what
    the backward pass takes: each row's largest logit m and sum(exp((x - m) /
    temperature)) - 1, float32; log-sum-exp is m / temperature + log1p of the second."""
    return _C.token_logprob(input, target, temperature, ignore_index)


def token_logprob_backward(grad, input, target, lse, temperature=1.0, ignore_index=-100):
    """Gradient of the logits, given the log-probabilities' (float32)."""
    return _C.token_logprob_backward(grad, input, target, lse, temperature, ignore_index)


def policy_loss(input, target, old_logp, advantage, ref_logp=None, weight=None, clip_low=0.2, clip_high=0.2,
                kl_coef=0.0, temperature=1.0, ignore_index=-100):
    """(loss, logp, lse, coef) of the clipped policy loss with a KL term: with
    r = exp(logp - old_logp), d = ref_logp - logp and W = max(sum(weight), 1),

        1 / W sum weight (kl_coef (exp(d) - d - 1) - min(r A, clamp(r, 1 - clip_low, 1 + clip_high) A)).

    Per-token arguments are float32 in target's shape.  Tokens of weight 0 are not
    read; their logp is 0."""
    return _C.policy_loss(input, target, old_logp, advantage, ref_logp, weight, clip_low, clip_high, kl_coef,
                          temperature, ignore_index)


def policy_loss_backward(grad, coef, input, target, lse, temperature=1.0, ignore_index=-100):
    """Gradient of the logits, given the loss's (one float32 element)."""
    return _C.policy_loss_backward(grad, coef, input, target, lse, temperature, ignore_index)


def policy_loss_and_grad(input, target, old_logp, advantage, ref_logp=None, weight=None, clip_low=0.2, clip_high=0.2,
                         kl_coef=0.0, temperature=1.0, ignore_index=-100):
    """(loss, logp, gradient of the logits) of policy_loss in one call, for a loss gradient
    of 1.  A float16 gradient rounds what is below 3e-8 to 0 (a weight of 1 in 4096 rows
    times a softmax below 1.2e-4): a loss scale goes through policy_loss and
    policy_loss_backward.  Rows of more than 155648 logits in half precision, 77824 in
    float32, are read twice."""
    return _C.policy_loss_and_grad(input, target, old_logp, advantage, ref_logp, weight, clip_low, clip_high, kl_coef,
                                   temperature, ignore_index)


def preference_loss(input, target, offsets, ref_logp, beta=0.1, label_smoothing=0.0, ignore_index=-100):
    """(loss, reward, logp, lse, coef) over pairs of sequences packed along the rows of
    input [tokens, vocab]: sequence i is rows offsets[i] .. offsets[i + 1] - 1 (int64
    [2 pairs + 1]), the first half of the sequences are the preferred answers of the
    second half.  reward = beta (sum of logp - ref_logp), and the loss is the mean of
    -((1 - label_smoothing) log sigmoid(h) + label_smoothing log sigmoid(-h)) over the
    differences h of a pair's rewards; where h is infinite, a share of 0 has no part of it."""
    return _C.preference_loss(input, target, offsets, ref_logp, beta, label_smoothing, ignore_index)


def preference_loss_backward(grad, coef, input, target, lse, ignore_index=-100):
    """Gradient of the logits, given the loss's (one float32 element)."""
    return _C.preference_loss_backward(grad, coef, input, target, lse, ignore_index)


def dropout(input, p, seed, offset=0):
    """input / (1 - q) where kept, else 0, along the last dim's rows; q is p rounded to
    a multiple of 2^-16.  The mask is a function of (seed, offset, row, column) and is
    not stored: dropout_backward makes it again."""
    return _C.dropout(input, p, seed, offset)


def dropout_backward(grad, p, seed, offset=0):
    return _C.dropout_backward(grad, p, seed, offset)


def gated_residual_norm(input, residual, pre_weight, eps=1e-6, post_weight=None, gate=None, residual_scale=1.0,
                        p=0.0, seed=0, offset=0):
    """(out, y, rstd_post, rstd_pre) of the end of a block: with N(v, w) = v / sqrt(mean(v^2) + eps) * w,

        u = dropout(N(input, post_weight)),  out = residual_scale * residual + gate * u,  y = N(out, pre_weight).

    Without post_weight u is dropout(input), without gate the gate is 1.  gate is
    [cols] or [gates, cols], each gate for rows / gates neighbouring rows.  residual is
    of input's dtype or float32.  Without columns the roots are NaN."""
    return _C.gated_residual_norm(input, residual, pre_weight, eps, post_weight, gate, residual_scale, p, seed, offset)


def gated_residual_norm_backward(grad_y, grad_residual, input, out, rstd_post, rstd_pre, pre_weight, post_weight=None,
                                 gate=None, residual_scale=1.0, p=0.0, seed=0, offset=0):
    """Gradients of (input, residual, pre_weight, post_weight, gate), given those of y
    and out (grad_residual, None: 0); None for a weight that is None."""
    return _C.gated_residual_norm_backward(grad_y, grad_residual, input, out, rstd_post, rstd_pre, pre_weight,
                                           post_weight, gate, residual_scale, p, seed, offset)


_REDUCTION = {"none": 0, "mean": 1, "sum": 2}


def cross_entropy(input, target, weight=None, ignore_index=-100, reduction="mean"):
    """nll_loss(log_softmax(input, 1), target, ...), the composition of
    tensorplay/nn/functional.py:442-444 (forward only; its gradient is
    _log_softmax_backward_data(nll_loss_backward(...), log_probs, 1))."""
    out, _ = nll_loss(log_softmax(input, 1), target, weight, _REDUCTION[reduction], ignore_index)
    return out


class rocm:
    """ROCm runtime helpers (the counterpart of tensorplay.cuda for this backend)."""

    is_available = staticmethod(_C._rocm.is_available)
    device_count = staticmethod(_C._rocm.device_count)
    synchronize = staticmethod(_C._rocm.synchronize)
    set_stream = staticmethod(_C._rocm.set_stream)
    current_stream = staticmethod(_C._rocm.current_stream)
    empty_cache = staticmethod(_C._rocm.empty_cache)
    memory_stats = staticmethod(_C._rocm.memory_stats)
