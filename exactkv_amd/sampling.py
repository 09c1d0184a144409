"""The next token of each row of logits, drawn with given random numbers.

No counterpart in the reference, whose engine takes the largest logit (exactkv/engine.py:93-95). The draw is one
launch or four on the logits' GPU and its current stream; it waits for nothing, keeps nothing between calls and can be captured in a HIP
graph (with u, and settings given as tensors, rewritten between replays)."""
import functools

import torch

from . import _lib

_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
MAX_VOCAB = 1 << 19


@functools.lru_cache(maxsize=4096)
def _workspace(B, V):
    """Bytes of a call's workspace, which the sizes alone determine."""
    return _lib.load().exkv_sample_workspace(B, V)


def _setting(v, B, dtype, dev, what, kind):
    """(pointer or None, value) of a setting given as a number or as one entry per row."""
    if isinstance(v, torch.Tensor):
        if v.dtype is not dtype or v.shape != (B,) or v.get_device() != dev or not v.is_contiguous():
            raise ValueError(f"{what} must be a number or a contiguous {str(dtype)[6:]} [{B}] tensor on the logits' GPU")
        return v.data_ptr(), kind(0)
    try:
        if isinstance(v, (int, float)) and not isinstance(v, bool) and (kind is float or v == int(v)):
            return None, kind(v)
    except (OverflowError, ValueError):                # infinite or NaN where whole, whole past a float's range
        pass
    raise ValueError(f"{what} must be a number or a {str(dtype)[6:]} [{B}] tensor (got {v!r})")


def sample(logits, u, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, logprob=False):
    """One token a row: logits [B, V] (bf16, fp16 or fp32 on the GPU, V up to 2^19, rows contiguous, any row stride), u
    fp32 [B], uniform in [0, 1). With M a row's largest logit and w = exp((l - M) / temperature), its tokens are
    ordered by logit, equal ones by index; of them stay

        those with w >= min_p,
        of these the first top_k (0: all),
        of these the ones before whose weights add up to less than top_p of all (1: all; the first always stays),

    and the token is the first one with which the running sum of the weights passes u times their sum: u = 0 is the likeliest one.
    A temperature of 0 gives the largest logit (the first of equal ones) whatever u is. Each setting is a number, or a
    tensor with one entry per row (fp32; top_k int32), where values outside a range count as its nearest one. Returns int64 [B], and with logprob=True also fp32 [B], the
    logarithm of the probability with which each token was drawn.

    The same inputs give the same tokens: weights are made in fp64 and added up as whole multiples of 2^-43 of the largest;
    smaller ones than half of that are never drawn. A log-probability is off by at most 2^-25 and its own rounding, however
    unlikely its token. NaN and -infinity are never drawn; a row of nothing else gives token 0 with log-probability -infinity and sets an error bit
    (kernels.check_errors)."""
    dev = logits.get_device()
    if dev >= 0 and dev != _lib.current_device():
        with torch.cuda.device(dev):
            return sample(logits, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p, logprob=logprob)
    kind = _TYPES.get(logits.dtype)
    if kind is None or logits.dim() != 2 or dev < 0:
        raise ValueError("logits must be a bf16, fp16 or fp32 [rows, vocabulary] GPU tensor")
    B, V = logits.shape
    if not 1 <= V <= MAX_VOCAB:
        raise ValueError(f"sample takes 1 to {MAX_VOCAB} tokens (got {V})")
    if V > 1 and logits.stride(1) != 1:
        raise ValueError("logits: rows (the last axis) must be contiguous")
    if u.dtype is not torch.float32 or u.shape != (B,) or u.get_device() != dev or not u.is_contiguous():
        raise ValueError(f"u must be a contiguous fp32 [{B}] tensor on the logits' GPU")
    f32 = torch.float32
    tp, t = _setting(temperature, B, f32, dev, "temperature", float)
    kp, k = _setting(top_k, B, torch.int32, dev, "top_k", int)
    pp, p = _setting(top_p, B, f32, dev, "top_p", float)
    mp, m = _setting(min_p, B, f32, dev, "min_p", float)
    if not t >= 0 or not 0 <= k < 2 ** 31 or not 0 <= p <= 1 or not 0 <= m <= 1:
        raise ValueError(f"temperature and top_k must not be negative, top_p and min_p lie in [0, 1] (got {temperature!r}, "
                         f"{top_k!r}, {top_p!r}, {min_p!r})")
    token = torch.empty(B, dtype=torch.int64, device=logits.device)
    lp = torch.empty(B, dtype=f32, device=logits.device) if logprob else None
    need = _workspace(B, V)
    ws = torch.empty(need, dtype=torch.uint8, device=logits.device) if need else None
    _lib.call("exkv_sample", logits.data_ptr(), logits.stride(0) if B > 1 else V, kind, B, V, u.data_ptr(), tp, kp, pp, mp, t, k, p, m,
              token.data_ptr(), lp.data_ptr() if logprob else None, ws.data_ptr() if need else None, need,
              _lib.stream(dev))
    return (token, lp) if logprob else token


class Sampler:
    """sample() with its settings and a random generator: logits [B, V] -> tokens [B], as the engines' choose= takes it. The
    settings are numbers, or tensors with one entry for each row that is then asked for."""

    def __init__(self, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, generator=None):
        self.settings = dict(temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
        self.generator = generator

    def __call__(self, logits):
        u = torch.rand(logits.shape[0], generator=self.generator, device=logits.device)
        return sample(logits, u, **self.settings)
