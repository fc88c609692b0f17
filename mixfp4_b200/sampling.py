"""Drawing a token from logits: temperature, top-k, top-p and min-p, with random numbers that the caller brings.

    w_i    = exp((x_i - max x) / temperature)
    order  by value, largest first; equal values by index
    kept   the first top_k; of those the shortest run whose weights reach top_p of theirs; of those every w_i >= min_p
    token  the first index, in the vocabulary's order, at which the kept weights add up to more than uniform * their sum

The reference evaluates models and generates no tokens; the decoder harness (`llama_decode`) does.
"""

from __future__ import annotations

import torch

from . import _native as nat


def _setting(value, name: str, dtype: torch.dtype, rows: int, device, low: float, high: float):
    """(tensor or None, number): a checked number for all rows, or a tensor with one for each."""
    kind = type(value)
    if (kind is float and dtype is torch.float32 or kind is int) and low <= value <= high:
        return None, value
    if isinstance(value, torch.Tensor):
        if value.dtype != dtype:
            raise TypeError(f"{name} must be a number or a {dtype} tensor")
        if value.numel() != rows:
            raise ValueError(f"{name} must have one value for each of the {rows} rows, not {value.numel()}")
        if value.device != device:
            raise ValueError(f"{name} is on {value.device}, the logits on {device}")
        return value.contiguous(), 0
    if isinstance(value, bool) or not isinstance(value, int if dtype == torch.int32 else (int, float)):
        raise TypeError(f"{name} must be a number or a {dtype} tensor")
    if not low <= value <= high:
        raise ValueError(f"{name}={value} is not in [{low}, {high}]")
    return None, value


def sample_logits(logits: torch.Tensor, uniform: torch.Tensor, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
                  return_logprob: bool = False) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Tokens int64 [...] for logits [..., V] (bf16, f16 or fp32) and random numbers `uniform` fp32 [...] in [0, 1).

    temperature, top_k, top_p, min_p: a number, or a tensor with one value for each row (fp32; top_k int32) on the logits'
    device.  temperature 0 takes the first of the largest logits; top_k <= 0 or >= V, top_p 1 and min_p 0 filter nothing;
    top_p 0 keeps the largest alone.  Tensor values are not read by the host: a temperature that is not above zero counts
    as 0, a top_p or min_p outside [0, 1] as the nearer end, a uniform outside [0, 1) likewise; NaN as no filter, uniform NaN as 0.
    A logit of -inf or NaN is never chosen; +inf takes all the weight.  A row without a logit above -inf gives the token -1.
    return_logprob: also the natural logarithm of the token's share of the kept weights, fp32 [...] (-inf beside -1).

    Weights are integers, multiples of 2^-44 of the row's largest: results do not depend on the order of sums, and a token
    below half of that is never chosen.  One launch, no workspace; V up to `mixfp4_sample_max_vocab()` (524160)."""
    nat.require_cuda(logits, "logits")
    if logits.dtype not in nat.DTYPE_CODE:
        raise TypeError("logits must be bfloat16, float16 or float32")
    if logits.ndim == 0 or logits.shape[-1] == 0:
        raise ValueError("logits must have at least one column")
    if uniform.dtype != torch.float32:
        raise TypeError("uniform must be float32")
    device, vocab, lead = logits.device, logits.shape[-1], logits.shape[:-1]
    x = logits if logits.ndim == 2 else logits.reshape(-1, vocab)
    rows = x.shape[0]
    if uniform.numel() != rows:
        raise ValueError(f"uniform must have one number for each of the {rows} rows, not {uniform.numel()}")
    if uniform.device != device:
        raise ValueError(f"uniform is on {uniform.device}, the logits on {device}")
    t, t_all = _setting(temperature, "temperature", torch.float32, rows, device, 0.0, 3.0e38)
    k, k_all = _setting(top_k, "top_k", torch.int32, rows, device, -(2 ** 31), 2 ** 31 - 1)
    p, p_all = _setting(top_p, "top_p", torch.float32, rows, device, 0.0, 1.0)
    f, f_all = _setting(min_p, "min_p", torch.float32, rows, device, 0.0, 1.0)
    token = torch.empty_strided((rows,), (1,), dtype=torch.int64, device=device)      # a microsecond less than torch.empty
    logprob = torch.empty_strided((rows,), (1,), dtype=torch.float32, device=device) if return_logprob else None
    if rows:
        stride = x.stride(0)
        if x.stride(1) != 1 and vocab > 1 or rows > 1 and stride < vocab:
            x = x.contiguous()
            stride = vocab
        u = uniform.contiguous()
        with nat.on_device(device):
            st = nat.lib().mixfp4_sample(x.data_ptr(), nat.DTYPE_CODE[x.dtype], rows, vocab, max(stride, vocab), u.data_ptr(),
                                         nat.ptr(t), t_all, nat.ptr(k), k_all, nat.ptr(p), p_all, nat.ptr(f), f_all,
                                         token.data_ptr(), nat.ptr(logprob), nat.stream_ptr(device))
        nat.check("mixfp4_sample", st)
    if len(lead) != 1:
        token, logprob = token.reshape(lead), None if logprob is None else logprob.reshape(lead)
    return (token, logprob) if return_logprob else token
