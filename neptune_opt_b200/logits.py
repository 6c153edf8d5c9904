"""Penalties, biases, temperature and a grammar's mask on the logits of a batch (nb200_penalize_logits).

Per row and token, in this order, in fp32 and rounded once:

    x = x > 0 ? x / repetition : x * repetition    where the token is in the row's history
    x = x - frequency * count - presence           where it is among the history's output, count times
    x = x + bias                                   for the row's biased tokens (one that is named twice adds)
    x = x / temperature
    x = -inf                                       where the mask's bit is 0

logits is [rows, vocab] in float32, bfloat16 or float16. tokens [rows, history] int32/int64 holds each row's
tokens: the first token_lens (default: all), of which the first prompt_lens (default: none) are its prompt and
the others its output. repetition, presence, frequency and temperature are float32 [rows], each optional; the
caller keeps repetition and temperature positive (for one below 2^-128, whose reciprocal fp32 does not hold, its
largest value stands in, so that 0 stays 0). bias_index [rows, n] int32/int64 and bias_value [rows, n]
float32, n at most 1024. A token or index outside [0, vocab) is skipped. allowed [rows, ceil(vocab / 32)]
int32 has bit v % 32 of word v // 32 for token v; a row may allow nothing. One mask, history or bias list for
all rows may be passed expanded. The reference has no such operator; `softmax`, `log_softmax` and the folds take
its result.

No gradient: one that is asked for is refused (NotImplementedError). Errors follow the backend's convention:
TypeError for dtypes, ValueError for devices and shapes, NotImplementedError past the kernels' biases per row.
"""
from __future__ import annotations

from neptune_opt_b200.torch_op import run_cxx

MAX_BIASES = 1024


def validate_logits_inputs(logits, tokens, token_lens, prompt_lens, repetition, presence, frequency, bias_index,
                           bias_value, allowed, temperature):
    """Metadata-only contract."""
    import torch

    what = "penalize_logits"
    if not isinstance(logits, torch.Tensor) or logits.layout != torch.strided:
        raise TypeError(f"{what}: logits must be a strided tensor")
    if logits.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise TypeError(f"{what}: logits must be float32/bfloat16/float16, got {logits.dtype}")
    index, i32, f32 = (torch.int32, torch.int64), (torch.int32,), (torch.float32,)
    given = (("tokens", tokens, index, 2), ("token_lens", token_lens, i32, 1), ("prompt_lens", prompt_lens, i32, 1),
             ("repetition", repetition, f32, 1), ("presence", presence, f32, 1), ("frequency", frequency, f32, 1),
             ("bias_index", bias_index, index, 2), ("bias_value", bias_value, f32, 2), ("allowed", allowed, i32, 2),
             ("temperature", temperature, f32, 1))
    for name, t, dtypes, _ in given:
        if t is not None and (not isinstance(t, torch.Tensor) or t.layout != torch.strided or t.dtype not in dtypes):
            raise TypeError(f"{what}: {name} must be a strided tensor of {' or '.join(str(d) for d in dtypes)}")
    if logits.device.type not in ("cuda", "meta"):
        raise ValueError(f"{what}: inputs must be CUDA tensors, got {logits.device}")
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError(f"{what}: logits must be [rows, vocab], got {tuple(logits.shape)}")
    for name, t, _, dims in given:
        if t is not None and (t.dim() != dims or t.shape[0] != logits.shape[0] or t.device != logits.device):
            raise ValueError(f"{what}: {name} must be {'[rows]' if dims == 1 else '[rows, n]'} on the device of logits, "
                             f"got {tuple(t.shape)}")
    if tokens is None and any(t is not None for t in (token_lens, prompt_lens, repetition, presence, frequency)):
        raise ValueError(f"{what}: lengths or penalties without tokens")
    if (bias_index is None) != (bias_value is None) or (bias_index is not None and bias_index.shape != bias_value.shape):
        raise ValueError(f"{what}: bias_index and bias_value go together, of one shape")
    if allowed is not None and allowed.shape[1] != -(-logits.shape[1] // 32):
        raise ValueError(f"{what}: allowed must hold {-(-logits.shape[1] // 32)} words a row, got {allowed.shape[1]}")
    if bias_index is not None and bias_index.shape[1] > MAX_BIASES:
        raise NotImplementedError(f"{what}: {bias_index.shape[1]} biases per row exceed {MAX_BIASES}")


def penalize_logits(logits, tokens=None, token_lens=None, prompt_lens=None, *, repetition=None, presence=None,
                    frequency=None, bias_index=None, bias_value=None, allowed=None, temperature=None):
    """The logits a sampler takes: fresh, contiguous, in the dtype of `logits`."""
    contract = (logits, tokens, token_lens, prompt_lens, repetition, presence, frequency, bias_index, bias_value,
                allowed, temperature)
    return run_cxx("penalize_logits", logits, contract, validate_logits_inputs, *contract)
