"""Log probabilities of given tokens with their gradient, entropy, rank and alternatives (no counterpart in the reference)."""
import torch
from torch.autograd.function import once_differentiable

from . import _load_ext


def split_temperature(temperature):
    """(scalar, tensor or None) as the extension takes them."""
    if isinstance(temperature, torch.Tensor):
        if temperature.requires_grad:
            raise ValueError("the temperature is not differentiated: pass a tensor that does not require a gradient")
        return 1.0, temperature
    return float(temperature), None


class TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, scalar, rows):
        logprobs, entropy, stats = _load_ext().token_logprobs(logits, tokens, scalar, rows, True)
        ctx.set_materialize_grads(False)
        ctx.scalar = scalar
        ctx.save_for_backward(logits, tokens, rows, entropy, stats)
        return logprobs, entropy

    @staticmethod
    @once_differentiable
    def backward(ctx, g_logprobs, g_entropy):
        logits, tokens, rows, entropy, stats = ctx.saved_tensors
        if g_logprobs is None and g_entropy is None:
            return None, None, None, None
        return _load_ext().token_logprobs_backward(logits, tokens, ctx.scalar, rows, entropy, stats, g_logprobs, g_entropy), None, None, None


def token_logprobs(logits, tokens, temperature):
    scalar, rows = split_temperature(temperature)
    if logits.requires_grad and torch.is_grad_enabled():
        return TokenLogprobs.apply(logits, tokens, scalar, rows)
    return _load_ext().token_logprobs(logits, tokens, scalar, rows, False)[:2]


def top_logprobs(logits, top_n, tokens, temperature):
    scalar, rows = split_temperature(temperature)
    return _load_ext().top_logprobs(logits, top_n, tokens, scalar, rows)
