"""rapid_sampling_b200 -- B200 (sm_100a) drop-in for the reference sampler's torch extension.

Exports the reference module's three functions (``sampling.cpp:5-9``) with the same names and
positional order::

    states = setup_rand(seed, B)
    ids = batch_sampling_temperature_topk_topp(logits, states, temperature, top_k, top_p)
    ids = batch_sampling_repetition_temperature_topk_topp(logits, penalties, states, presence_penalty,
                                                          repetition_penalty, penalty_decay,
                                                          temperature, top_k, top_p)

The functions live in a compiled PyTorch extension built in-tree by ``rapid_sampling_b200._build``.
There is no CPU or eager fallback: importing the functions without the built extension raises.
"""
import importlib
import os

_HERE = os.path.dirname(os.path.abspath(__file__))
_ext = None


def _load_ext():
    global _ext
    if _ext is None:
        import torch  # noqa: F401  libtorch must be loaded before the extension
        try:
            _ext = importlib.import_module("rapid_sampling_b200._rs_torch")
        except ImportError as e:
            raise ImportError("rapid_sampling_b200: the compiled extension is missing (%s). Build it with "
                              "`python -m rapid_sampling_b200._build`; there is no CPU fallback." % e) from e
    return _ext


def setup_rand(seed, B):
    return _load_ext().setup_rand(seed, B)


def batch_sampling_temperature_topk_topp(logits, states, temperature, top_k, top_p):
    return _load_ext().batch_sampling_temperature_topk_topp(logits, states, temperature, top_k, top_p)


def batch_sampling_repetition_temperature_topk_topp(logits, penalties, states, presence_penalty, repetition_penalty,
                                                    penalty_decay, temperature, top_k, top_p):
    return _load_ext().batch_sampling_repetition_temperature_topk_topp(
        logits, penalties, states, presence_penalty, repetition_penalty, penalty_decay, temperature, top_k, top_p)


def batch_sampling_temperature_topk_topp_any(logits, states, temperature, top_k, top_p):
    """Same call for fp32, fp16 or bf16 logits (the reference accepts fp32 only, sampling.cu:976). 16-bit logits are
    read directly and widened exactly, so the ids equal those of the fp32 call on ``logits.float()``."""
    return _load_ext().batch_sampling_temperature_topk_topp_any(logits, states, temperature, top_k, top_p)


def batch_sampling_repetition_temperature_topk_topp_any(logits, penalties, states, presence_penalty, repetition_penalty,
                                                        penalty_decay, temperature, top_k, top_p):
    return _load_ext().batch_sampling_repetition_temperature_topk_topp_any(
        logits, penalties, states, presence_penalty, repetition_penalty, penalty_decay, temperature, top_k, top_p)


def batch_sampling_rows(logits, states, temperature=None, top_k=None, top_p=None, penalties=None, presence_penalty=0.0,
                        repetition_penalty=0.0, penalty_decay=0.0, return_prob=False):
    """Per-row parameters: `temperature` (float32), `top_k` (int32) and `top_p` (float32) are CUDA tensors of B values, or
    None for the neutral value in every row.  Row b is sampled exactly as a one-row call of the functions above with its
    values would sample it.  With `return_prob` the result is (ids, probability of each id under the full softmax, kept
    probability mass).  The reference takes scalars only (sampling.cpp:2-3)."""
    return _load_ext().batch_sampling_rows(logits, states, temperature, top_k, top_p, penalties, presence_penalty,
                                           repetition_penalty, penalty_decay, return_prob)


def batch_token_logprobs(logits, tokens, temperature=1.0):
    """Log probability of one given token per row, and the row's entropy, under softmax(logits / temperature): float32
    tensors of the tokens' shape.  Differentiable with respect to the logits (both results, first order, in reverse mode:
    second derivatives and forward-mode tangents are refused).

    logits: float32, float16 or bfloat16, (V,), (B, V) or (B, T, V), every position a row; any strides but along V, and any
    V up to 1048576.  tokens: int32 or int64, the logits' shape without V.  temperature: a number, or a float32 CUDA tensor
    of one value, one per row, or one per sequence; not differentiated.

    A negative token marks a position that is not scored (padding): 0, 0 and no gradient, whatever its logits hold.
    Unlike the sampling calls, nothing is replaced: -inf masks a token; a row of nothing but -inf has log probability -inf,
    entropy 0 and gradient 0; NaN or +inf makes its row NaN.  A token >= V gives NaN and no gradient, a temperature outside
    [0.001, 1000] in a tensor counts as 1, and either raises ValueError from the next call on the device."""
    if hasattr(temperature, "is_cuda"):
        return _load_ext().token_logprobs(logits, tokens, 1.0, temperature)
    return _load_ext().token_logprobs(logits, tokens, float(temperature), None)


def batch_top_logprobs(logits, top_n, tokens=None, temperature=1.0):
    """(log probabilities, ranks, entropies, top log probabilities, top ids): what `batch_token_logprobs` computes, the
    tokens' ranks, and the `top_n` (at most 64) most probable tokens of every row in falling order, equal logits by rising
    id.  A token's rank (int32, from 1) is its place in that order.  Without tokens the first two are None.

    Slots behind the last token that a mask of -inf leaves hold -inf and id -1; so do all slots of a position that is not
    scored (negative token; rank 0).  Rows with NaN or +inf: NaN, id -1, rank 0.  Not differentiable."""
    if hasattr(temperature, "is_cuda"):
        return _load_ext().top_logprobs(logits, top_n, tokens, 1.0, temperature)
    return _load_ext().top_logprobs(logits, top_n, tokens, float(temperature), None)


def lm_head_quantize(weight):
    """(codes, scales) of an lm_head's weights (V, K), float32, float16 or bfloat16, K a multiple of 16: float8_e4m3fn codes
    (V, K) and float32 scales (ceil(V / 128), ceil(K / 128)), one for each block of 128 x 128:
    scale = max(amax / 448, 2^-126), code = the value nearest to weight / scale."""
    return _load_ext().lm_head_quantize(weight)


def lm_head_logits(hidden, codes, scales, dtype=None, out=None):
    """Logits (..., V) = hidden (..., K) times the weights that `codes` and `scales` stand for (`lm_head_quantize`, or any
    e4m3 checkpoint with a float32 scale for each block of 128 x 128).  The hidden states (float32, float16 or bfloat16) are
    quantized within the call, a scale for each row's 128 columns; sums are float32.  The result has `dtype` (float32,
    float16 or bfloat16; float32 unless `out` says otherwise) and goes to `out` where given, whose rows may lie apart.
    Rows of hidden and out lie at equal distances.  Not differentiable."""
    import torch
    if dtype is None:
        dtype = torch.float32 if out is None else out.dtype
    return _load_ext().lm_head_logits(hidden, codes, scales, dtype, out)


def kernel_launch_count():
    return _load_ext().kernel_launch_count()


def device_status():
    """Synchronises the current stream and returns the device status word of this device (0 = ok, else a negative
    RS_ERR_* code such as "a bounded on-chip wait gave up"), clearing it.  Sampling calls check a host mirror of the
    word by themselves and raise on the NEXT call; this is the explicit, synchronising form."""
    return _load_ext().device_status()


def release_workspaces():
    """Drops the per-(device, stream) scratch buffers the sampling calls keep between calls."""
    return _load_ext().release_workspaces()


__all__ = ["setup_rand", "batch_sampling_temperature_topk_topp", "batch_sampling_repetition_temperature_topk_topp",
           "batch_sampling_temperature_topk_topp_any", "batch_sampling_repetition_temperature_topk_topp_any", "batch_sampling_rows",
           "batch_token_logprobs", "batch_top_logprobs", "lm_head_quantize", "lm_head_logits",
           "kernel_launch_count", "device_status", "release_workspaces"]
