"""What surrounds a sampling call, as cases whose time matters: the lm_head that makes the logits, and the log
probabilities of what was sampled from them.

`listed()` names twelve cases and says what each stands for, `draw(rng)` gives further ones from the same ranges,
`prepare(case, seed)` makes what a program has on the GPU before the call, `run(state)` is one call, `work(case)` the bytes
and operations it cannot do without, and `exact(case, seed)` the same results in 64 bits.  With `own` set, `run` calls the
package; without it, it computes the same from elementary tensor operations.

A case is a dict:

  op       "score"     batch_token_logprobs: log probability of each position's token, and the entropy
           "train"     the same with its backward pass: log probabilities, entropies and the gradient of the logits
           "top"       batch_top_logprobs: the token's log probability and rank, the entropy and the top_n alternatives
           "head"      lm_head_logits: hidden states times an fp8 head with a scale per block of 128
           "quantize"  lm_head_quantize: a head's weights to fp8 codes and scales
  B, T, V  sequences, positions of each, vocabulary ("score", "train", "top")
  M, K, V  tokens, width of the hidden states, vocabulary ("head"); K, V for "quantize"
  dtype    of the logits, of the head's output, or of the weights
  shifted  "score": the logits are all but the last position of longer sequences, a view that is not contiguous
  padded   sequences of different length; positions behind a sequence's end have token -1
  masked   a share of the ids is set to -inf in every row, as constrained decoding does; in the first row, all of them
  rowwise  a temperature per position, in a tensor
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
BLOCK = 128
E4M3_MAX = 448.0
SMALLEST_SCALE = 2.0 ** -126

# ranges of draw(): logits in one call, and the head's multiplications, stay within the largest listed case's
SCORE_MAX = 8 * 511 * 151936
TRAIN_MAX = 4 * 512 * 151936
TOP_MAX = 1024 * 100256
HEAD_MAX = 2048 * 4096 * 65536
WEIGHTS_MAX = 151936 * 4096


def _logprobs(name, op, B, T, V, dtype, **more):
    c = dict(name=name, op=op, B=B, T=T, V=V, dtype=dtype, temperature=1.0, rowwise=False, padded=False, masked=False)
    if op == "score":
        c["shifted"] = False
    if op == "top":
        c["top_n"] = 20
    c.update(more)
    return c


def _head(name, M, K, V, dtype):
    return dict(name=name, op="head", M=M, K=K, V=V, dtype=dtype)


def listed():
    return [
        # one position of one stream: the latency of a call
        _logprobs("score_b1", "score", 1, 1, 32768, "f32"),
        # prompts scored under the model: every position but the last predicts its successor
        _logprobs("score_prompts", "score", 8, 511, 151936, "bf16", shifted=True),
        # a small policy-gradient step over an odd vocabulary in half precision
        _logprobs("train_small", "train", 2, 61, 50303, "f16", temperature=0.8),
        # a training step on rollouts of different lengths: logits, entropy bonus, gradient
        _logprobs("train_rollouts", "train", 4, 512, 151936, "bf16", padded=True),
        # logprobs of one chat stream
        _logprobs("top_b1", "top", 1, 1, 151936, "f32", top_n=20, temperature=0.7),
        # batched serving with logprobs on, every request with its own temperature
        _logprobs("top_serving", "top", 64, 1, 151936, "bf16", top_n=5, rowwise=True),
        # logprobs of a long prompt under a mask of allowed ids
        _logprobs("top_prompt", "top", 1, 1024, 100256, "f32", top_n=20, masked=True),
        # the head of one decoding stream, and of batched serving: the weights' bytes
        _head("head_b1", 1, 4096, 151936, "f32"),
        _head("head_serving", 64, 4096, 151936, "f32"),
        # the head over all positions of a prompt: arithmetic
        _head("head_prompt", 2048, 4096, 65536, "bf16"),
        # weights brought to fp8: a small head, and a large one after an update of the weights
        dict(name="quantize_small", op="quantize", K=1040, V=32768, dtype="bf16"),
        dict(name="quantize_large", op="quantize", K=4096, V=151936, dtype="bf16"),
    ]


def _log_uniform(rng, lo, hi):
    return int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))


def draw(rng):
    op = rng.choices(["score", "train", "top", "head", "quantize"], [3, 3, 3, 3, 1])[0]
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "quantize":
        K = 16 * _log_uniform(rng, 8, 512)
        return dict(op=op, K=K, V=_log_uniform(rng, 256, min(262144, WEIGHTS_MAX // K)), dtype=dtype)
    if op == "head":
        K = 16 * _log_uniform(rng, 32, 512)
        V = _log_uniform(rng, 1000, min(262144, WEIGHTS_MAX // K))
        return dict(op=op, M=_log_uniform(rng, 1, min(2048, HEAD_MAX // (K * V))), K=K, V=V, dtype=dtype)
    V = _log_uniform(rng, 256, 1048576)
    most = {"score": SCORE_MAX, "train": TRAIN_MAX, "top": TOP_MAX}[op]
    if dtype == "f32" and op != "top":
        most //= 2
    rows = _log_uniform(rng, 1, min(4096, most // V))
    B = rng.choice([1, 2, 3, 8]) if rows > 8 else rows
    c = _logprobs("", op, B, max(1, rows // B), V, dtype, temperature=rng.choice([1.0, 1.0, 0.6, 0.8, 1.3]),
                  rowwise=rng.random() < 0.3, padded=rng.random() < 0.3, masked=rng.random() < 0.2)
    if op == "score":
        c["shifted"] = rng.random() < 0.5
    if op == "top":
        c["top_n"] = rng.choice([1, 2, 5, 10, 20, 20, 32, 64])
    del c["name"]
    return c


def _lengths(case):
    """Scored positions of each sequence."""
    B, T = case["B"], case["T"]
    return [T - (17 * b + 5) % (T // 2 + 1) if case["padded"] else T for b in range(B)]


def _weights(rows, cols, dtype, gen):
    w = torch.randn((rows, cols), generator=gen, device="cuda", dtype=torch.float32)
    w *= 0.02
    w *= torch.exp(0.5 * torch.randn((1, cols), generator=gen, device="cuda"))     # channels of different strength
    return w.to(dtype)


def _fp8(x, rows):
    """Codes and scales of x, a scale for each block of `rows` by 128."""
    n, k = x.shape
    blocks = torch.nn.functional.pad(x.float(), (0, -k % BLOCK, 0, -n % rows))
    blocks = blocks.view(blocks.shape[0] // rows, rows, blocks.shape[1] // BLOCK, BLOCK)
    most = blocks.abs().amax(dim=(1, 3))
    scales = (most / torch.full_like(most, E4M3_MAX)).clamp_min(SMALLEST_SCALE)     # by a tensor: a true quotient
    codes = (blocks / scales[:, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return codes.reshape(blocks.shape[0] * rows, -1)[:n, :k].contiguous(), scales


def _wide(codes, scales, rows, dtype):
    """The values that codes and scales stand for."""
    s = scales.to(dtype).repeat_interleave(rows, 0)[:codes.shape[0]].repeat_interleave(BLOCK, 1)[:, :codes.shape[1]]
    return codes.to(dtype) * s


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, dtype, V = case["op"], DTYPES[case["dtype"]], case["V"]
    if op == "quantize":
        return {"case": case, "weight": _weights(V, case["K"], dtype, gen)}
    if op == "head":
        codes, scales = _fp8(_weights(V, case["K"], torch.bfloat16, gen), BLOCK)
        hidden = torch.randn((case["M"], case["K"]), generator=gen, device="cuda")
        hidden *= torch.exp(torch.randn((1, case["K"]), generator=gen, device="cuda"))
        return {"case": case, "hidden": hidden.bfloat16(), "codes": codes, "scales": scales}
    B, T = case["B"], case["T"]
    long = T + 1 if case.get("shifted") else T
    x = torch.randn((B, long, V), generator=gen, device="cuda")
    x *= 2.5
    ids = torch.randint(0, V, (B, long, 8), generator=gen, device="cuda")     # a confident model
    x.scatter_add_(-1, ids, 6 * torch.rand((B, long, 8), generator=gen, device="cuda"))
    if case["masked"]:
        x[:, :, torch.rand(V, generator=gen, device="cuda") < 0.4] = -math.inf
        x[0, 0] = -math.inf
    x = x.to(dtype)
    logits = x[:, :T]
    tokens = torch.randint(0, V, (B, T), generator=gen, device="cuda")
    likely = torch.rand((B, T), generator=gen, device="cuda") < 0.6
    tokens = torch.where(likely, logits.argmax(-1), tokens)
    if case["padded"]:
        lengths = torch.tensor(_lengths(case), device="cuda")
        tokens[torch.arange(T, device="cuda") >= lengths[:, None]] = -1
    s = {"case": case, "logits": logits, "tokens": tokens, "temperature": case["temperature"]}
    if case["rowwise"]:
        s["temperature"] = 0.5 + torch.rand((B, T), generator=gen, device="cuda")
    if op == "train":
        s["logits"].requires_grad_(True)
        s["g_logprobs"] = torch.randn((B, T), generator=gen, device="cuda")
        s["g_entropy"] = torch.full((B, T), 0.01, device="cuda")
    return s


def _plain_logprobs(x, tokens, temperature, dtype=torch.float32):
    """(z - max z, its exponential, its sum, log probabilities, entropies, scored) in `dtype`."""
    scored = tokens >= 0
    at = tokens.clamp_min(0)[..., None]
    t = temperature[..., None].to(dtype) if torch.is_tensor(temperature) else temperature
    z = x.detach().to(dtype) / t
    m = z.amax(-1, keepdim=True)
    empty = m == -math.inf
    z = z - torch.where(empty, torch.zeros_like(m), m)
    e = z.exp()
    s = e.sum(-1, keepdim=True)
    log_s = torch.where(empty, torch.zeros_like(s), s.log())
    mean = torch.where(e > 0, z * e, torch.zeros_like(e)).sum(-1, keepdim=True) / torch.where(empty, torch.ones_like(s), s)
    zero = torch.zeros_like(s[..., 0])
    logprobs = torch.where(scored, (z.gather(-1, at) - log_s)[..., 0], zero)
    entropy = torch.where(scored, (log_s - mean)[..., 0], zero)
    return z, e, s, log_s, logprobs, entropy, scored, empty, at, t


def _plain_train(x, tokens, temperature, g, h, dtype=torch.float32):
    z, e, s, log_s, logprobs, entropy, scored, empty, at, t = _plain_logprobs(x, tokens, temperature, dtype)
    g, h = g.to(dtype)[..., None], h.to(dtype)[..., None]
    p = e / torch.where(empty, torch.ones_like(s), s)
    grad = -g * p - h * torch.where(p > 0, p * (z - log_s + entropy[..., None]), torch.zeros_like(p))
    grad.scatter_add_(-1, at, g.expand_as(at))
    grad = torch.where(scored[..., None] & ~empty, grad / t, torch.zeros_like(grad))
    return logprobs, entropy, grad


def _plain_top(x, tokens, temperature, top_n, dtype=torch.float32):
    z, e, s, log_s, logprobs, entropy, scored, empty, at, t = _plain_logprobs(x, tokens, temperature, dtype)
    x = x.float()
    x_t = x.gather(-1, at)
    before = torch.arange(x.shape[-1], device=x.device) < at
    ranks = 1 + ((x > x_t) | ((x == x_t) & before)).sum(-1)
    ranks = torch.where(scored, ranks, torch.zeros_like(ranks)).int()
    order = x.sort(dim=-1, descending=True, stable=True)
    n = min(top_n, x.shape[-1])
    ids = order.indices[..., :n]
    there = (order.values[..., :n] > -math.inf) & scored[..., None]
    top = torch.where(there, z.gather(-1, ids) - log_s, torch.full_like(z[..., :n], -math.inf))
    ids = torch.where(there, ids, torch.full_like(ids, -1)).int()
    more = (0, top_n - n)
    return logprobs, ranks, entropy, torch.nn.functional.pad(top, more, value=-math.inf), torch.nn.functional.pad(ids, more, value=-1)


def _run_own(state):
    import rapid_sampling_b200 as sampler
    c, op = state["case"], state["case"]["op"]
    if op == "quantize":
        return sampler.lm_head_quantize(state["weight"])
    if op == "head":
        return sampler.lm_head_logits(state["hidden"], state["codes"], state["scales"], dtype=DTYPES[c["dtype"]])
    if op == "score":
        return sampler.batch_token_logprobs(state["logits"], state["tokens"], state["temperature"])
    if op == "top":
        return sampler.batch_top_logprobs(state["logits"], c["top_n"], state["tokens"], state["temperature"])
    logprobs, entropy = sampler.batch_token_logprobs(state["logits"], state["tokens"], state["temperature"])
    grad, = torch.autograd.grad((logprobs, entropy), state["logits"], (state["g_logprobs"], state["g_entropy"]))
    return logprobs.detach(), entropy.detach(), grad


def run(state):
    if own:
        return _run_own(state)
    c, op = state["case"], state["case"]["op"]
    if op == "quantize":
        return _fp8(state["weight"], BLOCK)
    if op == "head":
        a = _wide(*_fp8(state["hidden"], 1), 1, torch.float32)
        return (a @ _wide(state["codes"], state["scales"], BLOCK, torch.float32).t()).to(DTYPES[c["dtype"]])
    args = state["logits"], state["tokens"], state["temperature"]
    if op == "score":
        return _plain_logprobs(*args)[4:6]
    if op == "top":
        return _plain_top(*args, c["top_n"])
    logprobs, entropy, grad = _plain_train(*args, state["g_logprobs"], state["g_entropy"])
    return logprobs, entropy, grad.to(state["logits"].dtype)


def work(case):
    """Logits of the scored positions read once, and for the gradient written once (all positions: the padded ones' zeros
    too); tokens (8 bytes), temperatures and results.  Arithmetic per logit: scaling, exponential and the two sums (5); for
    the gradient the exponential again, both terms and the scaling (7); for the alternatives a comparison each with the
    list's last and with the token (2).  The head: its codes, scales and hidden states once, two operations a product."""
    op, V, size = case["op"], case["V"], SIZE[case["dtype"]]
    if op == "quantize":
        n = V * case["K"]
        return {"bytes": n * (size + 1) + 4 * -(-V // BLOCK) * -(-case["K"] // BLOCK), "flops": 3 * n}
    if op == "head":
        M, K = case["M"], case["K"]
        return {"bytes": V * K + 4 * -(-V // BLOCK) * -(-K // BLOCK) + 2 * M * K + size * M * V, "flops": 2 * M * K * V}
    rows, scored = case["B"] * case["T"], sum(_lengths(case))
    total = scored * V * size + rows * (8 + 8 + (4 if case["rowwise"] else 0))
    flops = 5 * scored * V
    if op == "train":
        return {"bytes": total + rows * V * size + scored * V * size + rows * 8, "flops": flops + 7 * scored * V}
    if op == "top":
        return {"bytes": total + rows * (4 + 8 * case["top_n"]), "flops": flops + 2 * scored * V}
    return {"bytes": total, "flops": flops}


def _nearest_e4m3(v):
    """v in 64 bits to the nearest value with 3 bits behind the leading one, ties to even; spacing 2^-9 below 2^-6."""
    exponent = torch.frexp(v).exponent - 1
    step = torch.ldexp(torch.ones_like(v), exponent.clamp_min(-6) - 3)
    return (torch.round(v / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def _exact_fp8(x, rows):
    """(codes as values, scales) in 64 bits.  A code is by definition the one nearest to the value's quotient by its block's
    scale, quotient and scale both held in 32 bits: 16-bit weights lie on borders between two codes so often that it matters."""
    n, k = x.shape
    codes = torch.empty((n, k), dtype=torch.float64, device=x.device)
    scales = torch.empty((-(-n // rows), -(-k // BLOCK)), dtype=torch.float64, device=x.device)
    for j in range(scales.shape[1]):
        v = x[:, j * BLOCK:(j + 1) * BLOCK].double()
        most = torch.nn.functional.pad(v.abs().amax(1), (0, -n % rows)).view(-1, rows).amax(1)
        scales[:, j] = (most / E4M3_MAX).clamp_min(SMALLEST_SCALE)
        held = scales[:, j].float().double().repeat_interleave(rows)[:n]
        codes[:, j * BLOCK:(j + 1) * BLOCK] = _nearest_e4m3((v / held[:, None]).float().double())
    return codes, scales


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        return _exact_fp8(s["weight"], BLOCK)
    if op == "head":
        if case["M"] * case["K"] * case["V"] > 1.5e14:
            return None
        codes, scales = _exact_fp8(s["hidden"], 1)
        a = codes * scales.float().double().repeat_interleave(BLOCK, 1)[:, :case["K"]]
        out = torch.empty((case["M"], case["V"]), dtype=torch.float64, device="cuda")
        for at in range(0, case["V"], 64 * BLOCK):
            w = s["codes"][at:at + 64 * BLOCK].double()
            w *= s["scales"][at // BLOCK:at // BLOCK + 64].double().repeat_interleave(BLOCK, 0)[:w.shape[0]].repeat_interleave(
                BLOCK, 1)[:, :case["K"]]
            out[:, at:at + w.shape[0]] = a @ w.t()
        return out
    B, T, V = case["B"], case["T"], case["V"]
    logprobs = torch.zeros((B, T), dtype=torch.float64, device="cuda")
    entropy = torch.zeros_like(logprobs)
    grad = torch.zeros((B, T, V), dtype=torch.float64, device="cuda") if op == "train" else None
    top = torch.full((B, T, case["top_n"]), -math.inf, dtype=torch.float64, device="cuda") if op == "top" else None
    many = max(1, (1 << 25) // V)
    for b in range(B):
        for r in range(0, T, many):
            at = slice(r, r + many)
            t = s["tokens"][b, at]
            heat = s["temperature"][b, at, None].double() if case["rowwise"] else case["temperature"]
            z = s["logits"].detach()[b, at].double() / heat
            total = torch.logsumexp(z, -1, keepdim=True)
            use = (t >= 0)[:, None] & (total > -math.inf)
            logp = z - total
            p = torch.where(use, logp.exp(), 0.0)
            logp_p = torch.where(p > 0, logp * p, 0.0)
            H = -logp_p.sum(-1, keepdim=True)
            lp_t = torch.where(total > -math.inf, logp, -math.inf).gather(-1, t.clamp_min(0)[:, None])
            logprobs[b, at] = torch.where(t >= 0, lp_t[:, 0], 0.0)
            entropy[b, at] = H[:, 0]
            if op == "top":
                n = min(case["top_n"], V)
                top[b, at, :n] = torch.where(use, torch.where(use, logp, -math.inf).topk(n, -1).values, -math.inf)
            if op == "train":
                g, h = s["g_logprobs"][b, at, None].double(), s["g_entropy"][b, at, None].double()
                d = -g * p - h * (logp_p + H * p)
                d.scatter_add_(-1, t.clamp_min(0)[:, None], g)
                grad[b, at] = torch.where(use, d / heat, 0.0)
    if op == "score":
        return logprobs, entropy
    if op == "top":
        return logprobs, None, entropy, top, None
    return logprobs, entropy, grad
