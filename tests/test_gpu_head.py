"""GPU: the lm_head in 8-bit floating point against its definition in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def nearest_e4m3(v):
    exponent = torch.frexp(v).exponent - 1
    step = torch.ldexp(torch.ones_like(v), exponent.clamp_min(-6) - 3)
    return (torch.round(v / step) * step).clamp(-448.0, 448.0)


def quantized(x, rows):
    """(codes as float64 values, scales float32) of x (n, k), a scale for each block of rows x 128."""
    n, k = x.shape
    pad = torch.nn.functional.pad(x.double(), (0, -k % 128, 0, -n % rows))
    b = pad.view(pad.shape[0] // rows, rows, pad.shape[1] // 128, 128)
    most = b.abs().amax(dim=(1, 3))
    scales = (most / 448.0).clamp_min(2.0 ** -126).float()        # the 64-bit quotient of 32-bit values rounds as the 32-bit one
    codes = nearest_e4m3((b / scales.double()[:, None, :, None]).float().double())
    return codes.reshape(pad.shape)[:n, :k], scales


def wide(codes, scales, rows):
    return codes.double() * scales.double().repeat_interleave(rows, 0)[:codes.shape[0]].repeat_interleave(128, 1)[:, :codes.shape[1]]


def make(rows, K, dtype, seed, sigma=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, K, generator=gen, device="cuda") * sigma
    return (x * torch.exp(torch.randn(1, K, generator=gen, device="cuda"))).to(DT[dtype])


def check(hidden, codes, scales, out):
    """Products are exact.  A block's sum of 128 takes at most 128 additions in the tensor core, each of which may cut what
    lies below the last place of the larger operand (2^-23 of the partial sum), the sum over the blocks one rounding of
    2^-24 for the scales, one for the product with them fused into the addition; all relative to the sum of magnitudes.  Then
    half a step of the output's type."""
    a = wide(*quantized(hidden.reshape(-1, hidden.shape[-1]), 1), 1)
    w = wide(codes, scales, 128)
    want = a @ w.t()
    size = a.abs() @ w.abs().t()
    blocks = scales.shape[1]
    bound = (128 + blocks + 2) * 2.0 ** -23 * size
    got = out.reshape(-1, out.shape[-1]).double()
    half = torch.finfo(out.dtype).eps / 2
    limit = bound + half * (want.abs() + bound) + torch.finfo(out.dtype).smallest_normal * half * 2
    off = (got - want).abs()
    assert bool((off <= limit).all()), (float((off / limit).max()), float(off.max()))
    # as a whole: errors of single additions do not line up
    if out.dtype == torch.float32:
        assert float(off.norm() / want.norm()) < 2e-6


@pytest.mark.parametrize("V,K", [(128, 128), (1, 16), (130, 144), (1000, 1040), (257, 512)])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_weights_to_codes(V, K, dtype):
    import rapid_sampling_b200 as rs
    w = make(V, K, dtype, V + K, 0.02)
    if V > 128:
        w[128:, :128] = 0                                   # a block of nothing but zeros
    w[0, 1] = -0.0
    codes, scales = rs.lm_head_quantize(w)
    assert codes.dtype == torch.float8_e4m3fn and codes.shape == (V, K) and scales.shape == (-(-V // 128), -(-K // 128))
    want, want_scales = quantized(w, 128)
    assert torch.equal(scales, want_scales)
    assert torch.equal(codes.double(), want)


def test_weights_of_all_sizes():
    """Scales from the smallest to the largest, quotients on the borders between codes, rows at odd addresses."""
    import rapid_sampling_b200 as rs
    gen = torch.Generator(device="cuda").manual_seed(5)
    w = torch.randn(128 * 8, 384, generator=gen, device="cuda")
    for i, e in enumerate([-140, -126, -120, -80, -61, -40, 60, 115]):
        w[128 * i:128 * (i + 1)] *= 2.0 ** e
    w[5, :64] = torch.arange(64, device="cuda").float() * 2.0 ** -142        # subnormal
    codes, scales = rs.lm_head_quantize(w)
    want, want_scales = quantized(w, 128)
    assert torch.equal(scales, want_scales) and torch.equal(codes.double(), want)
    grid = (torch.arange(128 * 128, device="cuda").float() / 64).view(128, 128)    # 448 = 7 * 2^6: quotients that are borders
    grid[0, 0] = 448.0
    codes, scales = rs.lm_head_quantize(grid)
    want, want_scales = quantized(grid, 128)
    assert torch.equal(scales, want_scales) and torch.equal(codes.double(), want)
    odd = make(200, 161, "bf16", 6)[:, 1:]
    codes, scales = rs.lm_head_quantize(odd)
    want, want_scales = quantized(odd, 128)
    assert torch.equal(scales, want_scales) and torch.equal(codes.double(), want)


@pytest.mark.parametrize("M,K,V", [(1, 16, 1), (1, 128, 128), (3, 144, 200), (16, 256, 129), (17, 1024, 1000), (33, 1040, 777), (64, 512, 4096),
                                   (65, 384, 300), (128, 2048, 515), (129, 640, 1030), (200, 256, 999), (256, 512, 640), (257, 384, 515),
                                   (300, 1040, 50303), (1000, 512, 2000)])
def test_products(M, K, V):
    import rapid_sampling_b200 as rs
    hidden = make(M, K, "bf16", M)
    codes, scales = rs.lm_head_quantize(make(V, K, "bf16", V, 0.02))
    check(hidden, codes, scales, rs.lm_head_logits(hidden, codes, scales))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
def test_types(dtype, out):
    import rapid_sampling_b200 as rs
    codes, scales = rs.lm_head_quantize(make(1000, 528, "f32", 3, 0.02))
    for M in (5, 150):
        hidden = make(M, 528, dtype, 4)
        got = rs.lm_head_logits(hidden, codes, scales, dtype=DT[out])
        assert got.dtype == DT[out]
        check(hidden, codes, scales, got)


@pytest.mark.parametrize("spread", [4, 1])
def test_whole_numbers(spread):
    """Small whole numbers, for any error of layout to show.  A block's sum is exact: it stays below 448^2 + 127 * 21 < 2^18.
    With block scales of 2^-1 and 1 all four blocks' sum stays below 2^20 in steps of 2^-1, so it is exact too; with 2^-4 to
    2^3 it may need 27 bits, and each of the four additions may round by 2^-24 of a partial sum."""
    import rapid_sampling_b200 as rs
    gen = torch.Generator(device="cuda").manual_seed(8)
    M, K, V = 70, 400, 333
    hidden = torch.randint(-7, 8, (M, K), generator=gen, device="cuda").float()
    hidden[:, ::128] = 7 * 64.0                           # amax 448: scale 1
    w = torch.randint(-3, 4, (V, K), generator=gen, device="cuda").float()
    w[::128, ::128] = 448.0
    codes, scales = rs.lm_head_quantize(w)
    assert bool((scales == 1).all())
    scales = scales * 2.0 ** torch.randint(-spread, max(spread, 1), scales.shape, generator=gen, device="cuda").float()
    got = rs.lm_head_logits(hidden, codes, scales).double()
    values = wide(codes, scales, 128)
    want = hidden.double() @ values.t()
    if spread == 1:
        assert torch.equal(got, want)
    partial = sum((hidden[:, k:k + 128].double() @ values[:, k:k + 128].t()).abs() for k in range(0, K, 128))
    assert bool(((got - want).abs() <= 4 * 2.0 ** -24 * partial).all())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_many_tokens_into_rows_of_any_alignment(dtype):
    """Results stored in boxes, in vectors and one by one; nothing beside them is touched."""
    import rapid_sampling_b200 as rs
    K, V, M = 256, 1000, 333
    codes, scales = rs.lm_head_quantize(make(V, K, "bf16", 1, 0.02))
    hidden = make(M, K, "bf16", 2)
    got = rs.lm_head_logits(hidden, codes, scales, dtype=DT[dtype])
    check(hidden, codes, scales, got)
    for pad, first in ((24, 8), (24, 1), (9, 0), (9, 3)):
        buf = torch.full((M, V + pad), 7.0, device="cuda", dtype=DT[dtype])
        rs.lm_head_logits(hidden, codes, scales, out=buf[:, first:first + V])
        assert torch.equal(buf[:, first:first + V], got), (pad, first)
        assert bool((buf[:, :first] == 7).all()) and bool((buf[:, first + V:] == 7).all())


def test_shapes_strides_and_out():
    import rapid_sampling_b200 as rs
    K, V = 256, 300
    codes, scales = rs.lm_head_quantize(make(V, K, "bf16", 1, 0.02))
    big = make(12, K, "bf16", 2).view(3, 4, K)
    got = rs.lm_head_logits(big, codes, scales)
    assert got.shape == (3, 4, V)
    check(big, codes, scales, got)
    last = big[:, -1]                                       # rows 4 K apart
    assert torch.equal(rs.lm_head_logits(last, codes, scales), got[:, -1])
    assert torch.equal(rs.lm_head_logits(big[1, 2], codes, scales), got[1, 2])
    same = big[:1, 0].expand(5, K)
    assert torch.equal(rs.lm_head_logits(same, codes, scales), got[:1, 0].expand(5, V))
    odd = make(6, K + 3, "f16", 3)[:, 3:]                   # rows at odd addresses
    check(odd, codes, scales, rs.lm_head_logits(odd, codes, scales))
    buf = torch.full((12, V + 5), 7.0, device="cuda")
    ret = rs.lm_head_logits(big.view(12, K), codes, scales, out=buf[:, 2:2 + V])
    assert ret.data_ptr() == buf[:, 2:].data_ptr() and torch.equal(buf[:, 2:2 + V], got.view(12, V))
    assert bool((buf[:, :2] == 7).all()) and bool((buf[:, 2 + V:] == 7).all())
    assert rs.lm_head_logits(big[:0], codes, scales).shape == (0, 4, V)


def test_not_finite():
    import rapid_sampling_b200 as rs
    K, V = 256, 260
    w = make(V, K, "f32", 1, 0.02)
    codes, scales = rs.lm_head_quantize(w)
    hidden = make(4, K, "f32", 2)
    clean = rs.lm_head_logits(hidden, codes, scales)
    hidden[1, 200] = math.nan
    hidden[2, 3] = math.inf
    got = rs.lm_head_logits(hidden, codes, scales)
    assert torch.equal(got[[0, 3]], clean[[0, 3]]) and torch.isnan(got[1:3]).all()
    w[200, 7] = math.nan
    codes, scales = rs.lm_head_quantize(w)
    got = rs.lm_head_logits(hidden[:1], codes, scales)
    assert torch.isnan(got[:, 128:256]).all() and torch.equal(got[:, :128], clean[:1, :128]) and torch.equal(got[:, 256:], clean[:1, 256:])


def test_refusals():
    import rapid_sampling_b200 as rs
    K, V = 256, 300
    w = make(V, K, "bf16", 1, 0.02)
    codes, scales = rs.lm_head_quantize(w)
    h = make(4, K, "bf16", 2)
    for bad in (lambda: rs.lm_head_quantize(w.double()), lambda: rs.lm_head_quantize(w.cpu()), lambda: rs.lm_head_quantize(w[0]),
                lambda: rs.lm_head_quantize(w[:, :250]), lambda: rs.lm_head_quantize(w.t()), lambda: rs.lm_head_quantize(w[:0]),
                lambda: rs.lm_head_logits(h.double(), codes, scales), lambda: rs.lm_head_logits(h.cpu(), codes, scales),
                lambda: rs.lm_head_logits(h[:, :128], codes, scales), lambda: rs.lm_head_logits(h, codes.float(), scales),
                lambda: rs.lm_head_logits(h, codes[:, :128], scales), lambda: rs.lm_head_logits(h, codes, scales[:2]),
                lambda: rs.lm_head_logits(h, codes, scales.double()), lambda: rs.lm_head_logits(h, codes, scales, dtype=torch.float64),
                lambda: rs.lm_head_logits(h, codes, scales, dtype="float32"),
                lambda: rs.lm_head_logits(h, codes, scales, out=torch.empty(4, V - 1, device="cuda")),
                lambda: rs.lm_head_logits(h, codes, scales, out=torch.empty(1, V, device="cuda").expand(4, V)),
                lambda: rs.lm_head_logits(h, codes, scales, dtype=torch.float16, out=torch.empty(4, V, device="cuda")),
                lambda: rs.lm_head_logits(torch.stack([h, h, h])[::2, 1:], codes, scales)):
        with pytest.raises(ValueError):
            bad()


def test_capture_and_two_streams():
    import rapid_sampling_b200 as rs
    K, V = 512, 5003
    codes, scales = rs.lm_head_quantize(make(V, K, "bf16", 1, 0.02))
    hs = [make(m, K, "bf16", m) for m in (1, 40, 300)]
    want = [rs.lm_head_logits(h, codes, scales) for h in hs]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graphs = []
    for st in (side, torch.cuda.Stream()):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            outs = [rs.lm_head_logits(h, codes, scales) for h in hs]
        graphs.append((graph, outs, st))
    for _ in range(3):
        for graph, outs, st in graphs:
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for _, outs, _ in graphs:
            assert all(torch.equal(a, b) for a, b in zip(outs, want))
    # two eager calls at once
    st2 = torch.cuda.Stream()
    with torch.cuda.stream(side):
        a = [rs.lm_head_logits(hs[1], codes, scales) for _ in range(20)]
    with torch.cuda.stream(st2):
        b = [rs.lm_head_logits(hs[2], codes, scales) for _ in range(20)]
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[1]) for x in a) and all(torch.equal(x, want[2]) for x in b)
    assert rs.device_status() == 0


def test_from_hidden_states_to_a_scored_token():
    """A decode step: head, sampler, log probabilities of what it drew."""
    import rapid_sampling_b200 as rs
    K, V, B = 512, 8192, 6
    w = make(V, K, "bf16", 1, 0.1)
    codes, scales = rs.lm_head_quantize(w)
    states = rs.setup_rand(1, B)
    for step in range(3):
        hidden = make(B, K, "bf16", 100 + step)
        logits = rs.lm_head_logits(hidden, codes, scales)
        ids = rs.batch_sampling_temperature_topk_topp(logits, states, 0.8, 20, 0.9)
        lp, rank, ent, top, top_ids = rs.batch_top_logprobs(logits, 20, ids, 0.8)
        assert bool((rank >= 1).all()) and bool((rank <= 20).all())
        assert torch.equal(top_ids.gather(1, (rank.long() - 1)[:, None])[:, 0], ids)
        want = torch.log_softmax(wide(*quantized(hidden, 1), 1) @ wide(codes, scales, 128).t() / 0.8, -1)
        # logits to 2e-5 of their size (the bound of the products above), so differences to twice that over the temperature
        assert float((lp.double() - want.gather(1, ids.long()[:, None])[:, 0]).abs().max()) < 1e-3


@pytest.mark.parametrize("B,V_local,penalised", [(3, 4100, False), (40, 16384, True), (70, 151936, False)])
def test_vocab_parallel_sampling_from_hidden_states(B, V_local, penalised):
    """The vocab-parallel sampler's own path from hidden states: the product, whatever its slabs, and the ids and states of a
    plain call on its logits."""
    import rapid_sampling_b200 as rs
    from rapid_sampling_b200.vocab_parallel import VocabParallelSampler
    K = 256
    codes, scales = rs.lm_head_quantize(make(V_local, K, "bf16", 1, 0.2))
    hidden = make(B, K, "bf16", 2)
    a, b = VocabParallelSampler(B, V_local, 0, 1), VocabParallelSampler(B, V_local, 0, 1)
    st_a, st_b = rs.setup_rand(5, B), rs.setup_rand(5, B)
    pen_a, pen_b = (torch.zeros(B, V_local, device="cuda"), torch.zeros(B, V_local, device="cuda")) if penalised else (None, None)
    buf = torch.empty(B, V_local, device="cuda")
    for step in range(3):
        got = a.sample_hidden(hidden, codes, scales, st_a, 0.8, 50, 0.9, pen_a, 0.1, 0.1, 0.95, out=buf)
        check(hidden, codes, scales, buf)
        want = b.sample(buf, st_b, 0.8, 50, 0.9, pen_b, 0.1, 0.1, 0.95)
        assert torch.equal(got, want) and torch.equal(st_a, st_b)
        if penalised:
            assert torch.equal(pen_a, pen_b)
    assert a.project(hidden, codes, scales, st_a, 0.8, 50, 0.9).shape == (B, V_local)
    for bad in (lambda: a.project(hidden[:1], codes, scales, st_a, 0.8, 50, 0.9), lambda: a.project(hidden, codes[:128], scales, st_a, 0.8, 50, 0.9),
                lambda: a.project(hidden, codes, scales, st_a, 0.8, 50, 0.9, out=buf.half()),
                lambda: VocabParallelSampler(B, V_local, 0, 1, T=2).project(hidden, codes, scales, st_a, 0.8, 50, 0.9)):
        with pytest.raises(ValueError):
            bad()


def test_weights_beyond_32_bits():
    """Codes whose offsets pass 2^31, made and multiplied."""
    import rapid_sampling_b200 as rs
    K = 16384
    V = 2 ** 31 // K + 1000
    w = torch.zeros(V, K, dtype=torch.bfloat16, device="cuda")
    some = list(range(128)) + list(range(V - 300, V))
    w[some] = make(len(some), K, "bf16", 1, 0.02)
    codes, scales = rs.lm_head_quantize(w)
    blocks = sorted({v // 128 for v in some})
    rows = torch.tensor([v for b in blocks for v in range(128 * b, min(128 * b + 128, V))], device="cuda")
    want, want_scales = quantized(w[rows], 128)
    assert torch.equal(scales[blocks], want_scales) and torch.equal(codes[rows].double(), want)
    values = wide(want, want_scales, 128)
    for M in (2, 40, 100, 130):
        hidden = make(M, K, "bf16", M)
        got = rs.lm_head_logits(hidden, codes, scales)[:, rows].double()
        a = wide(*quantized(hidden, 1), 1)
        bound = (128 + K // 128 + 2) * 2.0 ** -23 * (a.abs() @ values.abs().t()) + 2.0 ** -24 * (a @ values.t()).abs()
        assert bool(((got - a @ values.t()).abs() <= bound + 1e-30).all())


def test_results_beyond_32_bits():
    """A result of more than 2^31 elements, aligned and not."""
    import rapid_sampling_b200 as rs
    K, V, M = 16, 1048579, 2100
    codes, scales = rs.lm_head_quantize(make(V, K, "bf16", 1, 0.02))
    hidden = make(M, K, "bf16", 2)
    for columns in (V, V - 3):
        got = rs.lm_head_logits(hidden, codes[:columns], scales[:-(-columns // 128)], dtype=torch.bfloat16)
        for rows, cols in ((slice(0, 3), slice(0, 300)), (slice(M - 5, M), slice(columns - 300, columns))):
            first = (columns - 300) // 128 * 128 if cols.start else 0
            want = rs.lm_head_logits(hidden[rows], codes[first:columns], scales[first // 128:-(-columns // 128)], dtype=torch.float32)
            want = want[:, -300:] if cols.start else want[:, :300]
            # the same products to the last bits of fp32, rounded to bf16
            assert bool(((got[rows, cols].float() - want).abs() <= 2.0 ** -8 * want.abs() * 1.001 + 1e-6).all())
        del got


def test_a_graph_notices_that_its_logits_were_written_over():
    """log p's backward pass needs the logits: `out` into them must not pass unseen."""
    import rapid_sampling_b200 as rs
    codes, scales = rs.lm_head_quantize(make(300, 256, "f32", 1, 0.02))
    h = make(4, 256, "f32", 2)
    logits = rs.lm_head_logits(h, codes, scales).requires_grad_(True)
    lp, _ = rs.batch_token_logprobs(logits, torch.zeros(4, dtype=torch.long, device="cuda"))
    with pytest.raises(ValueError):
        rs.lm_head_logits(h, codes, scales, out=logits)
    with torch.no_grad():
        rs.lm_head_logits(2 * h, codes, scales, out=logits)
    with pytest.raises(RuntimeError):
        lp.sum().backward()
    with torch.inference_mode():
        buf = torch.empty(4, 300, device="cuda")
        rs.lm_head_logits(h, codes, scales, out=buf)
    before = buf.clone()
    rs.lm_head_logits(h, codes, scales, out=buf)              # no counter to keep
    assert torch.equal(buf, before)


@pytest.mark.parametrize("M,K,V", [
    (33, 4992, 2000), (3, 7088, 3094), (64, 4096, 19000), (50, 640, 40000),      # up to 64 tokens: own runs of a tile, equal runs, whole tiles
    (128, 8192, 1000), (100, 8192, 40000), (80, 512, 60000),                     # up to 128
    (286, 6928, 1301), (384, 1024, 5003), (600, 512, 40000),                     # more, one CTA a tile
    (512, 16384, 500), (256, 8192, 19000), (700, 640, 9001)])                    # pairs
def test_every_way_of_giving_out_the_work(M, K, V):
    import rapid_sampling_b200 as rs
    codes, scales = rs.lm_head_quantize(make(V, K, "bf16", M, 0.02))
    h = make(M, K, "bf16", K)
    out = rs.lm_head_logits(h, codes, scales)
    check(h, codes, scales, out)
    assert torch.equal(out, rs.lm_head_logits(h, codes, scales))
    assert rs.device_status() == 0


@pytest.mark.parametrize("M", [1, 40, 100, 200, 300])
def test_the_largest_K(M):
    import rapid_sampling_b200 as rs
    codes, scales = rs.lm_head_quantize(make(270, 65536, "bf16", 1, 0.01))
    h = make(M, 65536, "bf16", 2)
    check(h, codes, scales, rs.lm_head_logits(h, codes, scales))


@pytest.mark.parametrize("shape", [(0,), (0, 4), (2, 0), (3, 2, 0), (3, 0, 2), (0, 0)])
def test_no_hidden_states(shape):
    """An empty result, whichever dimension is empty, into `out` as well."""
    import rapid_sampling_b200 as rs
    codes, scales = rs.lm_head_quantize(make(300, 256, "bf16", 1, 0.02))
    hidden = torch.empty(shape + (256,), device="cuda")
    assert rs.lm_head_logits(hidden, codes, scales).shape == shape + (300,)
    out = torch.empty(shape + (300,), device="cuda", dtype=torch.float16)
    assert rs.lm_head_logits(hidden, codes, scales, out=out) is out or out.shape == shape + (300,)
    with pytest.raises(ValueError):
        rs.lm_head_logits(hidden[..., :128], codes, scales)


def test_projecting_is_one_product():
    """However large the result: the hidden states are quantized once and multiplied once."""
    import rapid_sampling_b200 as rs
    from rapid_sampling_b200.vocab_parallel import VocabParallelSampler
    B, V, K = 1100, 32768, 128
    codes, scales = rs.lm_head_quantize(make(V, K, "bf16", 1, 0.2))
    hidden = make(B, K, "bf16", 2)
    vp, states = VocabParallelSampler(B, V, 0, 1), rs.setup_rand(5, B)
    before = rs.kernel_launch_count()
    logits = vp.project(hidden, codes, scales, states, 0.8, 50, 0.9)
    assert rs.kernel_launch_count() - before == 2
    assert torch.equal(logits, rs.lm_head_logits(hidden, codes, scales))
    other = rs.setup_rand(5, B)
    got = vp.sample(logits, states, 0.8, 50, 0.9, max_from_tiles=True)
    assert torch.equal(got, VocabParallelSampler(B, V, 0, 1).sample(logits, other, 0.8, 50, 0.9)) and torch.equal(states, other)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("M", [129, 300, 700])
def test_columns_behind_the_result_stay_as_they_are(M, dtype):
    """Rows at multiples of 16 and 32 bytes whose result ends anywhere within 16: what lies behind it in the same buffer is not
    written, nor what lies behind the last row."""
    import rapid_sampling_b200 as rs
    K, per = 128, 16 // (4 if dtype == "f32" else 2)
    hidden = make(M, K, "bf16", 2)
    codes, scales = rs.lm_head_quantize(make(1100, K, "bf16", 1, 0.02))
    for V in list(range(1, 2 * per + 2)) + [127, 129, 255, 257, 258, 259, 500, 639, 1001, 1002, 1003, 1005, 1007, 1023]:
        got = rs.lm_head_logits(hidden, codes[:V], scales[:-(-V // 128)])
        check(hidden, codes[:V], scales[:-(-V // 128)], got)
        for first in (0, per):
            for wide in (-(-(first + V) // per) * per, -(-(first + V) // (2 * per)) * 2 * per + 2 * per):
                buf = torch.full((M + 1, wide), 7.0, device="cuda", dtype=DT[dtype])
                rs.lm_head_logits(hidden, codes[:V], scales[:-(-V // 128)], out=buf[:M, first:first + V])
                assert torch.equal(buf[:M, first:first + V], got.to(DT[dtype])), (V, first, wide)
                assert bool((buf[:M, :first] == 7).all()) and bool((buf[:M, first + V:] == 7).all()) and bool((buf[M] == 7).all()), (V, first, wide)
