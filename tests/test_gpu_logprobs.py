"""GPU: log probabilities of given tokens, their gradient, ranks and alternatives, against plain 64-bit forms."""
import math

import pytest
import torch

from logprob_ref import close, close_grad, reference

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def make(rows, V, dtype, seed, sigma=2.5):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(tuple(rows) + (V,), generator=gen, device="cuda") * sigma).to(DT[dtype])
    t = torch.randint(0, V, tuple(rows), generator=gen, device="cuda")
    return x, t


def check_all(x, t, temperature=1.0, top_n=5, grads=True):
    """Every output of both calls, and the gradient of both results."""
    import rapid_sampling_b200 as rs
    V = x.shape[-1]
    gen = torch.Generator(device="cuda").manual_seed(99)
    g = torch.randn(x.shape[:-1], generator=gen, device="cuda")
    h = torch.randn(x.shape[:-1], generator=gen, device="cuda")
    want = reference(x, t, temperature, top_n, g, h)
    lp, ent = rs.batch_token_logprobs(x, t, temperature)
    assert lp.dtype == ent.dtype == torch.float32 and lp.shape == t.shape
    close(lp, want["logprobs"], V)
    close(ent, want["entropy"], V)
    lp2, rank, ent2, top, ids = rs.batch_top_logprobs(x, top_n, t, temperature)
    close(lp2, want["logprobs"], V)
    close(ent2, want["entropy"], V)
    assert rank.dtype == ids.dtype == torch.int32
    assert torch.equal(rank, want["ranks"])
    assert torch.equal(ids, want["ids"])
    close(top, want["top"], V)
    if grads:
        leaf = x.detach().clone(memory_format=torch.preserve_format).requires_grad_(True)
        lp3, ent3 = rs.batch_token_logprobs(leaf, t, temperature)
        close(lp3.detach(), want["logprobs"], V)      # (a row's bits depend on its address within 16 bytes, and a copy's differs)
        close(ent3.detach(), want["entropy"], V)
        got, = torch.autograd.grad((lp3, ent3), leaf, (g, h))
        assert got.dtype == x.dtype and got.shape == x.shape
        close_grad(got, want["grad"], x, g, h, temperature, want)
    assert rs.device_status() == 0


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,V", [((1,), 1), ((3,), 2), ((2,), 7), ((5,), 31), ((4,), 256), ((3,), 257), ((2, 3), 1000), ((37,), 4099),
                                    ((1,), 32768), ((2, 2), 50303), ((700,), 515), ((1,), 151936)])
def test_sizes_and_types(rows, V, dtype):
    x, t = make(rows, V, dtype, V + 1)
    check_all(x, t, 1.0, top_n=min(20, 64))


@pytest.mark.parametrize("n", [1, 2, 31, 64])
def test_list_lengths(n):
    x, t = make((6,), 5000, "f32", n)
    check_all(x, t, 0.7, top_n=n, grads=False)
    x, t = make((6,), 40, "bf16", n)       # fewer ids than slots for the longest
    check_all(x, t, 0.7, top_n=n, grads=False)


@pytest.mark.parametrize("temperature", [0.001, 0.1, 1.7, 1000.0])
def test_temperatures(temperature):
    x, t = make((9,), 3000, "f32", 5)
    check_all(x, t, temperature)


def test_row_temperatures():
    x, t = make((4, 5), 2049, "bf16", 6)
    per_row = 0.3 + torch.rand(4, 5, device="cuda")
    check_all(x, t, per_row)
    check_all(x, t, per_row[:, 0].contiguous())       # one per sequence
    wide = (0.3 + torch.rand(5, 8, device="cuda"))[:, ::2].t()
    check_all(x, t, wide)                              # any strides
    check_all(x, t, torch.tensor(0.6, device="cuda"))
    check_all(x[:, 0], t[:, 0], per_row[:, 0])


def test_views_and_token_types():
    big, t = make((3, 7), 1001, "f16", 7)
    check_all(big[:, :-1], t[:, 1:])                                   # shifted, rows at odd addresses
    check_all(big[:, 1:], t[:, :-1].int())
    check_all(big[:, ::2], t[:, ::2])
    check_all(big[1], t[1])
    check_all(big[:, :, 3:], t % 998)                                  # columns cut off on the left
    check_all(big[..., :513], t % 513)
    check_all(big[0, 0], t[0, 0])                                      # (V,)
    check_all(big[:1, 0].expand(4, 1001), t[0, :4])                    # one row for four tokens
    check_all(big.transpose(0, 1), t.t())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_masks(dtype):
    x, t = make((12,), 3001, dtype, 8)
    low = torch.finfo(DT[dtype]).min
    gen = torch.Generator(device="cuda").manual_seed(3)
    x[0] = -math.inf                                                   # nothing left
    x[1] = low                                                         # nothing but the lowest value: uniform
    x[2, torch.rand(3001, generator=gen, device="cuda") < 0.99] = -math.inf
    x[3, torch.rand(3001, generator=gen, device="cuda") < 0.99] = low
    x[4] = -math.inf
    x[4, 2999] = 1.0                                                   # one left
    x[5] = low
    x[5, 17] = 3.0
    x[6, int(t[6])] = -math.inf                                        # the token itself masked
    x[7] = -math.inf
    x[7, :3] = 2.0                                                     # three left, all equal
    x[8, ::2] = -math.inf
    x[9] = 0.0
    x[9, ::3] = -0.0                                                   # zeros of either sign are equal
    check_all(x, t, 1.0, top_n=20)
    check_all(x, t, 0.01, top_n=20)
    check_all(x, t, 100.0, top_n=20)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_masked_tokens_of_rows_shared_by_several_ctas(dtype):
    """A masked token's rank counts every other id that is masked and lies before it, and nothing else."""
    x, t = make((3,), 70003, dtype, 23)
    x[:, 30000:60001] = -math.inf
    t[:] = torch.tensor([30000, 45679, 60000], device="cuda")
    x[2] = -math.inf
    check_all(x, t, 1.0, top_n=20)


def test_a_second_derivative_is_refused():
    import rapid_sampling_b200 as rs
    x, t = make((2,), 100, "f32", 24)
    leaf = x.requires_grad_(True)
    lp, _ = rs.batch_token_logprobs(leaf, t)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(lp.sum(), leaf, create_graph=True)


def test_not_finite_rows():
    x, t = make((6,), 2050, "f32", 9)
    x[1, 5] = math.nan
    x[3, 2049] = math.inf
    x[4, 7] = -math.nan
    check_all(x, t, 1.0, top_n=4)
    x[5] = math.nan
    check_all(x, t, 1.0, top_n=64)


def test_padded_positions():
    x, t = make((4, 9), 777, "bf16", 10)
    t[1, 4:] = -1
    t[2] = -100
    x[2] = math.nan                                                    # does not matter
    check_all(x, t, 1.0, top_n=3)


@pytest.mark.parametrize("V", [600, 5003, 40000, 151936])
def test_ties(V):
    gen = torch.Generator(device="cuda").manual_seed(V)
    x = torch.zeros(8, V, device="cuda")
    x[1] = torch.randint(0, 16, (V,), generator=gen, device="cuda").float() * 0.5
    x[2] = torch.randint(0, 2, (V,), generator=gen, device="cuda").float()
    x[3, V // 2:] = 1.0
    x[4, V - 3:] = 1.0
    x[5] = torch.arange(V, device="cuda").float() / V                  # rising: the last ones win
    x[6] = -torch.arange(V, device="cuda").float() / V
    x[7, ::7] = 2.0
    t = torch.tensor([0, 1, V - 1, V // 2, V - 1, V - 5, 3, 8], device="cuda")
    check_all(x, t, 1.0, top_n=20)
    check_all(x.half(), t, 1.0, top_n=64, grads=False)


@pytest.mark.parametrize("dtype,E", [("f32", 4), ("bf16", 8)])
def test_large_logits_crowded_in_few_threads(dtype, E):
    """More large logits in the vectors of a few threads than the candidate list holds, most of them different."""
    V = 200000
    x, t = make((3,), V, dtype, 12, sigma=0.1)
    j = torch.arange(V, device="cuda")
    for r, threads in enumerate([1, 7, 30]):
        crowd = ((j // E) % 256) < threads
        x[r, crowd] = (5 + torch.rand(int(crowd.sum()), device="cuda")).to(x.dtype)
    check_all(x, t, 1.0, top_n=64, grads=False)


@pytest.mark.parametrize("V,rows", [(1000, 3), (9000, 300), (70000, 300)])
def test_large_logits_crowded_in_rows_of_one_cta(V, rows):
    """The same where a row has one CTA, of each size; most rows ordinary, so that other CTAs run beside."""
    x, t = make((rows,), V, "f32", 25, sigma=0.1)
    j = torch.arange(V, device="cuda")
    for r, (every, width) in enumerate([(1024, 64), (2048, 300), (512, 8)]):
        crowd = (j % every) < width
        x[r, crowd] = 5 + torch.rand(int(crowd.sum()), device="cuda")
    x[rows - 1] = 1.0
    check_all(x, t, 1.0, top_n=64, grads=False)
    check_all(x, t, 1.0, top_n=3, grads=False)


def test_confident_rows_keep_their_digits():
    """log p = -log1p(the rest) where p is nearly 1: relative, not absolute, accuracy (three roundings and the sum's error).
    The rest's terms are added apart from the maximum's own 1 but for those of the one thread that holds it, in which they
    may be lost: with the rest spread evenly that is 1/256 of it at most."""
    import rapid_sampling_b200 as rs
    V = 65536
    x = torch.full((3, V), 0.0, device="cuda")
    for r, top in enumerate([20.0, 30.0, 40.0]):
        x[r, 1234] = top
    t = torch.full((3,), 1234, device="cuda")
    lp, ent = rs.batch_token_logprobs(x, t)
    want = reference(x, t)
    assert bool(((lp.double() - want["logprobs"]).abs() <= (1 / 256 + 1e-4) * want["logprobs"].abs()).all()), (lp, want["logprobs"])
    assert bool(((ent.double() - want["entropy"]).abs() <= (1 / 256 + 1e-4) * want["entropy"].abs()).all())


def test_gradient_against_differences():
    import rapid_sampling_b200 as rs
    x, t = make((2,), 50, "f32", 13, sigma=1.0)
    leaf = x.clone().requires_grad_(True)
    lp, ent = rs.batch_token_logprobs(leaf, t, 0.8)
    (2 * lp.sum() - 0.3 * ent.sum()).backward()
    step = 1e-4
    x64 = x.double()

    def value(y):
        w = reference(y, t, 0.8)
        return float(2 * w["logprobs"].sum() - 0.3 * w["entropy"].sum())
    for j in range(0, 50, 7):
        a, b = x64.clone(), x64.clone()
        a[1, j] += step
        b[1, j] -= step
        slope = (value(a) - value(b)) / (2 * step)
        # central differences in 64 bits: step^2 * third derivative (below 10 here) + rounding 1e-12; the kernel's: 3e-5
        assert abs(slope - float(leaf.grad[1, j])) < 1e-4


def test_incoming_gradients():
    """One result unused, a broadcast gradient, one with strides of its own, and a padded slice of the leaf."""
    import rapid_sampling_b200 as rs
    x, t = make((3, 6), 900, "f32", 14)
    ones = torch.ones(3, 6, device="cuda")
    leaf = x.clone().requires_grad_(True)
    rs.batch_token_logprobs(leaf, t)[0].sum().backward()
    want = reference(x, t, 1.0, 0, ones, None)
    close_grad(leaf.grad, want["grad"], x, ones, None, 1.0, want)
    leaf.grad = None
    rs.batch_token_logprobs(leaf, t)[1].sum().backward()
    want = reference(x, t, 1.0, 0, None, ones)
    close_grad(leaf.grad, want["grad"], x, None, ones, 1.0, want)
    leaf.grad = None
    g = torch.randn(6, 3, device="cuda").t()
    lp, _ = rs.batch_token_logprobs(leaf, t)
    lp.backward(g)
    want = reference(x, t, 1.0, 0, g, None)
    close_grad(leaf.grad, want["grad"], x, g, None, 1.0, want)
    leaf.grad = None
    lp, _ = rs.batch_token_logprobs(leaf[:, :-1], t[:, 1:])
    lp.sum().backward()
    want = reference(x[:, :-1], t[:, 1:], 1.0, 0, ones[:, 1:], None)
    close_grad(leaf.grad[:, :-1], want["grad"], x[:, :-1], ones[:, 1:], None, 1.0, want)
    assert not leaf.grad[:, -1].any()
    row = x[0, 0].clone().requires_grad_(True)                     # a row used by several tokens: gradients add up
    rs.batch_token_logprobs(row.expand(6, 900), t[0])[0].sum().backward()
    want = reference(x[0, 0].expand(6, 900), t[0], 1.0, 0, ones[0], None)["grad"].sum(0)
    assert float((row.grad.double() - want).abs().max()) < 6 * 3 * 5e-6 + 1e-6


def test_refusals_and_device_errors():
    import rapid_sampling_b200 as rs
    x, t = make((4,), 128, "f32", 15)
    for bad in (lambda: rs.batch_token_logprobs(x.double(), t), lambda: rs.batch_token_logprobs(x.cpu(), t),
                lambda: rs.batch_token_logprobs(x, t.float()), lambda: rs.batch_token_logprobs(x, t[:3]),
                lambda: rs.batch_token_logprobs(x.t(), t[:1].expand(128)), lambda: rs.batch_token_logprobs(x, t.cpu()),
                lambda: rs.batch_token_logprobs(x, t, 0.0), lambda: rs.batch_token_logprobs(x, t, 2000.0),
                lambda: rs.batch_token_logprobs(x, t, float("nan")), lambda: rs.batch_token_logprobs(x, t, torch.ones(3, device="cuda")),
                lambda: rs.batch_token_logprobs(x, t, torch.ones(4)), lambda: rs.batch_token_logprobs(x, t, torch.ones(4, device="cuda").double()),
                lambda: rs.batch_token_logprobs(x, t, torch.ones(4, device="cuda", requires_grad=True)),
                lambda: rs.batch_top_logprobs(x, 0), lambda: rs.batch_top_logprobs(x, 65), lambda: rs.batch_top_logprobs(x[None, None], 3),
                lambda: rs.batch_token_logprobs(torch.zeros(1, 1048577, device="cuda"), t[:1]),
                lambda: rs.batch_token_logprobs(torch.zeros(4, 0, device="cuda"), t)):
        with pytest.raises(ValueError):
            bad()
    lp, ent = rs.batch_token_logprobs(x[:0], t[:0])                 # no rows: no work
    assert lp.shape == ent.shape == (0,)
    assert rs.batch_top_logprobs(x[:0], 3)[3].shape == (0, 3)
    # a token that is no column: its row NaN, no gradient, the others untouched, and the next call raises
    t2 = t.clone()
    t2[2] = 128
    leaf = x.clone().requires_grad_(True)
    lp, ent = rs.batch_token_logprobs(leaf, t2)
    torch.cuda.synchronize()
    assert torch.isnan(lp[2]) and torch.isnan(ent[2]) and not torch.isnan(lp[[0, 1, 3]]).any()
    grad, = torch.autograd.grad(lp[[0, 1, 3]].sum(), leaf)
    assert not grad[2].any() and bool(grad[3].any())
    with pytest.raises(ValueError, match="token"):
        rs.batch_token_logprobs(x, t)
    assert rs.device_status() == 0
    # a temperature out of range counts as 1
    heat = torch.tensor([1.0, 0.0, 1.0, float("nan")], device="cuda")
    lp, _ = rs.batch_token_logprobs(x, t, heat)
    close(lp, reference(x, t)["logprobs"], 128)
    with pytest.raises(ValueError, match="Temperature"):
        rs.batch_top_logprobs(x, 2)
    assert rs.device_status() == 0
    _, _, _, _, ids = rs.batch_top_logprobs(x, 2, t2)
    assert rs.device_status() == -11 and ids[2].tolist() == [-1, -1]     # the explicit read clears what it reports
    rs.batch_top_logprobs(x, 2)


def test_without_tokens():
    import rapid_sampling_b200 as rs
    x, _ = make((5,), 1234, "bf16", 16)
    lp, rank, ent, top, ids = rs.batch_top_logprobs(x, 7, temperature=0.5)
    want = reference(x, None, 0.5, 7)
    assert lp is None and rank is None
    close(ent, want["entropy"], 1234)
    close(top, want["top"], 1234)
    assert torch.equal(ids, want["ids"])


def test_same_bits_every_time_and_in_every_batch():
    """A row's results do not depend on the run; the list does not depend on how many CTAs share the row either."""
    import rapid_sampling_b200 as rs
    x, t = make((600,), 20000, "bf16", 17)
    a = rs.batch_top_logprobs(x, 20, t)
    b = rs.batch_top_logprobs(x, 20, t)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    c = rs.batch_top_logprobs(x[:2], 20, t[:2])
    assert torch.equal(a[4][:2], c[4]) and torch.equal(a[1][:2], c[1])
    close(c[0], a[0][:2].double(), 20000)


def test_capture_streams_and_two_graphs():
    """First calls inside a capture, replays with new inputs, two graphs at once on two streams."""
    import rapid_sampling_b200 as rs
    x, t = make((16,), 30001, "bf16", 18)
    y, s = make((16,), 30001, "bf16", 19)
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for a, b, st in ((x, t, streams[0]), (y, s, streams[1])):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            outs.append(rs.batch_top_logprobs(a, 20, b) + tuple(rs.batch_token_logprobs(a, b)))
        graphs.append(graph)
    for rep in range(3):
        x.copy_(make((16,), 30001, "bf16", 20 + rep)[0])
        torch.cuda.synchronize()
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for out, a, b in ((outs[0], x, t), (outs[1], y, s)):
            want = rs.batch_top_logprobs(a, 20, b) + tuple(rs.batch_token_logprobs(a, b))
            assert all(torch.equal(p, q) for p, q in zip(out, want))
    with torch.cuda.stream(streams[0]):
        got = rs.batch_token_logprobs(y, s)
    streams[0].synchronize()
    assert torch.equal(got[0], rs.batch_token_logprobs(y, s)[0])


def test_captured_training_step():
    import rapid_sampling_b200 as rs
    x, t = make((2, 40), 5001, "f32", 21)
    leaf = x.clone().requires_grad_(True)
    g = torch.randn(2, 40, device="cuda")

    def step():
        lp, ent = rs.batch_token_logprobs(leaf, t, 0.9)
        return torch.autograd.grad((lp * g).sum() + 0.1 * ent.sum(), leaf)[0]
    want = step().clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_offsets_beyond_32_bits():
    """Rows of one tensor whose element offsets pass 2^31, read and, for the gradient, written."""
    import rapid_sampling_b200 as rs
    V = 1048576
    rows = 2 ** 31 // V + 3
    x = torch.empty(rows, V, dtype=torch.bfloat16, device="cuda")
    t = torch.full((rows,), -1, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(1)
    for r in (0, rows - 1):
        x[r] = torch.randn(V, generator=gen, device="cuda").bfloat16()
        t[r] = 77 + r
    pick = [0, rows - 1]
    want = reference(x[pick], t[pick], 1.0, 5, torch.ones(2, device="cuda"), None)
    lp, rank, ent, top, ids = rs.batch_top_logprobs(x, 5, t)
    close(lp[pick], want["logprobs"], V)
    assert torch.equal(ids[pick], want["ids"]) and torch.equal(rank[pick], want["ranks"])
    x.requires_grad_(True)
    lp, ent = rs.batch_token_logprobs(x, t)
    grad, = torch.autograd.grad(lp.sum(), x)
    close_grad(grad[pick], want["grad"], x[pick], torch.ones(2, device="cuda"), None, 1.0, want)
    assert not grad[1].any() and not grad[rows - 2].any()


def test_follows_a_sampling_call():
    """As a serving step uses them: sample, then the sampled ids' log probabilities, ranks and alternatives."""
    import rapid_sampling_b200 as rs
    x, _ = make((8,), 50304, "f32", 22)
    T = torch.tensor([0.7, 1.0] * 4, device="cuda")
    ids, prob, _ = rs.batch_sampling_rows(x, rs.setup_rand(3, 8), T, torch.full((8,), 40, dtype=torch.int32, device="cuda"),
                                          torch.full((8,), 0.95, device="cuda"), return_prob=True)
    lp, rank, ent, top, top_ids = rs.batch_top_logprobs(x, 40, ids, T)
    # the sampler's probability is a 32-bit softmax of its own: 2e-6 relative
    assert bool(((lp.exp() - prob).abs() <= 2e-5 * prob).all())
    assert bool((rank <= 40).all()) and torch.equal(top_ids.gather(1, (rank.long() - 1)[:, None])[:, 0], ids)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_subnormal_logits_are_ordered(dtype):
    """Values below the smallest normal one differ and are counted and listed in their order."""
    V = 2500
    step = {"f32": 2.0 ** -149, "f16": 2.0 ** -24, "bf16": 2.0 ** -133}[dtype]
    k = torch.arange(V, device="cuda") * 37 % 101 - 50
    x = (k.double() * step).to(DT[dtype])[None].repeat(3, 1)
    assert len(x.float().unique()) == 101
    check_all(x, torch.tensor([0, 1200, 2499], device="cuda"), 1.0, top_n=64)


def test_first_calls_of_a_process_inside_a_capture():
    """Nothing needs a call outside a capture first."""
    import subprocess
    import sys
    code = """
import torch, rapid_sampling_b200 as rs
x = torch.randn(6, 5000, device="cuda"); t = torch.randint(0, 5000, (6,), device="cuda")
w = torch.randn(5000, 256, device="cuda"); h = {m: torch.randn(m, 256, device="cuda") for m in (4, 50, 200)}
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    a = rs.batch_token_logprobs(x, t) + rs.batch_top_logprobs(x, 5, t)
    codes, scales = rs.lm_head_quantize(w)
    b = [rs.lm_head_logits(v, codes, scales) for v in h.values()]
g.replay(); torch.cuda.synchronize()
want = rs.batch_token_logprobs(x, t) + rs.batch_top_logprobs(x, 5, t)
assert all(torch.equal(p, q) for p, q in zip(a, want))
c2, s2 = rs.lm_head_quantize(w)
assert torch.equal(codes.float(), c2.float()) and torch.equal(scales, s2)
assert all(torch.equal(p, rs.lm_head_logits(v, c2, s2)) for p, v in zip(b, h.values()))
print("fine")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=240)
    assert r.returncode == 0 and "fine" in r.stdout, r.stderr[-2000:]


def test_calls_from_several_threads():
    """Two host threads with streams of their own."""
    import threading
    import rapid_sampling_b200 as rs
    codes, scales = rs.lm_head_quantize(torch.randn(3000, 512, device="cuda") * 0.05)
    data = [(make((9,), 20000, "bf16", 40 + i), torch.randn(70 * (i + 1), 512, device="cuda")) for i in range(2)]
    want = [(rs.batch_top_logprobs(x, 10, t), rs.lm_head_logits(h, codes, scales)) for (x, t), h in data]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        (x, t), h = data[i]
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            for _ in range(50):
                a, b = rs.batch_top_logprobs(x, 10, t), rs.lm_head_logits(h, codes, scales)
            st.synchronize()
            if not (all(torch.equal(p, q) for p, q in zip(a, want[i][0])) and torch.equal(b, want[i][1])):
                wrong.append(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [th.start() for th in threads]
    [th.join() for th in threads]
    assert not wrong


def test_one_temperature_in_a_tensor_of_any_shape():
    import rapid_sampling_b200 as rs
    for rows in ((5,), (2, 3), ()):
        x, t = make(rows, 1000, "f32", 60)
        t = t.reshape(rows)
        want = rs.batch_top_logprobs(x, 5, t, 0.625)
        for shape in ((), (1,), (1, 1)):
            one = torch.full(shape, 0.625, device="cuda")
            assert all(torch.equal(a, b) for a, b in zip(rs.batch_top_logprobs(x, 5, t, one), want))
            assert torch.equal(rs.batch_token_logprobs(x, t, one)[0], rs.batch_token_logprobs(x, t, 0.625)[0])


def test_logits_further_apart_than_the_largest_number():
    """Their difference over the temperature is finite: a log probability is its correctly scaled value."""
    x = torch.tensor([[3e38, -3e38, 0.0, 2.9e38], [-3.4e38, 3.4e38, -math.inf, 1e38]], device="cuda")
    for temperature in (2.0, 4.0, 1000.0):
        for token in range(4):
            check_all(x, torch.full((2,), token, device="cuda"), temperature)


def test_a_backward_pass_captured_beside_an_eager_graph_is_refused():
    """In a process of its own: without the refusal, torch's engine would end it."""
    import subprocess
    import sys
    code = """
import torch, rapid_sampling_b200 as rs
t = torch.randint(0, 5000, (6,), device="cuda")
h = torch.randn(6, 64, device="cuda")
for weight in (None, torch.randn(64, 5000, device="cuda", requires_grad=True)):
    leaf = torch.randn(6, 5000, device="cuda", requires_grad=True) if weight is None else weight
    logits = (lambda: leaf) if weight is None else (lambda: h @ leaf)
    def step():
        loss = rs.batch_token_logprobs(logits(), t)[0].sum()
        loss.backward()
        return loss
    kept = rs.batch_token_logprobs(logits(), t)[0].sum()          # an eager graph that stays
    leaf.grad = torch.zeros_like(leaf)
    torch.cuda.synchronize()
    try:
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            step()
    except RuntimeError as e:
        assert "alive" in str(e), e
    else:
        raise SystemExit("not refused")
    torch.cuda.synchronize()
    kept.backward()                                               # the process and the graph go on
    want = leaf.grad.clone()
    del kept
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    leaf.grad.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.allclose(leaf.grad, want, rtol=0, atol=1e-4)
print("fine")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=240)
    assert r.returncode == 0 and "fine" in r.stdout, r.stdout[-500:] + r.stderr[-2000:]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V", [1010, 1578, 2048])
def test_the_most_probable_token_of_short_rows(V, dtype):
    """A list of one in rows that 64 threads read: quick, and right, whatever shared memory held before."""
    import rapid_sampling_b200 as rs
    for rows in ((5,), (3000,)):
        x, t = make(rows, V, dtype, 70)
        rs.batch_top_logprobs(torch.full_like(x, 3.0), 40)          # leaves keys behind
        check_all(x, t, 0.8, top_n=1, grads=False)
    # as quick as a list of two, within noise (36 passes over the row took eight times as long)
    def us(n):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        best = 1e9
        for _ in range(20):
            a.record()
            rs.batch_top_logprobs(x, n)
            b.record()
            b.synchronize()
            best = min(best, a.elapsed_time(b))
        return best
    assert us(1) < 2 * us(2)


@pytest.mark.parametrize("rows,dtype", [((2,), "f32"), ((2,), "f16"), ((300,), "bf16"), ((300,), "f32")])
def test_the_longest_rows_and_lists(rows, dtype):
    x, t = make(rows, 1048576, dtype, 80)
    check_all(x, t, 0.9, top_n=64, grads=False)


# distances in elements between a row's maximum and its runner-up: a neighbour in the same 16 bytes, and other vectors of the same
# thread, in the same step and in later ones, whatever the number of threads
def _runners_up(V, size):
    E = 16 // size
    return sorted({d for d in [1, 2] + [E * nt * k for nt in (64, 128, 256) for k in (1, 3, 4, 9)] if 8 + d < V})


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V,rows", [(4, 0), (9, 0), (1500, 0), (1500, 400), (5000, 400), (5003, 400), (70000, 0), (70003, 0), (70003, 400)])
def test_confident_rows_keep_the_runner_up(V, rows, dtype):
    """Rows of one token of probability nearly one and one other, which the same thread may hold: log p = -log1p(r) with
    r = exp(-gap / T), H = log1p(r) + gap/T r / (1 + r), and gradients of +-r / (1 + r).  The exponent's argument has three roundings of
    2^-24, so r is off by 2^-23 * 2 gap/T at most, and by 2^-22 for the exponential; sums, log1p, expm1 and quotients take
    another 2^-21 at most.  (Gaps of 16-bit types too: all values are whole.)"""
    import rapid_sampling_b200 as rs
    size = 4 if dtype == "f32" else 2
    cases = [(gap, d, at, way) for gap in (3.0, 8.0, 17.0, 40.0) for d in (_runners_up(V, size) or [1]) for at in (0, min(8, V - 1 - d), V - 1 - d) for way in (0, 1)]
    cases = cases * (1 + rows // len(cases))
    n = len(cases)
    x = torch.full((n, V), -math.inf, device="cuda")
    gap = torch.tensor([c[0] for c in cases], device="cuda")
    r = torch.arange(n, device="cuda")
    one, other = (torch.tensor([at + (0 if way == first else d) for _, d, at, way in cases], device="cuda") for first in (0, 1))
    x[r, one] = 3.0
    x[r, other] = 3.0 - gap
    x = x.to(DT[dtype])
    for T in (1.0, 0.5):
        z = gap.double() / T
        rest = torch.exp(-z)
        tol = 2.0 ** -23 * 2 * z + 2.0 ** -20
        want, H = -torch.log1p(rest), torch.log1p(rest) + z * rest / (1 + rest)
        lp, ent = rs.batch_token_logprobs(x, one, T)
        assert bool(((lp.double() - want).abs() <= tol * want.abs()).all()), (lp, want)
        assert bool(((ent.double() - H).abs() <= tol * H).all()), (ent, H)
        lp2, rank, ent2, top, ids = rs.batch_top_logprobs(x, 2, one, T)
        assert torch.equal(lp2, top[:, 0]) and bool((rank == 1).all()) and torch.equal(ids.long(), torch.stack([one, other], 1))
        assert bool(((lp2.double() - want).abs() <= tol * want.abs()).all()) and bool(((ent2.double() - H).abs() <= tol * H).all())
        second = want - z
        assert bool(((top[:, 1].double() - second).abs() <= tol * second.abs()).all())
        leaf = x.clone().requires_grad_(True)
        grad, = torch.autograd.grad(rs.batch_token_logprobs(leaf, one, T)[0].sum(), leaf)
        want = rest / (1 + rest) / T
        half = torch.finfo(DT[dtype]).eps / 2 * want + torch.finfo(DT[dtype]).smallest_normal * torch.finfo(DT[dtype]).eps
        assert bool(((grad[r, one].double() - want).abs() <= tol * want + half).all())
        assert bool(((grad[r, other].double() + want).abs() <= tol * want + half).all())
        grad[r, one] = grad[r, other] = 0
        assert not grad.any()
    assert rs.device_status() == 0


def test_a_graph_that_holds_the_first_calls_reports_what_its_replays_meet():
    """A process whose first calls are captured ones: a replay with a bad token or temperature raises from the next call."""
    import subprocess
    import sys
    code = """
import torch, rapid_sampling_b200 as rs
x = torch.randn(6, 5000, device="cuda"); t = torch.randint(0, 5000, (6,), device="cuda"); heat = torch.ones(6, device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    lp, _ = rs.batch_token_logprobs(x, t, heat)
def refused(word):
    g.replay(); torch.cuda.synchronize()
    try:
        rs.batch_top_logprobs(x, 3)
    except ValueError as e:
        assert word in str(e), e
    else:
        raise SystemExit("not raised")
    assert rs.device_status() == 0
g.replay(); torch.cuda.synchronize()
assert torch.equal(lp, rs.batch_token_logprobs(x, t, heat)[0])
t[2] = 5000
refused("token")
t[2] = 7; heat[3] = 0
refused("Temperature")
heat[3] = 1
g.replay(); torch.cuda.synchronize()
assert torch.equal(lp, rs.batch_token_logprobs(x, t, heat)[0])
print("fine")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=240)
    assert r.returncode == 0 and "fine" in r.stdout, r.stdout[-500:] + r.stderr[-2000:]


def test_an_error_of_a_sampling_call_is_reported_once():
    """Whichever call raises it."""
    import rapid_sampling_b200 as rs
    x, t = make((4,), 4096, "f32", 90)
    heat = torch.tensor([1.0, 0.0, 1.0, 1.0], device="cuda")
    codes, scales = rs.lm_head_quantize(torch.randn(256, 64, device="cuda"))
    for call in (lambda: rs.batch_token_logprobs(x, t), lambda: rs.batch_top_logprobs(x, 3),
                 lambda: rs.lm_head_logits(torch.zeros(2, 64, device="cuda"), codes, scales)):
        rs.batch_sampling_rows(x, rs.setup_rand(1, 4), heat)
        torch.cuda.synchronize()
        with pytest.raises(ValueError, match="Temperature"):
            call()
        assert rs.device_status() == 0
        call()


def test_forward_mode_is_refused():
    """Tangents are not propagated: results without one would count as constants."""
    import rapid_sampling_b200 as rs
    import torch.autograd.forward_ad as fwd
    x, t = make((3,), 100, "f32", 91)
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        heat = fwd.make_dual(torch.ones(3, device="cuda"), torch.ones(3, device="cuda"))
        for bad in (lambda: rs.batch_token_logprobs(dual, t), lambda: rs.batch_token_logprobs(x, t, heat)):
            with pytest.raises((ValueError, RuntimeError)):
                bad()
        close(rs.batch_token_logprobs(x, t)[0], reference(x, t)["logprobs"], 100)
        close(rs.batch_token_logprobs(fwd.unpack_dual(dual).primal, t)[0], reference(x, t)["logprobs"], 100)
        with torch.inference_mode():                                    # tangents are off
            close(rs.batch_token_logprobs(dual, t)[0], reference(x, t)["logprobs"], 100)
    with pytest.raises((ValueError, RuntimeError)):
        torch.func.jvp(lambda y: rs.batch_token_logprobs(y, t)[0], (x,), (torch.ones_like(x),))


def test_a_captured_backward_pass_that_stops_before_such_leaves_is_not_refused():
    """Only the leaves that the pass reaches matter: a gradient of the logits alone leaves the weight behind them alone."""
    import subprocess
    import sys
    code = """
import torch, rapid_sampling_b200 as rs
t = torch.randint(0, 5000, (6,), device="cuda")
h = torch.randn(6, 64, device="cuda")
w = torch.randn(64, 5000, device="cuda", requires_grad=True)
other = torch.randn(5000, device="cuda", requires_grad=True)
kept = (w * 2).sum()                                          # an eager graph of the weight that stays
def step(inputs=None):
    logits = h @ w + other
    lp, ent = rs.batch_token_logprobs(logits, t, 0.9)
    return torch.autograd.grad(lp.sum() + 0.1 * ent.sum(), inputs or [logits])[0]
want, want_other = step().clone(), step([other]).clone()
side = torch.cuda.Stream()
side.wait_stream(torch.cuda.current_stream())
with torch.cuda.stream(side):
    step()
    step([other])
torch.cuda.current_stream().wait_stream(side)
torch.cuda.synchronize()
for inputs, expect in ((None, want), ([other], want_other)):
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step(inputs)
    got.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, expect)
for bad in (lambda: step([w]), lambda: rs.batch_token_logprobs(h @ w, t)[0].sum().backward()):      # reach it
    try:
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            bad()
    except RuntimeError as e:
        assert "alive" in str(e), e
    else:
        raise SystemExit("not refused")
    torch.cuda.synchronize()
kept.backward()
print("fine")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=240)
    assert r.returncode == 0 and "fine" in r.stdout, r.stdout[-500:] + r.stderr[-2000:]


def test_a_captured_backward_pass_into_an_eager_forward_pass_is_refused():
    """Before the engine spoils the capture: torch's generators stay usable."""
    import subprocess
    import sys
    code = """
import torch, rapid_sampling_b200 as rs
t = torch.randint(0, 5000, (6,), device="cuda")
h = torch.randn(6, 64, device="cuda")
w = torch.randn(64, 5000, device="cuda", requires_grad=True)
logits = h @ w                                                # eager, on the default stream
for bad in (lambda x: torch.autograd.grad(rs.batch_token_logprobs(x, t)[0].sum(), x), lambda x: rs.batch_token_logprobs(x, t)[0].sum().backward()):
    try:
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            bad(logits)
    except RuntimeError as e:
        assert "eager graph" in str(e), e
    else:
        raise SystemExit("not refused")
    torch.cuda.synchronize()
    torch.randn(3, device="cuda")
x = logits.detach().requires_grad_(True)                      # the way to do it
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    got, = torch.autograd.grad(rs.batch_token_logprobs(x, t)[0].sum(), x)
g.replay()
torch.cuda.synchronize()
want, = torch.autograd.grad(rs.batch_token_logprobs(logits, t)[0].sum(), logits)
assert torch.equal(got, want)
print("fine")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=240)
    assert r.returncode == 0 and "fine" in r.stdout, r.stdout[-500:] + r.stderr[-2000:]
