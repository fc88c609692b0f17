"""sample_logits against a plain implementation in 64 bits."""

import math

import pytest
import torch

import mixfp4_b200 as mx

pytestmark = pytest.mark.gpu

INF = math.inf


def _reference(x, u, t, k, p, f):
    """One row, doubles: (token, log probability)."""
    x = [(-INF if math.isnan(v) else v) for v in x]
    top = max(x)
    if top == -INF:
        return -1, -INF
    order = sorted(range(len(x)), key=lambda i: (-x[i], i))
    if not t > 0:
        return order[0], 0.0
    w = [1.0 if v == top else math.exp((v - top) / t) if top != INF else 0.0 for v in x]
    if k > 0:
        order = order[:k]
    if p < 1:
        goal, run, n = p * math.fsum(w[i] for i in order), 0.0, 0
        while n == 0 or run < goal:
            run += w[order[n]]
            n += 1
            if n == len(order):
                break
        order = order[:n]
    kept = sorted(i for i in order if w[i] >= min(f, 1.0) and w[i] > 0)
    total = math.fsum(w[i] for i in kept)
    run = 0.0
    for i in kept:
        run += w[i]
        if run > u * total:
            break
    return i, math.log(w[i] / total)


def _check(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    token, logprob = mx.sample_logits(logits, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p, return_logprob=True)
    rows = logits.shape[0]
    each = lambda v: v.double().tolist() if isinstance(v, torch.Tensor) else [v] * rows
    t, k, p, f = each(temperature), each(top_k), each(top_p), each(min_p)
    x = logits.double().cpu().tolist()
    for r, (a, b, v) in enumerate(zip(token.tolist(), logprob.tolist(), u.double().tolist())):
        want, lp = _reference(x[r], v, t[r], int(k[r]), p[r], f[r])
        assert a == want, (r, a, want)
        # the log of a share: weights and sums are held to 2^-44 of the largest, the result is rounded to 24 bits
        assert b == lp or abs(b - lp) <= 2.0 ** -24 * abs(lp) + 1e-9, (r, b, lp)


def _logits(rows, vocab, dtype, seed, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn((rows, vocab), generator=g)).to(dtype).cuda(), torch.rand(rows, generator=g).cuda()


SETTINGS = [dict(), dict(temperature=0.0), dict(temperature=0.6, top_k=1), dict(top_k=50, top_p=0.9), dict(temperature=1.4, top_p=0.5),
            dict(min_p=0.1), dict(temperature=0.8, top_k=20, top_p=0.95, min_p=0.02), dict(top_p=0.0), dict(top_k=1000, top_p=0.999),
            dict(min_p=1.0), dict(temperature=0.05), dict(temperature=50.0, top_p=0.99)]


@pytest.mark.parametrize("settings", SETTINGS, ids=lambda s: "-".join(f"{k}{v}" for k, v in s.items()) or "plain")
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_against_64_bits(dtype, settings):
    for rows, vocab, seed in ((3, 1, 1), (5, 17, 2), (40, 1001, 3), (2, 40003, 4)):
        _check(*_logits(rows, vocab, dtype, seed), **settings)


@pytest.mark.parametrize("rows", [1, 8, 30, 100])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_every_split_of_a_row(rows, dtype):
    """Rows of 1 to 8 CTAs; a vocabulary past what shared memory holds of fp32 rows in the last."""
    _check(*_logits(rows, 9000, dtype, rows), temperature=0.9, top_k=300, top_p=0.97)
    if rows == 1:
        _check(*_logits(1, 500000, dtype, 9), temperature=0.9, top_p=0.9)


def test_equal_values_are_counted_off_by_index():
    x = torch.zeros((64, 5003), device="cuda")
    u = ((torch.arange(64, dtype=torch.float32) + 0.5) / 64).cuda()
    for settings in (dict(), dict(top_k=1), dict(top_k=37), dict(top_k=4999, top_p=0.5), dict(top_p=0.25), dict(top_p=0.9), dict(top_k=5003)):
        _check(x, u, **settings)
    x[:, 100:4000] = 2.0
    for settings in (dict(top_k=3000), dict(top_k=4500), dict(top_p=0.5), dict(top_p=0.99), dict(top_k=4200, top_p=0.999)):
        _check(x, u, **settings)
    few = torch.randint(-3, 4, (64, 3001), generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    for settings in (dict(top_k=700), dict(top_p=0.6), dict(top_k=300, top_p=0.9), dict(temperature=0.0)):
        _check(few, u, **settings)
    zeros = torch.where(few == 0, -few, few)                 # zeros of both signs are one value
    zeros[:, ::2] = few[:, ::2]
    _check(zeros, u, top_k=1500)


def test_masked_rows_and_values_that_are_not_finite():
    x, u = _logits(8, 3000, torch.float32, 5)
    lowest = torch.finfo(torch.float32).min
    x[0] = -INF
    x[1] = math.nan
    x[2, :-1] = -INF
    x[3, 1:] = lowest
    x[4] = lowest
    x[5, [7, 2999]] = INF
    x[6, ::2] = math.nan
    x[7, 100:] = -INF
    for settings in (dict(), dict(temperature=0.0), dict(top_k=5), dict(top_p=0.9), dict(top_k=50, top_p=0.5, min_p=0.05)):
        _check(x, u, **settings)
    token, logprob = mx.sample_logits(x, u, return_logprob=True)
    assert token[:3].tolist() == [-1, -1, 2999] and logprob[:3].tolist() == [-INF, -INF, 0.0]


def test_a_setting_for_each_row():
    x, u = _logits(50, 2000, torch.bfloat16, 8)
    pick = lambda values, dtype: torch.tensor([values[i % len(values)] for i in range(50)], dtype=dtype, device="cuda")
    _check(x, u, temperature=pick([0.0, 0.7, 1.0, 1.5, 0.3], torch.float32), top_k=pick([0, 5, 100, -1], torch.int32),
           top_p=pick([1.0, 0.9, 0.5], torch.float32), min_p=pick([0.0, 0.0, 0.05, 0.2, 0.0, 0.0, 1.0], torch.float32))


def test_ends_of_the_random_numbers():
    x, _ = _logits(6, 700, torch.float32, 3)
    u = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, 2.0, -1.0, math.nan], device="cuda")
    token = mx.sample_logits(x, u, top_k=9).tolist()
    kept = x.topk(9, dim=1).indices.sort(dim=1).values.tolist()
    assert token == [kept[0][0], kept[1][-1], kept[2][-1], kept[3][-1], kept[4][0], kept[5][0]]


def test_strides_shapes_streams_and_capture():
    x, u = _logits(6, 1500, torch.bfloat16, 4)
    want = mx.sample_logits(x, u, top_p=0.9)
    wide = torch.full((6, 1777), 50.0, dtype=torch.bfloat16, device="cuda")
    wide[:, 3:1503] = x
    assert torch.equal(mx.sample_logits(wide[:, 3:1503], u, top_p=0.9), want)
    assert torch.equal(mx.sample_logits(x.t().contiguous().t(), u, top_p=0.9), want)
    assert torch.equal(mx.sample_logits(x.reshape(2, 3, 1500), u.reshape(2, 3), top_p=0.9), want.reshape(2, 3))
    assert mx.sample_logits(x[0], u[0], top_p=0.9).shape == () and mx.sample_logits(x[:0], u[:0]).shape == (0,)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(g, stream=side):
            token = mx.sample_logits(x, u, top_p=0.9)
    x.copy_(x.flip(0))
    u.copy_(u.flip(0))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(token, want.flip(0))


def test_head_and_sampling_together():
    """A step's end as the decoder runs it: head product in FP8, then a token; the token follows from the logits."""
    g = torch.Generator().manual_seed(2)
    head = mx.quantize_fp8_weight((0.05 * torch.randn((5000, 512), generator=g)).to(torch.bfloat16).cuda())
    h, u = torch.randn((12, 512), generator=g).to(torch.bfloat16).cuda(), torch.rand(12, generator=g).cuda()
    _check(mx.fp8_linear(h, head), u, temperature=0.8, top_k=40, top_p=0.95)


def test_logits_rewritten_just_before_the_call():
    a, u = _logits(3, 6000, torch.bfloat16, 1)
    b, _ = _logits(3, 6000, torch.bfloat16, 2)
    want = [mx.sample_logits(x, u, top_k=30, top_p=0.9) for x in (a, b)]
    x, got = a.clone(), []
    for i in range(20):
        x.copy_((a, b)[i % 2])
        got.append(mx.sample_logits(x, u, top_k=30, top_p=0.9))
    assert all(torch.equal(t, want[i % 2]) for i, t in enumerate(got))


def test_logits_past_2_31_elements():
    rows, vocab = 4400, 500000
    x = torch.zeros((rows, vocab), dtype=torch.bfloat16, device="cuda")
    at = torch.arange(rows, device="cuda") * 113 % vocab
    x.scatter_(1, at[:, None], 50.0)
    u = torch.full((rows,), 0.5, device="cuda")
    for settings in (dict(top_k=5), dict(top_p=0.9), dict(temperature=0.0)):
        assert torch.equal(mx.sample_logits(x, u, **settings), at)


def test_decoder_draws_its_tokens():
    """The harness with an FP8 head, sampling within the captured decode step."""
    from mixfp4_b200.llama_decode import run

    keep = {}
    settings = {"temperature": 0.8, "top_k": 50, "top_p": 0.95, "min_p": 0.0}
    got = run(layers=1, batch=2, prompt=32, tokens=2, keep=keep, head="fp8", sampling=settings)
    assert got["head"] == "fp8" and got["sampling"] == settings and got["decode_ms_per_step"] > 0
    assert run(layers=1, batch=2, prompt=32, tokens=2, weights=keep["weights"])["sampling"] is None


def test_refusals():
    x, u = _logits(4, 100, torch.float32, 1)
    for bad in (dict(temperature=-1.0), dict(top_p=1.5), dict(min_p=-0.1), dict(top_p=torch.ones(3, device="cuda"))):
        with pytest.raises(ValueError):
            mx.sample_logits(x, u, **bad)
    for bad in (dict(top_k=2.5), dict(top_k=torch.ones(4, device="cuda")), dict(temperature="1")):
        with pytest.raises(TypeError):
            mx.sample_logits(x, u, **bad)
    with pytest.raises(ValueError):
        mx.sample_logits(x, u[:3])
    with pytest.raises(TypeError):
        mx.sample_logits(x, u.double())
    with pytest.raises(TypeError):
        mx.sample_logits(x.double(), u)
    with pytest.raises(mx._native.MixFP4Error):
        mx.sample_logits(torch.zeros((1, 600000), device="cuda"), u[:1])


def test_settings_that_are_nan_filter_nothing():
    rows, nan = 6, torch.full((6,), math.nan, device="cuda")
    x, u = _logits(rows, 5000, torch.float32, 41)
    for k in (0, 40, 2000):                                 # no cut by count, a few candidates, many
        plain = mx.sample_logits(x, u, top_k=k, return_logprob=True)
        for settings in (dict(top_p=nan), dict(min_p=nan), dict(top_p=nan, min_p=nan)):
            got = mx.sample_logits(x, u, top_k=k, return_logprob=True, **settings)
            assert torch.equal(got[0], plain[0]) and torch.equal(got[1], plain[1]), (k, settings)
    assert torch.equal(mx.sample_logits(x, u, temperature=nan), x.argmax(-1))
    assert torch.equal(mx.sample_logits(x, nan), mx.sample_logits(x, torch.zeros_like(u)))
    assert torch.equal(mx.sample_logits(x, u, top_k=-7), mx.sample_logits(x, u))


@pytest.mark.parametrize("temperature", [1e-40, 1e-30, 1e30, 1e38, 3e38])
def test_values_and_temperatures_near_the_ends_of_fp32(temperature):
    """Differences of logits that overflow, and a width of the bins that does."""
    g = torch.Generator().manual_seed(43)
    for scale in (3e38, 1e38, 1e-38):
        x = (scale * (2 * torch.rand((4, 3001), generator=g) - 1)).cuda()
        u = torch.rand(4, generator=g).cuda()
        for settings in (dict(), dict(top_k=700), dict(top_p=0.6), dict(top_k=2000, top_p=0.99)):
            _check(x, u, temperature=temperature, **settings)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_logits_closer_together_than_a_bin(dtype):
    """All of a row within a bin or two: a top-k's candidates are those that were counted, not all that share their bin."""
    for rows, vocab, scale in ((20, 1500, 0.01), (6, 9000, 0.003), (3, 40003, 0.02)):
        for k in (1, 2, 20, 200):
            x, u = _logits(rows, vocab, dtype, 71 + k, scale)
            for settings in (dict(temperature=1.5), dict(top_p=0.5), dict(temperature=20.0, min_p=0.9)):
                _check(x, u, top_k=k, **settings)


@pytest.mark.parametrize("rows,vocab", [(1, 16384), (12, 16384), (20, 8192), (40, 4096)])
def test_shortest_slices_launch_after_launch(rows, vocab):
    """CTAs of 2048 logits, eight, four and two to a row: a CTA gets to its peers' memory as early as it ever does."""
    x, u = _logits(rows, vocab, torch.bfloat16, rows)
    _check(x, u, top_k=50, top_p=0.9)
    want = mx.sample_logits(x, u, top_k=50, top_p=0.9)
    got = [mx.sample_logits(x, u, top_k=50, top_p=0.9) for _ in range(300)]
    assert torch.equal(torch.stack(got), want.expand(300, rows))


@pytest.mark.parametrize("rows,vocab,dtype,k,step", [
    (64, 4096, torch.bfloat16, 50, 256), (1, 32768, torch.float32, 200, 256), (1, 32000, torch.bfloat16, 200, 250),
    (1, 4096, torch.float32, 50, 128), (1, 128256, torch.bfloat16, 300, 1002), (64, 4100, torch.float16, 100, 257)])
def test_top_k_of_rows_with_few_large_logits(rows, vocab, dtype, k, step):
    """Fewer than k large logits, each at the end of what a warp reads: the others that belong to the first k are found below them."""
    g = torch.Generator().manual_seed(k + vocab)
    u = torch.rand(rows, generator=g).cuda()
    for offset in (step - 1, 0, step // 2, step - 9):
        x = torch.rand((rows, vocab), generator=g)
        x[:, offset::step] = 5.0
        x = x.to(dtype).cuda()
        for settings in (dict(), dict(temperature=8.0), dict(temperature=4.0, top_p=0.7), dict(temperature=8.0, min_p=0.55)):
            _check(x, u, top_k=k, **settings)


def test_top_k_of_rows_that_rise_and_fall():
    """Rows in order, and in runs of every length up to a warp's share: the largest stand together, wherever that is."""
    x = torch.empty((40, 6007))
    ramp = torch.arange(6007, dtype=torch.float32)
    for r in range(40):
        run = 1 + 11 * r
        x[r] = (ramp % run) * (1 if r % 2 else -1) + ramp * 1e-5
    x, u = (x / 40).cuda(), torch.rand(40, generator=torch.Generator().manual_seed(5)).cuda()
    for k in (2, 17, 33, 64, 65, 130, 500, 513, 2000):
        _check(x, u, top_k=k, temperature=3.0)
    _check(x[:1].contiguous(), u[:1], top_k=400, temperature=3.0)


@pytest.mark.parametrize("temperature", [5e-324, 1e-310, 3e-309, 1e-307, 1e-300, 1e-60, 1e-45])
def test_temperatures_below_those_of_fp32(temperature):
    """A number is a double: down to the smallest, whose reciprocal is not finite, all the weight is the largest logits'."""
    g = torch.Generator().manual_seed(47)
    u = torch.tensor([0.1, 0.3, 0.6, 0.9], device="cuda")
    x = torch.randn((4, 3001), generator=g)
    x[0, [5, 900, 2000]] = 9.0                               # three share it
    x[1] = 1e-45 * torch.randint(0, 3, (3001,), generator=g)      # neighbours of the smallest size
    x[2, 17] = 3e38
    x[3] = x[3].abs().neg() * 1e-38
    for kind in (torch.float32, torch.bfloat16):
        for settings in (dict(), dict(top_k=2), dict(top_k=700), dict(top_p=0.6), dict(min_p=0.5), dict(top_k=2000, top_p=0.99)):
            _check(x.to(kind).cuda(), u, temperature=temperature, **settings)


def test_decoder_runs_the_head_that_it_was_asked_for(monkeypatch):
    from mixfp4_b200 import llama_decode

    device, norms = torch.device("cuda", torch.cuda.current_device()), []
    norm = llama_decode.rms_norm
    monkeypatch.setattr(llama_decode, "rms_norm", lambda *args: norms.append(norm(*args)) or norms[-1])
    fp8 = llama_decode.Decoder(1, 2, 16, device, head="fp8")
    plain = llama_decode.Decoder(1, 2, 16, device, weights=fp8.weights)
    again = llama_decode.Decoder(1, 2, 16, device, weights=fp8.weights, head="fp8")
    ids = torch.randint(0, llama_decode.VOCAB, (2, 9), generator=torch.Generator().manual_seed(3)).to(device)
    with torch.no_grad():
        for model, quantized in ((fp8, True), (plain, False), (again, True)):
            assert (model.head_fp8 is not None) == quantized
            logits = model.forward(ids, torch.arange(9, device=device), 9)
            last = norms[-1]
            assert torch.equal(logits, mx.fp8_linear(last, mx.quantize_fp8_weight(model.head)) if quantized else last @ model.head.T)
    with pytest.raises(ValueError):
        llama_decode.Decoder(1, 2, 16, device, weights=fp8.weights, head="fp4")


def test_harness_times_the_linears_without_the_sampler(monkeypatch):
    from mixfp4_b200 import llama_decode

    drawn, per_step = [], []
    sample = mx.sample_logits
    monkeypatch.setattr(mx, "sample_logits", lambda *args, **kwargs: drawn.append(1) or sample(*args, **kwargs))

    def step_once(fn, steps):
        before = len(drawn)
        fn()
        per_step.append(len(drawn) - before)
        return 1.0

    monkeypatch.setattr(llama_decode, "_time_graph", step_once)
    llama_decode.run(layers=1, batch=1, prompt=8, tokens=1, sampling={"temperature": 0.8})
    assert per_step == [1, 0]                                # a whole step, the linears alone
