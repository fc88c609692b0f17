"""The block-scaled FP8 quantizers and product against plain arithmetic in 64 bits."""

import pytest
import torch

import mixfp4_b200 as mx
from mixfp4_b200 import _native as nat

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
SUBNORMAL = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}


def _e4m3(v):
    """Nearest E4M3 value of doubles, ties to the even mantissa."""
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), (e - 1).clamp(min=-6) - 3)
    return (torch.round(v / step) * step).clamp(-448, 448)


def _reference(x, rows):
    """(code values, scales) as doubles, block by block."""
    r, k = x.shape
    values, scales = torch.zeros((r, k), dtype=torch.float64), torch.zeros((-(-r // rows), -(-k // 128)), dtype=torch.float64)
    x = x.double().cpu()
    for i in range(scales.shape[0]):
        for b in range(scales.shape[1]):
            part = x[i * rows: (i + 1) * rows, 128 * b: 128 * b + 128]
            s = (part.abs().max() / 448).float().double()
            s = s if s != 0 else torch.ones((), dtype=torch.float64)
            scales[i, b] = s
            values[i * rows: (i + 1) * rows, 128 * b: 128 * b + 128] = _e4m3((part / s).float().double())
    return values, scales


def _expand(values, scales, rows):
    s = scales.double().repeat_interleave(rows, 0)[: values.shape[0]].repeat_interleave(128, 1)[:, : values.shape[1]]
    return values.double() * s


def _data(r, k, dtype, seed, spread=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((r, k), generator=g)
    if spread:
        x *= torch.exp(torch.randn((r, 1), generator=g)) * torch.exp(2 * torch.randn((1, k), generator=g))
    return x.to(dtype).cuda()


def _check_product(y, a, b, out_dtype):
    """Sums of 128 products by the tensor core, each addition off by a whole step at most (it may cut instead of round);
    the scale products, the additions of the blocks and the result are rounded."""
    ref = a.double() @ b.double().T
    room = a.double().abs() @ b.double().abs().T
    blocks = -(-a.shape[1] // 128)
    limit = (2 * 128 + blocks + 4) * 2.0 ** -24 * room + HALF_STEP[out_dtype] * ref.abs() + SUBNORMAL[out_dtype]
    over = ref.abs() > torch.finfo(out_dtype).max             # what the type cannot hold is an infinity in it
    assert (y[over].isinf() & (y[over] > 0).eq(ref[over] > 0)).all()
    worst = ((y.double() - ref).abs() / limit)[~over].max().item()
    assert worst <= 1.0, worst


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 128), (3, 127), (5, 129), (128, 256), (130, 1500), (2, 4096)])
def test_quantizers_match_the_definition(dtype, rows, k):
    x = _data(rows, k, dtype, 7 * rows + k)
    q = mx.quantize_fp8_activations(x)
    values, scales = _reference(x, 1)
    assert torch.equal(q.codes.double().cpu(), values) and torch.equal(q.scales.double().cpu(), scales)
    w = mx.quantize_fp8_weight(x)
    values, scales = _reference(x, 128)
    assert torch.equal(w.codes.double().cpu(), values) and torch.equal(w.scales.double().cpu(), scales)
    for what, per in ((q, 1), (w, 128)):
        for out in (torch.bfloat16, torch.float16, torch.float32):
            dense = mx.dequantize_fp8(what, out)
            plain = (what.codes.float() * _expand(torch.ones(rows, k, device="cuda"), what.scales, per).float()).to(out)
            assert torch.equal(dense, plain)


def test_quantizer_block_extremes():
    x = torch.zeros((6, 384), device="cuda")
    x[1, 5] = 1e-45                                          # the scale would be zero
    x[2, :128] = torch.linspace(-1e-38, 1e-38, 128)          # a subnormal scale
    x[3, 130] = 3.0e38
    x[4, 0], x[4, 300] = float("inf"), float("nan")
    x[5] = torch.arange(384) * 2.0 ** -12
    q = mx.quantize_fp8_activations(x)
    assert (q.scales[:2] == 1).all() and (q.codes[:2].float() == 0).all()
    values, scales = _reference(x[[2, 3, 5]], 1)
    assert torch.equal(q.codes.double().cpu()[[2, 3, 5]], values) and torch.equal(q.scales.double().cpu()[[2, 3, 5]], scales)
    assert q.scales[4, 0].isinf() and q.scales[4, 1] == 1 and q.scales[4, 2].isnan()
    w = mx.quantize_fp8_weight(torch.ones((4, 384), device="cuda"))
    y = mx.fp8_linear(x, w)
    assert y[4].isnan().all() and y[[0, 1, 2, 3, 5]].isfinite().all()


def test_quantizer_takes_strides_and_leaves_other_memory():
    base = torch.full((40, 700), 5.0, device="cuda")
    for view in (base[3:20, 1:300], base[::2, 100:400], base[:, 7:8], base.t()[10:20, :30]):
        a, b = mx.quantize_fp8_activations(view), mx.quantize_fp8_activations(view.contiguous())
        assert torch.equal(a.codes.float(), b.codes.float()) and torch.equal(a.scales, b.scales)
    x = _data(130, 200, torch.bfloat16, 3)
    codes = torch.full((132, 256), 0x55, dtype=torch.uint8, device="cuda")
    scales = torch.full((2, 256), -7.0, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    assert nat.lib().mixfp4_fp8_quantize_rows(x.data_ptr(), nat.BF16, 130, 200, 200, codes.data_ptr(), 256, scales.data_ptr(), 256, stream) == 0
    assert (codes[130:] == 0x55).all() and (codes[:130, 200:] == 0).all() and (scales[:, 130:] == -7).all() and (scales[:, :130] > 0).all()


SHAPES = [(1, 1, 1), (1, 128, 128), (1, 1024, 4096), (2, 130, 129), (7, 200, 1000), (16, 4096, 512), (17, 128, 14336), (32, 257, 300),
          (33, 1000, 2048), (64, 300, 4224), (65, 128, 128), (100, 384, 700), (129, 1000, 1500), (333, 515, 260), (777, 1024, 1024),
          (1024, 2048, 640), (2500, 2304, 384)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear_against_64_bits(m, n, k):
    x, w = _data(m, k, torch.bfloat16, m + k), _data(n, k, torch.bfloat16, n + k + 1)
    weight, q = mx.quantize_fp8_weight(w), mx.quantize_fp8_activations(x)
    a, b = _expand(q.codes, q.scales, 1), _expand(weight.codes, weight.scales, 128)
    for out in (torch.bfloat16, torch.float32) + ((torch.float16,) if m == 7 else ()):
        y = mx.fp8_linear(x, weight, out_dtype=out)
        assert y.shape == (m, n) and y.dtype == out
        _check_product(y, a, b, out)
        assert torch.equal(y, mx.fp8_linear(q, weight, out_dtype=out)), "quantized within the call or before it"
    assert mx.gemm_status() == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_linear_input_types_and_leading_dimensions(dtype):
    x, w = _data(30, 500, dtype, 1), _data(70, 500, torch.float32, 2)
    weight = mx.quantize_fp8_weight(w)
    q = mx.quantize_fp8_activations(x)
    y = mx.fp8_linear(x.reshape(2, 3, 5, 500), weight)
    assert y.shape == (2, 3, 5, 70) and y.dtype == dtype
    _check_product(y.reshape(30, 70), _expand(q.codes, q.scales, 1), _expand(weight.codes, weight.scales, 128), dtype)
    bias = torch.randn(70, device="cuda")
    assert torch.equal(mx.fp8_linear(x, weight, bias=bias), mx.fp8_linear(x, weight) + bias.to(dtype))
    assert torch.equal(mx.fp8_linear(x[0], weight), mx.fp8_linear(x[:1], weight)[0])
    assert mx.fp8_linear(x[:0], weight).shape == (0, 70)
    wide = torch.zeros((30, 777), dtype=dtype, device="cuda")
    wide[:, 5:505] = x
    assert torch.equal(mx.fp8_linear(wide[:, 5:505], weight), mx.fp8_linear(x, weight))
    assert torch.equal(mx.fp8_linear(x[:1].expand(4, 500), weight), mx.fp8_linear(x[:1], weight).expand(4, 70))


def test_linear_writes_nothing_but_its_rows():
    x, w = _data(70, 256, torch.bfloat16, 1), _data(130, 256, torch.bfloat16, 2)
    weight, q = mx.quantize_fp8_weight(w), mx.quantize_fp8_activations(x)
    for m in (3, 70):
        for ld in (130, 133, 160):
            y = torch.full((m + 2, ld), -9.0, dtype=torch.bfloat16, device="cuda")
            part = mx.quantize_fp8_activations(x[:m])
            rc = nat.lib().mixfp4_fp8_gemm(part.codes.data_ptr(), part.codes.stride(0), part.scales.data_ptr(), part.scales.stride(1),
                                           weight.codes.data_ptr(), weight.codes.stride(0), weight.scales.data_ptr(), m, 130, 256,
                                           y.data_ptr(), nat.BF16, ld, None, torch.cuda.current_stream().cuda_stream)
            assert rc == 0
            assert torch.equal(y[:m, :130], mx.fp8_linear(part, weight)) and (y[m:] == -9).all() and (y[:m, 130:] == -9).all()


def test_rows_do_not_depend_on_the_batch():
    """Within one arrangement a row's result is the same bits whatever stands beside it, and repeats of a call agree."""
    x, w = _data(64, 4096, torch.bfloat16, 5), _data(512, 4096, torch.bfloat16, 6)
    weight = mx.quantize_fp8_weight(w)
    y = mx.fp8_linear(x, weight, out_dtype=torch.float32)
    for _ in range(3):
        assert torch.equal(y, mx.fp8_linear(x, weight, out_dtype=torch.float32))
    perm = torch.randperm(64, device="cuda")
    assert torch.equal(mx.fp8_linear(x[perm], weight, out_dtype=torch.float32), y[perm])


def test_imported_tensors():
    w = _data(200, 300, torch.bfloat16, 9)
    weight = mx.quantize_fp8_weight(w)
    x = _data(20, 300, torch.bfloat16, 10)
    y = mx.fp8_linear(x, weight)
    dense = weight.codes.contiguous()                        # 300-byte rows: copied into aligned ones
    again = mx.FP8Weight.from_tensors(dense.view(torch.uint8), weight.scales.clone())
    assert again.codes.stride(0) % 16 == 0 and torch.equal(mx.fp8_linear(x, again), y)
    q = mx.quantize_fp8_activations(x)
    assert torch.equal(mx.fp8_linear(mx.FP8Activations.from_tensors(q.codes.contiguous(), q.scales.contiguous()), weight), y)
    assert torch.equal(q.dequantize(torch.float32), mx.dequantize_fp8(q, torch.float32))


def test_captured_and_on_another_stream():
    x, w = _data(5, 1024, torch.bfloat16, 1), _data(384, 1024, torch.bfloat16, 2)
    weight = mx.quantize_fp8_weight(w)
    want = mx.fp8_linear(x, weight)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, slots = [], [torch.zeros_like(x), torch.zeros_like(x)]
    with torch.cuda.stream(side):
        assert torch.equal(mx.fp8_linear(x, weight), want)
        torch.cuda.synchronize()
        for slot in slots:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                y = mx.fp8_linear(slot, weight)
            graphs.append((g, y))
    slots[0].copy_(x)
    slots[1].copy_(2 * x)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):                                      # two graphs of one stream's capture, at once
        for (g, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], want) and torch.equal(graphs[1][1], 2 * want)


def test_module_keeps_its_format():
    dense = torch.nn.Linear(300, 200, bias=True, device="cuda", dtype=torch.bfloat16)
    layer = mx.FP8Linear.from_linear(dense)
    x = _data(9, 300, torch.bfloat16, 4)
    y = layer(x)
    assert torch.equal(y, mx.fp8_linear(x, mx.quantize_fp8_weight(dense.weight), bias=dense.bias))
    layer = layer.half().cpu().cuda().bfloat16()
    assert layer.codes.dtype == torch.float8_e4m3fn and layer.scales.dtype == torch.float32
    assert torch.equal(layer(x), mx.fp8_linear(x, mx.quantize_fp8_weight(dense.weight), bias=layer.bias))
    other = mx.FP8Linear.from_linear(torch.nn.Linear(300, 200, device="cuda", dtype=torch.bfloat16))
    other.load_state_dict(layer.state_dict())
    assert torch.equal(other(x), layer(x))


def test_operands_rewritten_just_before_the_call():
    """The product starts under the tail of the kernel before it: whatever that writes, it is read as written."""
    k, n = 2048, 1500
    ws = [mx.quantize_fp8_weight(_data(n, k, torch.bfloat16, s)) for s in (1, 2)]
    held = mx.FP8Weight.from_tensors(ws[0].codes.clone(), ws[0].scales.clone())
    for m in (1, 20, 200, 1000):
        xs = [_data(m, k, torch.bfloat16, 10 + s) for s in (1, 2)]
        want = [mx.fp8_linear(x, w) for x, w in zip(xs, ws)]
        qs = [mx.quantize_fp8_activations(x) for x in xs]
        x, got = xs[0].clone(), []
        q = mx.FP8Activations.from_tensors(qs[0].codes.clone(), qs[0].scales.clone())
        torch.cuda.synchronize()
        for i in range(12):
            held.codes.copy_(ws[i % 2].codes)
            held.scales.copy_(ws[i % 2].scales)
            x.copy_(xs[i % 2])
            got.append(mx.fp8_linear(x, held))
            q.codes.copy_(qs[i % 2].codes)
            q.scales.copy_(qs[i % 2].scales)
            got.append(mx.fp8_linear(q, held))
        for i, y in enumerate(got):
            assert torch.equal(y, want[i // 2 % 2]), (m, i)


def test_a_weight_past_2_31_elements():
    n, k = 530000, 4096
    weight = mx.quantize_fp8_weight(torch.ones((n, k), dtype=torch.bfloat16, device="cuda").mul_(torch.arange(n, device="cuda").remainder_(7)[:, None] + 1))
    for m in (1, 70):
        x = _data(m, k, torch.bfloat16, m, spread=False)
        y = mx.fp8_linear(x, weight)
        tail = mx.FP8Weight.from_tensors(weight.codes[n - 208:], weight.scales[-2:])      # 530000 = 4140 * 128 + 80
        part = mx.fp8_linear(x, mx.quantize_fp8_weight(weight.dequantize(torch.bfloat16)[n - 80:]))
        q = mx.quantize_fp8_activations(x)
        _check_product(y[:, n - 80:], _expand(q.codes, q.scales, 1), _expand(weight.codes[n - 80:], weight.scales[-1:], 128), torch.bfloat16)
        assert part.shape == (m, 80) and tail.n == 208


def test_two_streams_at_once():
    weight = mx.quantize_fp8_weight(_data(3000, 1024, torch.bfloat16, 1))
    xs = [_data(m, 1024, torch.bfloat16, m) for m in (3, 50, 130, 600)]
    want = [mx.fp8_linear(x, weight) for x in xs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in xs], [[] for _ in xs]
    for _ in range(10):
        for x, st, out in zip(xs, streams, got):
            with torch.cuda.stream(st):
                out.append(mx.fp8_linear(x, weight))
    torch.cuda.synchronize()
    assert all(torch.equal(y, w) for out, w in zip(got, want) for y in out) and mx.gemm_status() == 0


def test_converted_model_and_checkpoint(tmp_path):
    class Tiny(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.up_proj, self.down_proj = torch.nn.Linear(256, 384, bias=False), torch.nn.Linear(384, 256)
            self.lm_head = torch.nn.Linear(256, 1000, bias=False)

        def forward(self, x):
            return self.lm_head(self.down_proj(torch.relu(self.up_proj(x))))

    torch.manual_seed(0)
    model = Tiny().to("cuda", torch.bfloat16)
    dense = {n: m.weight.detach().clone() for n, m in model.named_modules() if isinstance(m, torch.nn.Linear)}
    bias = model.down_proj.bias.detach().clone()
    rows = mx.quantize_model_weights(model, "oracle16", per_module_mode={"down_proj": "fp8", "lm_head": "fp8"})
    assert [(r["module_name"], r["format_granularity"]) for r in rows] == [("up_proj", "oracle16"), ("down_proj", "fp8"), ("lm_head", "fp8")]
    assert isinstance(model.up_proj, mx.MixFP4Linear) and isinstance(model.lm_head, mx.FP8Linear)
    x = _data(5, 256, torch.bfloat16, 3, spread=False)
    y = model(x)
    h = torch.relu(model.up_proj(x))
    h = mx.fp8_linear(h, mx.quantize_fp8_weight(dense["down_proj"]), bias=bias)
    assert torch.equal(y, mx.fp8_linear(h, mx.quantize_fp8_weight(dense["lm_head"])))
    path = str(tmp_path / "packed.pt")
    mx.save_packed(model, path)
    torch.manual_seed(1)
    other = Tiny().to("cuda", torch.bfloat16)
    assert set(mx.load_packed(other, path)) == {"up_proj", "down_proj", "lm_head"}
    assert torch.equal(other(x), y)


def test_refusals():
    x, weight = _data(4, 256, torch.bfloat16, 1), mx.quantize_fp8_weight(_data(64, 256, torch.bfloat16, 2))
    with pytest.raises(ValueError):
        mx.fp8_linear(x[:, :128], weight)
    with pytest.raises(TypeError):
        mx.fp8_linear(x, weight, out_dtype=torch.float64)
    with pytest.raises(TypeError):
        mx.fp8_linear(x.double(), weight, out_dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        mx.fp8_linear(x.cpu(), weight)
    with pytest.raises(ValueError):
        mx.FP8Weight.from_tensors(weight.codes, weight.scales[:, :1])
    with pytest.raises(TypeError):
        mx.FP8Weight.from_tensors(weight.codes, weight.scales.half())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n", [(40, 2051), (500, 2051), (1100, 2051), (500, 2048), (1100, 2064)])
def test_rows_of_y_at_any_offset_and_stride(m, n, dtype):
    """Few rows, one CTA a tile, CTA pairs: rows that are whole sectors and rows that are not; what lies between them stays."""
    k = 640
    x, w = _data(m, k, torch.bfloat16, 51), _data(n, k, torch.bfloat16, 52)
    q, weight = mx.quantize_fp8_activations(x), mx.quantize_fp8_weight(w)
    want = mx.fp8_linear(q, weight, out_dtype=dtype)
    _check_product(want, _expand(q.codes, q.scales, 1), _expand(weight.codes, weight.scales, 128), dtype)
    for offset, ldy in ((0, n), (1, n + 3), (0, -(-n // 32) * 32 + 32), (16, n + 1)):
        held = torch.full((offset + m * ldy + 64,), 7.0, dtype=dtype, device="cuda")
        status = nat.lib().mixfp4_fp8_gemm(q.codes.data_ptr(), q.codes.stride(0), q.scales.data_ptr(), q.scales.stride(1),
                                           weight.codes.data_ptr(), weight.codes.stride(0), weight.scales.data_ptr(), m, n, k,
                                           held[offset:].data_ptr(), nat.DTYPE_CODE[dtype], ldy, None,
                                           torch.cuda.current_stream().cuda_stream)
        assert status == 0
        rows = held[offset: offset + m * ldy].view(m, ldy)
        assert torch.equal(rows[:, :n], want), (offset, ldy)
        assert (held[:offset] == 7).all() and (rows[:, n:] == 7).all() and (held[offset + m * ldy:] == 7).all()


def test_outputs_past_2_31_elements():
    m, n, k = 17000, 128256, 128                             # 2.18e9 elements
    x, w = _data(m, k, torch.bfloat16, 61, spread=False), _data(n, k, torch.bfloat16, 62, spread=False)
    weight, q = mx.quantize_fp8_weight(w), mx.quantize_fp8_activations(x)
    y = mx.fp8_linear(q, weight)
    a, b = _expand(q.codes, q.scales, 1), _expand(weight.codes, weight.scales, 128)
    for rows, cols in ((slice(0, 3), slice(0, n)), (slice(m - 3, m), slice(0, n)), (slice(0, m), slice(n - 5, n))):
        _check_product(y[rows, cols], a[rows], b[cols], torch.bfloat16)


def _kernels(call):
    """What `call` returns, and the names of the kernels that it launched (none where the profiler is not to be had)."""
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA], acc_events=True) as prof:
        result = call()
        torch.cuda.synchronize()
    return result, [e.name for e in prof.events() if e.device_type == torch.autograd.DeviceType.CUDA]


@pytest.mark.parametrize("m,n,k,out,kernel", [
    (4096, 4099, 4096, torch.bfloat16, "fp8_pair_kernel"), (4096, 4099, 4096, torch.float32, "fp8_pair_kernel"),
    (2048, 4096, 4096, torch.bfloat16, "fp8_pair_kernel"), (2000, 4112, 4000, torch.float16, "fp8_pair_kernel"),
    (5000, 8200, 1100, torch.float32, "fp8_pair_kernel"), (1100, 8976, 2944, torch.bfloat16, "fp8_pair_kernel"),
    (1100, 9000, 2944, torch.bfloat16, "fp8_gemm_kernel<128, false, false>")])       # off its sectors pairs cost more
def test_many_blocks_and_tiles(m, n, k, out, kernel):
    """256 x 256 tiles of CTA pairs: their ring of stages wraps within a tile, a pair takes several tiles one after the other (4096 x 4099:
    272 tiles for 74 pairs), K ends inside a block, rows of y on their sectors and off them.  The kernel's name says that a case is still
    what it stands for."""
    x, w = _data(m, k, torch.bfloat16, m + k), _data(n, k, torch.bfloat16, n + k)
    q, weight = mx.quantize_fp8_activations(x), mx.quantize_fp8_weight(w)
    y, names = _kernels(lambda: mx.fp8_linear(q, weight, out_dtype=out))
    assert not names or any(kernel in name for name in names), names
    a, b = _expand(q.codes, q.scales, 1), _expand(weight.codes, weight.scales, 128)
    # What rounds to infinity is what lies half a step past the largest value: fp16 holds 65504, its next step would be 65536, so
    # everything below 65520 is 65504.  The sum's own error moves that border.
    largest = torch.finfo(out).max
    border = largest * (1 + HALF_STEP[out] / (2 - 2 * HALF_STEP[out]))      # (2 - 2h) 2^e is the largest, h 2^e half a step there
    ref, room = a @ b.T, (2 * 128 + -(-k // 128) + 4) * 2.0 ** -24 * (a.abs() @ b.abs().T)
    over = y.isinf()
    assert (ref[over].abs() + room[over] >= border).all() and ((y[over] > 0) == (ref[over] > 0)).all()
    assert ((y.double() - ref).abs()[~over] <= (room + HALF_STEP[out] * ref.abs() + SUBNORMAL[out])[~over]).all()
    assert torch.equal(mx.fp8_linear(x, weight, out_dtype=out), y) and mx.gemm_status() == 0


def test_tiles_and_columns_around_2_31_elements():
    """Codes and scales past element 2^31 (row 524288) are those of the rows by themselves, and so are the columns of a product."""
    n, k = 530000, 4096
    dense = torch.empty((n, k), dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(81))
    weight = mx.quantize_fp8_weight(dense)
    parts = {}
    for first, last in ((524288 - 128, 524288 + 128), (n - 208, n)):              # whole tiles: 530000 = 4139 * 128 + 208
        part = parts[first, last] = mx.quantize_fp8_weight(dense[first:last])
        assert torch.equal(weight.codes[first:last].view(torch.uint8), part.codes.view(torch.uint8))
        assert torch.equal(weight.scales[first // 128: -(-last // 128)], part.scales)
        for out in (torch.bfloat16, torch.float32):
            assert torch.equal(weight.dequantize(out)[first:last], part.dequantize(out))
    for m in (1, 70, 300):
        x = _data(m, k, torch.bfloat16, 82 + m, spread=False)
        q = mx.quantize_fp8_activations(x)
        y, a = mx.fp8_linear(x, weight), _expand(q.codes, q.scales, 1)
        for (first, last), part in parts.items():
            b = _expand(part.codes, part.scales, 128)
            _check_product(y[:, first:last], a, b, torch.bfloat16)
            _check_product(mx.fp8_linear(x, part), a, b, torch.bfloat16)
