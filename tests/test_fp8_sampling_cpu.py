"""What of the block-scaled FP8 linear and of token sampling needs no GPU: refusals, at the C boundary before any CUDA call and in
Python, and the converter's choice of layers."""

import copy
import ctypes
import os
import re

import pytest
import torch

import mixfp4_b200 as mx
from mixfp4_b200 import _native as nat
from mixfp4_b200 import convert, llama_decode

ONE = ctypes.c_void_p(64)       # never dereferenced: validation fails first
ODD = ctypes.c_void_p(66)


def _with(args, **changed):
    args = list(args)
    for at, value in changed.items():
        args[int(at[1:])] = value
    return args


def test_sizes():
    h = nat.lib()
    assert [h.mixfp4_fp8_scale_rows(m) for m in (-1, 0, 1, 128, 129)] == [0, 0, 128, 128, 256]
    assert h.mixfp4_fp8_workspace_bytes(1, 4096) == 0                       # quantized by the product itself
    assert h.mixfp4_fp8_workspace_bytes(100, 300) == 100 * 384 + 128 * 3 * 4
    assert h.mixfp4_fp8_workspace_bytes(0, 300) == 0 and h.mixfp4_sample_max_vocab() == 524160


def test_quantizers_refuse():
    h = nat.lib()
    rows = (ONE, nat.BF16, 4, 256, 256, ONE, 256, ONE, 128, None)
    for changed, status in (({"a0": None}, -1), ({"a5": None}, -1), ({"a7": None}, -1), ({"a1": 7}, -4), ({"a2": 0}, -2), ({"a3": 0}, -2),
                            ({"a4": 255}, -2), ({"a6": 240}, -2), ({"a8": 127}, -2), ({"a5": ODD}, -3), ({"a6": 264}, -3), ({"a7": ODD}, -3),
                            ({"a8": 130}, -3), ({"a3": 1 << 40, "a4": 1 << 40, "a6": 1 << 41}, -2)):
        assert h.mixfp4_fp8_quantize_rows(*_with(rows, **changed)) == status, changed
    tiles = (ONE, nat.BF16, 4, 256, 256, ONE, 256, ONE, None)
    for changed, status in (({"a0": None}, -1), ({"a7": None}, -1), ({"a1": -1}, -4), ({"a2": -3}, -2), ({"a4": 128}, -2), ({"a6": 128}, -2),
                            ({"a6": 264}, -3), ({"a5": ODD}, -3), ({"a7": ODD}, -3)):
        assert h.mixfp4_fp8_quantize_tiles(*_with(tiles, **changed)) == status, changed
    dequant = (ONE, 256, ONE, 2, 1, 128, 4, 256, ONE, nat.BF16, 256, None)
    for changed, status in (({"a0": None}, -1), ({"a8": None}, -1), ({"a5": 64}, -5), ({"a6": 0}, -2), ({"a1": 255}, -2), ({"a10": 255}, -2),
                            ({"a3": -1}, -2), ({"a9": 9}, -4)):
        assert h.mixfp4_fp8_dequant(*_with(dequant, **changed)) == status, changed


def test_products_refuse():
    h = nat.lib()
    gemm = (ONE, 256, ONE, 128, ONE, 256, ONE, 4, 64, 256, ONE, nat.BF16, 64, None, None)
    for changed, status in (({"a0": None}, -1), ({"a2": None}, -1), ({"a4": None}, -1), ({"a6": None}, -1), ({"a10": None}, -1), ({"a1": 255}, -2),
                            ({"a3": 4}, -2), ({"a5": 128}, -2), ({"a7": 0}, -2), ({"a8": 0}, -2), ({"a9": 0}, -2), ({"a12": 63}, -2), ({"a11": 5}, -4),
                            ({"a0": ODD}, -3), ({"a1": 264}, -3), ({"a4": ODD}, -3), ({"a5": 264}, -3), ({"a6": ODD}, -3), ({"a2": ODD}, -3),
                            ({"a7": 1 << 31}, -2)):
        assert h.mixfp4_fp8_gemm(*_with(gemm, **changed)) == status, changed
    linear = (ONE, nat.BF16, 100, 300, ONE, 304, ONE, 64, 300, ONE, nat.F32, 64, ONE, 1 << 20, None, None)
    for changed, status in (({"a0": None}, -1), ({"a1": 7}, -4), ({"a3": 299}, -2), ({"a4": None}, -1), ({"a5": 300}, -3), ({"a9": None}, -1),
                            ({"a12": None}, -7), ({"a13": 1000}, -7), ({"a12": ODD}, -3), ({"a10": 7}, -4)):
        assert h.mixfp4_fp8_linear(*_with(linear, **changed)) == status, changed
    few = _with(linear, a2=1, a12=None, a13=0)               # no workspace, but the same checks
    for changed, status in (({"a0": None}, -1), ({"a1": 7}, -4), ({"a3": 299}, -2), ({"a5": 300}, -3)):
        assert h.mixfp4_fp8_linear(*_with(few, **changed)) == status, changed


def test_sampling_refuses():
    h = nat.lib()
    args = (ONE, nat.F32, 2, 100, 100, ONE, None, 1.0, None, 0, None, 1.0, None, 0.0, ONE, None, None)
    for changed, status in (({"a0": None}, -1), ({"a5": None}, -1), ({"a14": None}, -1), ({"a2": 0}, -2), ({"a3": 0}, -2), ({"a4": 99}, -2),
                            ({"a3": 600000, "a4": 600000}, -10), ({"a1": 4}, -4), ({"a0": ODD}, -3), ({"a5": ODD}, -3), ({"a14": ODD}, -3),
                            ({"a2": 1 << 31}, -2)):
        assert h.mixfp4_sample(*_with(args, **changed)) == status, changed


def test_pointers_off_their_element_are_refused():
    h = nat.lib()
    off2, off4 = ctypes.c_void_p(65), ctypes.c_void_p(66)
    for dtype, off in ((nat.BF16, off2), (nat.F16, off2), (nat.F32, off4)):
        assert h.mixfp4_fp8_quantize_rows(off, dtype, 4, 256, 256, ONE, 256, ONE, 128, None) == -3
        assert h.mixfp4_fp8_quantize_tiles(off, dtype, 4, 256, 256, ONE, 256, ONE, None) == -3
        assert h.mixfp4_fp8_dequant(ONE, 256, ONE, 2, 1, 128, 4, 256, off, dtype, 256, None) == -3
        assert h.mixfp4_fp8_gemm(ONE, 256, ONE, 128, ONE, 256, ONE, 4, 64, 256, off, dtype, 64, None, None) == -3
        for m in (1, 1000):                                  # quantized by the product, and ahead of it
            assert h.mixfp4_fp8_linear(off, dtype, m, 256, ONE, 256, ONE, 64, 256, ONE, nat.F32, 64, ONE, 1 << 20, None, None) == -3
            assert h.mixfp4_fp8_linear(ONE, nat.F32, m, 256, ONE, 256, ONE, 64, 256, off, dtype, 64, ONE, 1 << 20, None, None) == -3
    assert h.mixfp4_fp8_dequant(ONE, 256, off4, 2, 1, 128, 4, 256, ONE, nat.BF16, 256, None) == -3
    args = (ONE, nat.F32, 2, 100, 100, ONE, None, 1.0, None, 0, None, 1.0, None, 0.0, ONE, None, None)
    for at in (0, 5, 6, 8, 10, 12, 15):
        assert h.mixfp4_sample(*_with(args, **{f"a{at}": off4})) == -3, at


def test_python_refusals():
    x = torch.zeros((2, 8))
    for call in (lambda: mx.quantize_fp8_weight(x), lambda: mx.quantize_fp8_activations(x), lambda: mx.sample_logits(x, torch.zeros(2))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    with pytest.raises(ValueError):
        mx.quantize_fp8_weight(torch.zeros(8))
    codes, scales = torch.zeros((200, 300), dtype=torch.uint8), torch.ones((2, 3))
    weight = mx.FP8Weight.from_tensors(codes, scales)        # a container may live on the host
    assert weight.codes.shape == (200, 300) and weight.codes.stride(0) == 384 and weight.nbytes() == 200 * 300 + 24
    for bad in ((codes, scales[:1]), (codes[0], scales), (codes[:0], scales)):
        with pytest.raises(ValueError):
            mx.FP8Weight.from_tensors(*bad)
    for bad in ((codes.float(), scales), (codes, scales.half())):
        with pytest.raises(TypeError):
            mx.FP8Weight.from_tensors(*bad)
    with pytest.raises(RuntimeError, match="CUDA"):
        mx.fp8_linear(torch.zeros((2, 300)), weight)
    with pytest.raises(ValueError):
        mx.fp8_linear(torch.zeros((2, 299)), weight)


def test_parts_that_the_kernels_cannot_read_are_refused():
    codes, scales = torch.zeros((200, 384), dtype=torch.float8_e4m3fn), torch.ones((2, 3))
    assert mx.FP8Weight(codes, scales).n == 200
    for bad in ((codes[:, ::2], scales[:, :2]), (codes, torch.ones((3, 2)).t()), (codes, torch.ones((2, 6))[:, ::2]), (codes, scales[:, :2]),
                (codes.view(torch.uint8)[:, 1:].view(torch.float8_e4m3fn), scales), (codes[:, :300].contiguous(), scales)):
        with pytest.raises(ValueError):
            mx.FP8Weight(*bad)
        if bad[1].shape == (-(-bad[0].shape[0] // 128), -(-bad[0].shape[1] // 128)):
            assert mx.FP8Weight.from_tensors(*bad).codes.stride(0) % 16 == 0
    rows = torch.zeros((5, 384), dtype=torch.float8_e4m3fn)
    good = mx.FP8Activations.from_tensors(rows, torch.ones((5, 3)))
    shape, kind = torch.Size((5, 384)), torch.bfloat16
    assert mx.FP8Activations(rows, good.scales, shape, kind).shape == shape
    assert mx.FP8Activations(rows, good.scales, torch.Size((1, 5, 384)), kind).codes.shape == (5, 384)
    wide = torch.ones((3, 256)).t()
    for bad in ((rows, torch.ones((5, 3)), shape), (rows, wide[:10:2], shape), (rows, torch.ones((3, 130)).t()[:5], shape),
                (rows, wide[1:6], shape), (rows, wide[252:], shape), (rows, good.scales, torch.Size((6, 384))), (rows, good.scales.double(), shape),
                (rows, good.scales, torch.Size((5, 300))), (rows[:4], good.scales, shape), (rows[:, ::2], good.scales[:, :2], shape)):
        with pytest.raises((ValueError, TypeError)):
            mx.FP8Activations(*bad, kind)
    assert mx.FP8Activations.from_tensors(rows[:0], torch.ones((0, 3))).shape == (0, 384)


def test_a_layer_follows_its_buffers():
    layer = mx.FP8Linear(mx.FP8Weight.from_tensors(torch.zeros((200, 300), dtype=torch.uint8), torch.ones((2, 3))))
    weight = layer.weight_fp8
    assert layer.weight_fp8 is weight and copy.deepcopy(layer).weight_fp8 is not weight
    packed = torch.ones((200, 300), dtype=torch.uint8).view(torch.float8_e4m3fn)             # rows off their 16 bytes
    layer.load_state_dict({"codes": packed, "scales": torch.full((2, 3), 2.0)}, assign=True)
    assert layer.weight_fp8 is not weight and layer.weight_fp8.codes.stride(0) == 384
    assert torch.equal(layer.weight_fp8.codes.view(torch.uint8), packed.view(torch.uint8)) and (layer.scales == 2).all()
    layer.half()
    assert layer.codes.dtype == torch.float8_e4m3fn and layer.scales.dtype == torch.float32


def test_converter_refuses_names_that_are_no_linear():
    model = torch.nn.Sequential(torch.nn.Linear(16, 16), torch.nn.ReLU())
    for name in ("1", "missing"):
        with pytest.raises(KeyError):
            mx.quantize_model_weights(model, "bf16", per_module_mode={name: "fp8"})
    assert mx.quantize_model_weights(model, "bf16") == []


def test_the_sampler_meets_its_cluster_before_it_writes_to_a_peer():
    """A peer's shared memory may be touched once the peer is known to have started: in the order of the code the cluster's first
    barrier is complete ahead of every access to a peer's memory.  (A CTA that is not running yet cannot be had on demand.)"""
    with open(os.path.join(os.path.dirname(mx.__file__), "csrc", "sample.cu")) as f:
        text = f.read()
    run = text[text.index("void run(int64_t r)"): text.index("sample_kernel(const SampleArgs a)")]
    run = re.sub(r"//[^\n]*", "", run)
    remote = re.search(r"\b(st_rank\d+|ld_rank\d+|add_rank\d+|find|choose_from_few)\(", run).start()
    complete = re.search(r"\b(all_started|meet)\(", run).start()
    assert complete < remote
    if run[complete:].startswith("all_started"):
        assert 0 <= run.find("started(ranks);") < run.index("griddepcontrol.wait") < complete


@pytest.mark.parametrize("filters", [["--top-k", "50"], ["--top-p", "0.9"], ["--min-p", "0.1"], ["--top-k", "0", "--top-p", "0.5"]])
def test_harness_refuses_filters_without_a_temperature(filters, monkeypatch, capsys):
    """Without a temperature no token is drawn: a filter would be dropped in silence."""
    monkeypatch.setattr("sys.argv", ["llama_decode", *filters])
    with pytest.raises(SystemExit):
        llama_decode.main()
    assert "--temperature" in capsys.readouterr().err


def test_converter_refuses_modes_before_it_converts():
    """A mode that does not exist, wherever it stands: no layer ahead of it has been replaced."""
    for args, kwargs in ((("oracle16",), dict(per_module_mode={"2": "fp4"})), (("fp9",), {}), (("fp9",), dict(per_module_mode={"0": "fp8"})),
                         (("fp8",), dict(per_module_mode={"2": "oracle17"}))):
        model = torch.nn.Sequential(torch.nn.Linear(16, 16), torch.nn.ReLU(), torch.nn.Linear(16, 16))
        held = list(model)
        with pytest.raises(ValueError, match="unsupported mode"):
            mx.quantize_model_weights(model, *args, **kwargs)
        assert all(a is b for a, b in zip(model, held))
    assert mx.quantize_model_weights(model, "fp9", per_module_mode={"0": "bf16", "2": "fp16"}) == []     # a mode that no layer takes


def test_checkpoints_with_fp8_layers_carry_a_version_of_their_own():
    """A reader that knows packed layers alone refuses the whole file instead of failing at such an entry, half-way through the model."""
    weight = mx.FP8Weight.from_tensors(torch.randint(0, 100, (200, 300), dtype=torch.uint8), torch.rand((2, 3)))
    model = torch.nn.Sequential(torch.nn.Linear(300, 200), mx.FP8Linear(weight, torch.rand(200)))
    state = convert.packed_state(model)
    assert state["version"] == 2 and list(state["layers"]) == ["1"]
    assert convert.packed_state(torch.nn.Sequential(torch.nn.ReLU()))["version"] == 1
    for version in (1, 2):                                   # 1: as such checkpoints were written at first
        other = torch.nn.Sequential(torch.nn.Linear(300, 200), torch.nn.Linear(300, 200))
        assert mx.load_packed(other, dict(state, version=version), device="cpu") == ["1"]
        assert torch.equal(other[1].codes.view(torch.uint8), model[1].codes.view(torch.uint8))
        assert torch.equal(other[1].scales, model[1].scales) and torch.equal(other[1].bias, model[1].bias)
    for version in (0, 3, None):
        with pytest.raises(ValueError, match="version"):
            mx.load_packed(other, dict(state, version=version), device="cpu")
