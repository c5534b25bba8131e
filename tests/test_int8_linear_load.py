"""KLinearInt8's weights: what a directory of safetensors and what the caller may hand over, and what is refused."""
from types import SimpleNamespace

import pytest
import torch

from ktransformers_b200.operators.linear import KLinearInt8, KTransformersLinear, int8_linear
from ktransformers_b200.util.custom_loader import SafeTensorLoader
from ktransformers_b200.util.utils import InferenceState

N, K = 6, 40
SHAPE = SimpleNamespace(in_features=K, out_features=N)


def saved(path, **tensors):
    from safetensors.torch import save_file
    save_file({f"blk.{name}": t.contiguous() for name, t in tensors.items()}, str(path / "model.safetensors"))
    return SafeTensorLoader(str(path))


def floats():
    return torch.randn((N, K), generator=torch.Generator().manual_seed(1))


# ------------------------------------------------------------------------------------------------------------------------- CPU (refused ahead of the first copy to a GPU)
@pytest.mark.parametrize("name", ["weight_scale", "weight_scale_inv"])
@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.bfloat16, torch.float32])
def test_scales_of_other_formats_are_no_biases(tmp_path, dtype, name):
    lin = KLinearInt8("blk", saved(tmp_path, weight=floats().to(dtype), **{name: torch.rand(N)}), None, SHAPE)
    with pytest.raises(ValueError, match="KLinearInt8"):
        lin.load(device="cuda")
    assert not lin.loaded and lin.weight is None


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.float8_e5m2, torch.uint8, torch.int16, torch.int64])
def test_weights_of_other_types_are_refused(tmp_path, dtype):
    w = floats().to(dtype)
    for lin, given in ((KLinearInt8("blk", saved(tmp_path, weight=w), None, SHAPE), None), (KLinearInt8("blk", None, None, SHAPE), (w, torch.rand(N))), (KLinearInt8("blk", None, None, SHAPE), w)):
        with pytest.raises(ValueError, match="KLinearInt8"):
            lin.load(given, device="cuda")


def test_float_weights_take_a_bias_and_nothing_else():
    for given in ((floats(), torch.rand(N, 1)), (floats(), torch.rand(N + 1)), (floats(), torch.rand(N), torch.rand(N)), (floats().t(),), (floats()[:, 1:],)):
        with pytest.raises(ValueError, match="KLinearInt8"):
            KLinearInt8("blk", None, None, SHAPE).load(given, device="cuda")


def test_an_int8_weight_without_its_scales_is_refused(tmp_path):
    with pytest.raises(KeyError, match="blk.weight_scale"):
        KLinearInt8("blk", saved(tmp_path, weight=torch.zeros((N, K), dtype=torch.int8)), None, SHAPE).load(device="cuda")


# ------------------------------------------------------------------------------------------------------------------------- GPU
@pytest.mark.gpu
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("kind", ["int8", "int8 column", "bf16", "fp16", "fp32"])
def test_a_checkpoint_stands_for_its_weights(tmp_path, kind, bias):
    """against the product in 64 bits: a code is half a step off, 1 / 254 of its row's largest value on either side"""
    w, b = floats(), {"bias": torch.randn(N)} if bias else {}
    if kind.startswith("int8"):
        codes, scale = KLinearInt8.quantize(w)
        w = codes.double() * scale.double()[:, None]
        ld = saved(tmp_path, weight=codes, weight_scale=scale[:, None] if kind == "int8 column" else scale, **b)
        half = torch.zeros((), dtype=torch.float64)
    else:
        w = w.to({"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}[kind])
        ld, w = saved(tmp_path, weight=w, **b), w.double()
        half = w.abs().amax(1) / 254
    lin = KTransformersLinear("blk", ld, None, torch.nn.Linear(K, N, bias=False), generate_op="KLinearInt8", prefill_op="None")
    lin.load(mode=InferenceState.GENERATE)
    x = torch.randn((5, K), generator=torch.Generator().manual_seed(2))
    y, xd = lin(x.cuda()).cpu().double(), x.double()
    ref = xd @ w.T + (b["bias"].double() if bias else 0.0)
    # |x w - x' w'| <= |x| |w - w'| + |x - x'| (|w| + |w - w'|), summed over K; 1 % for the scales' own roundings
    x_half = xd.abs().amax(1, keepdim=True) / 254
    bound = 1.01 * (xd.abs().sum(1, keepdim=True) * half + x_half * (w.abs().sum(1) + K * half)) + 2.0 ** -20 * (ref.abs() + 1)
    assert ((y - ref).abs() <= bound).all() and lin.generate_linear.has_bias == bias


@pytest.mark.gpu
@pytest.mark.parametrize("rows,T", [(64, 1), (2000, 5), (7168, 20), (2000, 200)])
def test_weights_made_on_the_stream_just_ahead(rows, T):
    """The int8 weight is the bytes of another integer linear's result, whose kernel lets its dependents start before it is done; then bytes that are copied over them"""
    g = torch.Generator().manual_seed(rows)
    rn = lambda *shape: torch.randn(shape, generator=g).cuda()
    many, scale, x = [rn(rows, 512) for _ in range(4)], torch.ones(rows, device="cuda"), rn(T, 1024).bfloat16()
    w1, s1 = KLinearInt8.quantize(rn(512, 512))
    made = [int8_linear(m.bfloat16(), w1, s1).view(torch.int8) for m in many]      # [rows, 1024]: bytes of bf16 numbers
    torch.cuda.synchronize()
    want = [int8_linear(x, w, scale) for w in made]
    torch.cuda.synchronize()
    got = [int8_linear(x, int8_linear(m.bfloat16(), w1, s1).view(torch.int8), scale) for m in many]
    weight, copied = torch.empty_like(made[0]), []
    for w in made:
        weight.copy_(w)
        copied.append(int8_linear(x, weight, scale))
    assert all(torch.equal(a, b) for a, b in zip(got + copied, want + want)) and not torch.equal(want[0], want[1])
