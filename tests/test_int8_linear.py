"""The 8-bit integer linear: codes, exact sums, scales, strides and refusals, against 64-bit forms."""
import ctypes as C
import math
from types import SimpleNamespace

import pytest
import torch

from ktransformers_b200 import native
from ktransformers_b200.operators.linear import LINEAR_MAP, KLinearInt8, KTransformersLinear, int8_linear
from ktransformers_b200.util.utils import InferenceState

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def codes_of(x):
    """(codes, scales) of rows, as the format defines them: the scale and the quotient are numbers of 32 bits"""
    x = x.float()
    s = x.abs().amax(1) * (torch.ones(()) / 127)      # (times the rounded inverse)
    return torch.where(s[:, None] > 0, torch.round(x / s[:, None]), torch.zeros(())).clamp(-127, 127).to(torch.int64), s


def reference(x, w, ws, bias=None):
    c, s = codes_of(x)
    y = (c.double() @ w.double().T) * (s.double()[:, None] * ws.double())      # (products of at most 2^14 and sums below 2^53: exact)
    return y if bias is None else y + bias.double()


def inputs(T, K, N, dtype, seed=0, bias=True):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(T, K, generator=g) * torch.exp(torch.randn(T, 1, generator=g))).to(DT[dtype])
    w = torch.randint(-128, 128, (N, K), generator=g, dtype=torch.int8)
    return x, w, torch.rand(N, generator=g) * 1e-2, torch.randn(N, generator=g) if bias else None


def padded(w, extra=0):
    """on the GPU, rows at multiples of 16 bytes"""
    N, K = w.shape
    out = torch.full((N, (K + 15) // 16 * 16 + extra), 77, dtype=torch.int8, device="cuda")      # (what lies between rows is not read as weights)
    out[:, :K] = w.cuda()
    return out[:, :K]


def check(y, ref, x, w, ws, bias):
    """float(acc) and three products or sums are rounded to 32 bits, then once to the type"""
    c, s = codes_of(x)
    prod = ref - bias.double() if bias is not None else ref
    tol = HALF_STEP[x.dtype] * ref.abs() * (1 + 2.0 ** -6) + 4 * 2.0 ** -24 * (prod.abs() + ref.abs()) + (2.0 ** -25 if x.dtype == torch.float16 else 0.0)
    assert y.dtype == x.dtype and ((y.cpu().double() - ref).abs() <= tol).all()


# ------------------------------------------------------------------------------------------------------------------------- CPU
GOOD = dict(x=16, x_stride=64, weight=16, weight_stride=64, weight_scale=16, in_features=64, out_features=8, hidden_type=native.GGML_BF16, y=16, y_stride=8)


@pytest.mark.parametrize("bad", [dict(in_features=0), dict(out_features=0), dict(hidden_type=12), dict(in_features=200000, x_stride=200000, weight_stride=200000), dict(x_stride=63), dict(y_stride=7),
                                 dict(weight_stride=48), dict(weight_stride=72), dict(weight=8), dict(x=None), dict(weight_scale=None), dict(y=None)])
def test_refuses(bad):
    a = native.Int8LinearParams(**{**GOOD, **bad})
    assert native.lib().ktb200_int8_linear(C.byref(a), 1, 16, 1 << 20, None) == native.EINVAL
    assert b"int8_linear" in native.lib().ktb200_last_error()


def test_refuses_workspaces_and_takes_no_tokens():
    lib, a = native.lib(), native.Int8LinearParams(**GOOD)
    need = lib.ktb200_int8_linear_workspace(3, 64)
    assert need >= 3 * 64 + 12 and lib.ktb200_int8_linear_workspace(0, 64) == 0
    for ws, n in ((None, need), (24, need), (16, need - 1)):
        assert lib.ktb200_int8_linear(C.byref(a), 3, ws, n, None) == native.EINVAL
    assert lib.ktb200_int8_linear(None, 3, 16, need, None) == native.EINVAL
    assert lib.ktb200_int8_linear(C.byref(a), 0, None, 0, None) == native.OK


def test_wrapper_refuses_cpu_tensors():
    with pytest.raises(ValueError, match="CUDA tensors only"):
        int8_linear(torch.zeros(2, 16), torch.zeros(4, 16, dtype=torch.int8), torch.ones(4))


def test_weights_are_quantised_row_by_row():
    w = torch.randn(5, 40)
    w[3] = 0
    codes, scale = KLinearInt8.quantize(w)
    assert codes.dtype == torch.int8 and (codes[3] == 0).all() and scale[3] == 0
    assert ((codes.double() * scale.double()[:, None] - w.double()).abs() <= 0.5001 * scale.double()[:, None]).all()
    assert LINEAR_MAP["KLinearInt8"] is KLinearInt8


def test_linear_refuses_weights_that_do_not_fit():
    lin = KLinearInt8("k", None, None, SimpleNamespace(in_features=32, out_features=4))
    for w in ((torch.zeros(4, 31, dtype=torch.int8), torch.ones(4)), (torch.zeros(4, 32, dtype=torch.int8), torch.ones(3)), (torch.zeros(4, 32, dtype=torch.int8),),
              (torch.zeros(4, 32, dtype=torch.int8), torch.ones(4), torch.ones(5))):
        with pytest.raises(ValueError):
            lin.load(w, device="cuda:0" if torch.cuda.is_available() else "cuda")
    with pytest.raises(native.KTB200Error, match="Not Loaded"):
        lin.forward(torch.zeros(1, 32))


# ------------------------------------------------------------------------------------------------------------------------- GPU
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T,K,N", [(1, 16, 1), (1, 1, 1), (3, 7, 130), (140, 1, 9500), (1, 2048, 2048), (1, 5000, 129), (2, 7168, 576), (3, 33, 7), (5, 128, 128), (8, 1536, 1000), (16, 640, 333), (17, 4096, 130), (31, 272, 2112),
                                   (64, 1024, 257), (65, 144, 512), (100, 2000, 384), (128, 512, 2000), (129, 256, 128), (257, 1040, 1025), (500, 130, 260), (1200, 384, 777)])
def test_int8_linear(T, K, N, dtype):
    x, w, ws, bias = inputs(T, K, N, dtype, seed=T + K, bias=T % 2 == 1)
    y = int8_linear(x.cuda(), padded(w), ws.cuda(), bias.cuda() if bias is not None else None)
    check(y, reference(x, w, ws, bias), x, w, ws, bias)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 20, 200])
def test_int8_linear_reads_rows_anywhere(T):
    x, w, ws, bias = inputs(T, 300, 70, "bf16", seed=1)
    wide = torch.full((T, 311), math.nan, dtype=x.dtype, device="cuda")
    wide[:, 5:305] = x.cuda()      # rows that begin at no whole vector, NaN around them
    y = int8_linear(wide[:, 5:305], padded(w, 32), ws.cuda(), bias.cuda())
    check(y, reference(x, w, ws, bias), x, w, ws, bias)
    three = int8_linear(x.cuda().view(1, T, 300), padded(w), ws.cuda(), bias.cuda())
    assert three.shape == (1, T, 70) and torch.equal(three[0], y)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [4, 40, 300])
def test_int8_linear_rows_of_zeros_infinities_and_nan(T):
    x, w, ws, bias = inputs(T, 256, 96, "fp32", seed=2)
    x[0], x[1, 7], x[2, 9], x[3] = 0, math.inf, math.nan, x[3] * 1e-42      # (a row of subnormal numbers, whose scale is one too)
    y = int8_linear(x.cuda(), padded(w), ws.cuda(), bias.cuda()).cpu()
    assert torch.equal(y[0], bias) and y[1].isnan().all() and y[2].isnan().all()
    keep = [0] + list(range(3, T))
    ref = reference(x[keep], w, ws, bias)
    check(y[keep], ref, x[keep], w, ws, bias)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [7, 48, 260])
def test_int8_linear_leaves_rows_behind_the_batch(T):
    x, w, ws, bias = inputs(T, 512, 200, "bf16", seed=3)
    full = int8_linear(x.cuda(), padded(w), ws.cuda(), bias.cuda())
    lib, wp = native.lib(), padded(w)
    xd, wsd, bd = x.cuda(), ws.cuda(), bias.cuda()
    n = lib.ktb200_int8_linear_workspace(T, 512)
    for live in (0, 1, T // 2, T, T + 9):
        y = torch.full((T, 208), 5.0, dtype=torch.bfloat16, device="cuda")
        bsz, scratch = torch.tensor([live], dtype=torch.int32, device="cuda"), torch.empty(n, dtype=torch.uint8, device="cuda")
        a = native.Int8LinearParams(xd.data_ptr(), 512, wp.data_ptr(), wp.stride(0), wsd.data_ptr(), bd.data_ptr(), 512, 200, native.GGML_BF16, y.data_ptr(), 208, bsz.data_ptr())
        native.check(lib.ktb200_int8_linear(C.byref(a), T, scratch.data_ptr(), n, torch.cuda.current_stream().cuda_stream))
        m = min(live, T)
        assert torch.equal(y[:m, :200], full[:m]) and (y[m:] == 5).all() and (y[:, 200:] == 5).all()


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 30, 400])
def test_int8_linear_gives_the_same_bits_each_time_on_any_stream_and_in_a_graph(T):
    x, w, ws, _ = inputs(T, 1600, 1030, "bf16", seed=4)
    xd, wd, sd = x.cuda(), padded(w), ws.cuda()
    first = int8_linear(xd, wd, sd)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(5):
        for st in streams:
            with torch.cuda.stream(st):
                outs.append(int8_linear(xd, wd, sd))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = int8_linear(xd, wd, sd)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(first, o) for o in outs + [captured])


@pytest.mark.gpu
def test_extreme_sums_are_exact():
    K = 16384
    x = torch.ones(2, K)
    x[1] = -1
    w = torch.full((3, K), 127, dtype=torch.int8)
    w[1], w[2, ::2] = -128, -127
    y = int8_linear(x.cuda(), w.cuda(), torch.ones(3, device="cuda"))
    s = torch.ones(()) / 127
    want = torch.tensor([[127 * 127 * K, -127 * 128 * K, 0], [-127 * 127 * K, 127 * 128 * K, 0]]).float() * s
    assert torch.equal(y.cpu(), want)


@pytest.mark.gpu
def test_klinear_int8_through_the_linear_module():
    g = torch.Generator().manual_seed(6)
    orig = torch.nn.Linear(40, 24, bias=False)
    wf, x = torch.randn(24, 40, generator=g), torch.randn(2, 3, 40, generator=g)
    lin = KTransformersLinear("blk", None, None, orig, generate_op="KLinearInt8", prefill_op="None")
    lin.load(w=(wf, torch.arange(24.0)), mode=InferenceState.GENERATE)      # (rows of 40: padded to 48 where they are kept)
    codes, scale = KLinearInt8.quantize(wf)
    check(lin(x.cuda()).reshape(6, 24), reference(x.reshape(6, 40), codes, scale, torch.arange(24.0)), x.reshape(6, 40), codes, scale, torch.arange(24.0))
    lin.load(mode=InferenceState.UNLOAD)


@pytest.mark.gpu
def test_wrapper_refuses_what_does_not_fit():
    x, w, s = torch.zeros(2, 32, device="cuda"), torch.zeros(4, 32, dtype=torch.int8, device="cuda"), torch.ones(4, device="cuda")
    limit = torch.ones(1, dtype=torch.int32, device="cuda")
    assert int8_linear(x, w, s, s, limit).shape == (2, 4)
    for call in ((x[:, :31], w, s), (x.double(), w, s), (x, w.float(), s), (x, w.t().contiguous().t(), s), (x, w[:, 1:], s), (x, w, s[:3]), (x, w, s.half()), (x, w, s.cpu()), (x, w, s, s[:3]), (x, w, s, s.half()),
                 (x, w, s, s.cpu()), (x, w, s, None, limit.long()), (x, w, s, None, limit.cpu()), (x, w, s, None, limit[:0]), (x, torch.zeros(4, 40, dtype=torch.int8, device="cuda")[:, :32], s)):
        with pytest.raises(ValueError, match="int8_linear"):
            int8_linear(*call)
