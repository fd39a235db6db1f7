"""Products with 4-bit weights on the GPU against the formula in 64 bits."""
import pytest
import torch

from atorch_b200 import _lib, ops
from atorch_b200.ops import w4

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _weights(N, K, group, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    codes = torch.randint(0, 256, (N, -(-K // 32) * 16), generator=g, device=DEV, dtype=torch.uint8)
    scales = (torch.randn(N, -(-K // group), generator=g, device=DEV) * 0.01).bfloat16()
    return codes, scales, g


def _weight64(codes, scales, K, group):
    w = torch.empty(codes.shape[0], 2 * codes.shape[1], dtype=torch.float64, device=DEV)
    w[:, 0::2], w[:, 1::2] = (codes & 15).double(), (codes >> 4).double()
    return (w[:, :K] - 8) * scales.double().repeat_interleave(group, 1)[:, :K]


def _check(x, codes, scales, group, bias=None, weight_rounded=False):
    K = x.shape[-1]
    y = ops.w4_linear(x, codes, scales, group, bias)
    assert torch.equal(y, ops.w4_linear(x, codes, scales, group, bias))
    w, xd = _weight64(codes, scales, K, group), x.reshape(-1, K).double()
    want = xd @ w.t() + (0 if bias is None else bias.double())
    size = xd.abs() @ w.abs().t() + (0 if bias is None else bias.double().abs())
    # the result is rounded once; products are exact, and up to 2^7 fp32 sums (cut off at 22 bits) follow one another
    unit = 2.0 ** -8 if x.dtype == torch.bfloat16 else 2.0 ** -11
    tol = unit * 1.01 * want.abs() + 2.0 ** -15 * size + (2.0 ** -8 * size if weight_rounded else 0) + 2.0 ** -25
    assert y.shape == (*x.shape[:-1], codes.shape[0]) and y.dtype == x.dtype
    assert ((y.view_as(want).double() - want).abs() <= tol).all(), ((y.view_as(want).double() - want).abs() / tol).max()
    _lib.check_status(y.device)
    return y


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 4096, 4096), (1, 17, 31), (2, 64, 33), (3, 100, 129), (8, 256, 1000), (9, 33, 2048),
                                   (16, 1000, 1111), (17, 48, 264), (31, 333, 640), (32, 16, 11008), (33, 80, 96), (70, 50, 77)])
def test_product(M, N, K, group, dtype):
    codes, scales, g = _weights(N, K, group, M + N + K)
    x = torch.randn(M, K, generator=g, device=DEV).to(dtype)
    _check(x, codes, scales, group, torch.randn(N, generator=g, device=DEV).to(dtype) if M % 2 else None)


@pytest.mark.parametrize("M,N,K,dtype", [(65, 384, 512, torch.bfloat16), (300, 1000, 520, torch.bfloat16), (100, 64, 512, torch.float16),
                                         (128, 70000, 64, torch.bfloat16)])
def test_many_rows(M, N, K, dtype):
    codes, scales, g = _weights(N, K, 64)
    x = torch.randn(M, K, generator=g, device=DEV).to(dtype)
    _check(x, codes, scales, 64, torch.randn(N, generator=g, device=DEV).to(dtype), weight_rounded=True)


def test_strides_shapes_and_alignment():
    codes, scales, g = _weights(96, 256, 128)
    x = torch.randn(3, 5, 300, generator=g, device=DEV).bfloat16()
    _check(x[..., :256], codes, scales, 128)                                  # rows further apart
    _check(x[..., 3: 259], codes, scales, 128)                                # not on 16 bytes
    _check(torch.randn(256, 4, generator=g, device=DEV).half().t(), codes, scales, 128)
    _check(x[1, 2, :256], codes, scales, 128)                                 # a vector
    pad = torch.zeros(codes.numel() + 1, dtype=torch.uint8, device=DEV)[1:].view_as(codes)
    pad.copy_(codes)
    _check(x[0, :, :256].contiguous(), pad, scales, 128)
    assert ops.w4_linear(x[:0, 0, :256], codes, scales).shape == (0, 96)
    assert ops.w4_linear(x[0, :, :256], codes[:0], scales[:0]).shape == (5, 0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = ops.w4_linear(x[0, :, :256], codes, scales)
    side.synchronize()
    assert torch.equal(y, ops.w4_linear(x[0, :, :256], codes, scales))


def test_large_and_special_values():
    codes, scales, g = _weights(64, 512, 128)
    x = torch.randn(2, 512, generator=g, device=DEV)
    _check((x * 1e30).bfloat16(), codes, scales, 128)
    x = x.half()
    x[1, 77] = float("inf")
    y = ops.w4_linear(x, codes, scales)
    hit = _weight64(codes, scales, 512, 128)[:, 77]
    assert torch.isfinite(y[0]).all()
    assert torch.equal(torch.isnan(y[1]), hit == 0) and torch.equal(y[1][hit != 0], torch.sign(hit[hit != 0]).half() * float("inf"))


def test_offsets_over_31_bits():
    """Codes of more than 2 GB: the last rows are found."""
    N, K = 140000, 32768
    codes = torch.zeros(N, K // 2, dtype=torch.uint8, device=DEV)
    scales = torch.zeros(N, K // 128, dtype=torch.bfloat16, device=DEV)
    assert codes.numel() > 1 << 31
    few, few_scales, g = _weights(16, K, 128)
    codes[-16:], scales[-16:] = few, few_scales
    x = torch.randn(1, K, generator=g, device=DEV).bfloat16()
    y = ops.w4_linear(x, codes, scales)
    assert torch.equal(y[:, -16:], ops.w4_linear(x, few, few_scales)) and (y[:, :-16] == 0).all()


@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantise_is_near(group):
    g = torch.Generator(device=DEV).manual_seed(1)
    w = torch.randn(50, 333, generator=g, device=DEV)
    w[3] = 0
    codes, scales = ops.w4_quantize(w, group)
    got = ops.w4_dequantize(codes, scales, 333, group)
    step = scales.float().repeat_interleave(group, 1)[:, :333]
    # half a step, and what the rounding of the scale cuts off at 7
    assert ((got - w).abs() <= step * (0.5 + 7 * 2.0 ** -8)).all() and (got[3] == 0).all()
    cpu = ops.w4_quantize(w.cpu(), group)
    assert torch.equal(codes.cpu(), cpu[0]) and torch.equal(scales.cpu(), cpu[1])


def test_refusals():
    codes, scales, _ = _weights(32, 128, 128)
    x = torch.zeros(2, 128, device=DEV).bfloat16()
    for bad in ((x.float(), codes, scales), (x[:, :64], codes, scales), (x, codes.int(), scales), (x, codes, scales.half()),
                (x, codes, scales, 64), (x, codes, scales, 16), (x, codes[:, ::2], scales), (x, codes, scales, 128, x[0, :32].half()),
                (x, codes, scales, 128, x[0, :31]), (x.cpu(), codes, scales), (x, codes[:31], scales)):
        with pytest.raises(ValueError):
            ops.w4_linear(*bad)
    with pytest.raises(RuntimeError):
        ops.w4_linear(x.clone().requires_grad_(), codes, scales)
    with torch.no_grad():
        ops.w4_linear(x.clone().requires_grad_(), codes, scales)
    assert w4.GROUPS == (32, 64, 128)


@pytest.mark.parametrize("offset", [1, 2, 4, 8])
@pytest.mark.parametrize("M", [64, 72, 104, 300])
def test_codes_off_their_alignment(M, offset):
    codes, scales, g = _weights(104, 264, 64)
    x = torch.randn(M, 264, generator=g, device=DEV).bfloat16()
    pad = torch.zeros(codes.numel() + offset, dtype=torch.uint8, device=DEV)[offset:].view_as(codes)
    pad.copy_(codes)
    assert torch.equal(_check(x, pad, scales, 64, weight_rounded=M >= w4.EXPAND_ROWS), ops.w4_linear(x, codes, scales, 64))


@pytest.mark.parametrize("N", [104, 99, 513])
@pytest.mark.parametrize("M", [97, 104, 300])
def test_many_rows_of_any_layout(M, N):
    """Rows off 16 bytes, pitches that are no multiple of 8, one row many times over, outputs of any width: two launches of the package."""
    codes, scales, g = _weights(N, 256, 64)
    x = torch.randn(M, 300, generator=g, device=DEV).bfloat16()
    bias = torch.randn(N + 1, generator=g, device=DEV).bfloat16()[1:]
    for y in (x[:, :256], x[:, 3: 259], x[:, :259][:, 1: 257], x.view(-1)[: M * 256].view(M, 256), x[:1, :256].expand(M, 256),
              x.view(-1)[5: M * 261 + 5].view(M, 261)[:, :256]):
        _lib.lib()
        before = _lib.launch_count
        _check(y, codes, scales, 64, bias, weight_rounded=True)
        assert _lib.launch_count == before + 4
    assert ops.w4_linear(x[:, :256].reshape(M, 1, 256), codes, scales, 64).shape == (M, 1, N)


def test_gradients_and_tangents_are_refused():
    from tests.test_w4_beam_cpu import check_gradients_are_refused

    check_gradients_are_refused(DEV)


@pytest.mark.parametrize("M", [65, 96])
def test_weights_are_exact_below_the_expansion(M):
    codes, scales, g = _weights(200, 512, 128)
    assert M < w4.EXPAND_ROWS
    _check(torch.randn(M, 512, generator=g, device=DEV).bfloat16(), codes, scales, 128)
