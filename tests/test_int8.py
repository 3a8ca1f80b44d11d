"""8-bit integer products against plain implementations (oracle/serving_oracle.py)."""

from __future__ import annotations

import numpy as np
import pytest
import torch
import torch.nn as nn

import pare_amd as P
from oracle import serving_oracle as S
from pare_amd import _lib

gpu = pytest.mark.gpu
DEV = torch.device("cuda:0")
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
P8 = 0x1000  # a 16-byte aligned address that is never read: validation comes first


@pytest.mark.parametrize("change", [dict(dtype=_lib.PMI_U8), dict(stride=15), dict(M=-1), dict(K=0), dict(K=131073),
                                    dict(x=None), dict(codes=P8 + 8), dict(x=P8 + 1), dict(scales=None),
                                    dict(M=1 << 24)])
def test_quantize_refuses(change):
    a = dict(x=P8, dtype=_lib.PMI_F16, stride=1 << 20, codes=P8, scales=P8, M=2, K=16)
    a.update(change)
    assert _lib.lib().pmi_quantize_rows(*a.values(), None) < 0 and "pmi_quantize_rows" in _lib.last_error()


@pytest.mark.parametrize("change", [dict(dtype=_lib.PMI_I8), dict(M=-1), dict(N=-1), dict(K=0), dict(K=131073),
                                    dict(x=None), dict(w=P8 + 4), dict(y=None), dict(y=P8 + 1), dict(bias=P8 + 1),
                                    dict(N=1 << 24), dict(sx=None), dict(sw=None)])
def test_matmul_refuses(change):
    a = dict(x=P8, sx=P8, w=P8, sw=P8, bias=None, y=P8, dtype=_lib.PMI_F16, M=2, N=3, K=16)
    a.update(change)
    assert _lib.lib().pmi_matmul_w8a8(*a.values(), None) < 0 and "pmi_matmul_w8a8" in _lib.last_error()


@pytest.mark.parametrize("change", [dict(dtype=_lib.PMI_I8), dict(stride=15), dict(stride=1 << 40), dict(M=-1),
                                    dict(N=-1), dict(K=0), dict(K=131073), dict(x=None), dict(x=P8 + 1),
                                    dict(w=P8 + 4), dict(sw=None), dict(y=None), dict(y=P8 + 1), dict(bias=P8 + 1),
                                    dict(N=1 << 24), dict(scratch=None), dict(scratch=P8 + 4), dict(bytes=39)])
def test_matmul_rows_refuses(change):
    a = dict(x=P8, dtype=_lib.PMI_F16, stride=16, w=P8, sw=P8, bias=None, y=P8, M=2, N=3, K=16, scratch=P8, bytes=40)
    a.update(change)
    assert _lib.lib().pmi_matmul_w8a8_rows(*a.values(), None) < 0 and "pmi_matmul_w8a8_rows" in _lib.last_error()
    assert _lib.lib().pmi_matmul_w8a8_scratch_bytes(2, 16) == 40


def test_empty_calls_and_cpu_tensors():
    L = _lib.lib()
    assert L.pmi_quantize_rows(None, _lib.PMI_F16, 16, None, None, 0, 16, None) == _lib.PMI_OK
    assert L.pmi_matmul_w8a8(None, None, None, None, None, None, _lib.PMI_F16, 0, 3, 16, None) == _lib.PMI_OK
    w, s = torch.zeros(3, 16, dtype=torch.int8), torch.zeros(3)
    for call in (lambda: P.matmul_w8a8(torch.zeros(2, 16), w, s), lambda: P.quantize_rows(torch.zeros(2, 16)),
                 lambda: P.matmul_int8(w, s, w, s, 16, torch.float16), lambda: P.Int8Linear(w, s, 16)(torch.zeros(2, 16))):
        with pytest.raises(RuntimeError, match="HIP"):
            call()
    with pytest.raises(ValueError):
        P.Int8Linear(w, s, 17)
    with pytest.raises(ValueError):
        P.Int8Linear(w, s[:2], 16)


def _rows(M, K, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=g) * (0.2 + 4 * torch.rand(K, generator=g) ** 8)
    return x.to(dtype)


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,K", [(1, 1), (1, 16), (3, 17), (5, 100), (2, 4096), (70, 1000), (4, 14336), (1, 65552),
                                 (3, 8193), (2, 131072)])
def test_quantize_rows_equals_the_oracle_bit_for_bit(dtype, M, K):
    """One IEEE fp32 operation after another: equal codes and scales; zeros past K; rows of a
    wider tensor at any alignment, rows of zeros."""
    x = _rows(M, K, dtype, M * K)
    if M > 2:
        x[1] = 0
    codes, scales = P.quantize_rows(x.to(DEV))
    want, ws = S.quantize_rows(x.float().numpy())
    assert codes.shape == (M, -(-K // 16) * 16)
    np.testing.assert_array_equal(codes[:, :K].cpu().numpy(), want)
    np.testing.assert_array_equal(scales.cpu().numpy(), ws)
    assert (codes[:, K:] == 0).all()
    wide = torch.zeros(M, K + 3, dtype=dtype, device=DEV)
    wide[:, 1:K + 1] = x.to(DEV)
    again, s2 = P.quantize_rows(wide[:, 1:K + 1])
    assert torch.equal(again, codes) and torch.equal(s2, scales)
    turned = x.to(DEV).t().contiguous().t()
    assert torch.equal(P.quantize_rows(turned)[0], codes)


@gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("M,N,K", [(1, 5000, 4096), (1, 20000, 2048), (1, 130, 16384), (1, 130, 16385), (2, 12500, 8190), (3, 77, 4090),
                                   (4, 5200, 4096), (4, 300, 1024), (4, 300, 1009), (4, 300, 1000), (5, 300, 2048),
                                   (1, 40, 12289)])
def test_matmul_of_few_rows_is_the_two_calls(dtype, M, N, K):
    """Rows quantised inside the product or before it: the same bits, also in place of x, from
    strided and unaligned rows, and with rows of zeros, infinities and NaN."""
    g = torch.Generator().manual_seed(M * N + K)
    x = torch.randn(M, K + 3, generator=g).to(dtype).to(DEV)
    w, sw = P.quantize_rows(torch.randn(N, K, generator=g).to(DEV))
    bias = torch.randn(N, generator=g).to(dtype).to(DEV)

    def check(x):
        want = P.matmul_int8(*P.quantize_rows(x), w, sw, K, dtype, bias=bias)
        got = P.matmul_w8a8(x, w, sw, bias=bias)
        assert torch.equal(got.view(torch.uint8), want.view(torch.uint8))

    for first in (0, 1, 3):
        check(x[:, first:first + K])
    x[0, 5] = float("inf")
    x[-1, K - 1] = float("nan")
    check(x[:, :K])
    x[0] = 0
    check(x[:, :K])
    if N >= K:
        square = P.quantize_rows(torch.randn(K, K, generator=g).to(DEV))
        y = x[:, :K].contiguous()
        want = P.matmul_w8a8(y.clone(), *square)
        assert torch.equal(P.matmul_w8a8(y, *square, out=y).view(torch.uint8), want.view(torch.uint8))


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_the_smallest_rows(dtype):
    """Rows whose scale has no finite inverse, zeros among them."""
    x = (torch.randn(5, 40, generator=torch.Generator().manual_seed(2)) * 1e-38).to(dtype)
    x[:, 3:9] = 0
    codes, scales = P.quantize_rows(x.to(DEV))
    want, want_scales = S.quantize_rows(x.float().numpy())
    np.testing.assert_array_equal(scales.cpu().numpy(), want_scales)
    np.testing.assert_array_equal(codes[:, :40].cpu().numpy(), want)
    assert (want[:, 3:9] == 0).all()


@gpu
def test_rows_with_infinities_and_nan_are_not_finite():
    x = torch.ones(4, 64, dtype=torch.float16, device=DEV)
    x[1, 3], x[2, 60] = float("nan"), float("-inf")
    codes, scales = P.quantize_rows(x)
    assert torch.isfinite(scales).tolist() == [True, False, False, True]
    w, ws = P.quantize_rows(torch.randn(40, 64, device=DEV))
    y = P.matmul_w8a8(x, w, ws)
    assert torch.isfinite(y).all(1).tolist() == [True, False, False, True]


def _check(y, want, mag, dtype):
    """The sum is exact; the conversion of it to fp32, two scales and the bias are four roundings
    of 2^-24 of the terms, the output one of its type's (fp16: no less than 2^-25)."""
    tol = HALF[dtype] * np.abs(want) + 4 * 2.0 ** -24 * mag * (1 + HALF[dtype]) + (2.0 ** -25 if dtype == torch.float16 else 0)
    err = np.abs(y.cpu().double().numpy() - want)
    bad = err > tol
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, at most {(err / tol).max():.2f} times what is allowed, at " \
                          f"{np.argwhere(bad)[0]}"


def _case(M, N, K, dtype, bias, seed=0):
    x = _rows(M, K, dtype, seed + M)
    w, sw = P.quantize_rows((torch.randn(N, K, generator=torch.Generator().manual_seed(seed + N)) * 0.05).to(DEV))
    b = torch.randn(N, generator=torch.Generator().manual_seed(K)).to(dtype).to(DEV) if bias else None
    cx, sx = S.quantize_rows(x.float().numpy())
    bn = None if b is None else b.cpu().float().numpy()
    want = S.matmul_w8a8(cx, sx, w[:, :K].cpu().numpy(), sw.cpu().numpy(), bn)
    mag = np.abs(S.matmul_w8a8(cx, sx, w[:, :K].cpu().numpy(), sw.cpu().numpy())) + (0 if bn is None else np.abs(bn))
    return x.to(DEV), w, sw, b, want, mag


SIZES = [(1, 1, 1), (1, 5, 16), (1, 128, 4096), (2, 1000, 512), (3, 77, 100), (7, 257, 1040), (16, 512, 2048),
         (17, 300, 4096), (31, 64, 14336), (33, 1023, 528), (64, 2049, 256), (65, 130, 4096), (100, 511, 1000),
         (128, 1024, 1024), (129, 257, 4112), (200, 4096, 128), (256, 256, 4096), (300, 1111, 2000), (513, 769, 272),
         (1000, 520, 64), (1024, 2048, 512)]


@gpu
@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("dtype,bias", [(torch.float16, False), (torch.bfloat16, True), (torch.float32, True)])
def test_matmul_w8a8(M, N, K, dtype, bias):
    x, w, sw, b, want, mag = _case(M, N, K, dtype, bias)
    y = P.matmul_w8a8(x, w, sw, bias=b)
    assert y.dtype == dtype
    _check(y, want, mag, dtype)
    assert torch.equal(y, P.matmul_w8a8(x, w, sw, bias=b))


@gpu
@pytest.mark.parametrize("M", [1, 8, 40, 300])
def test_sums_at_the_ends_of_the_range(M):
    """Every code 127 or -127 over the longest rows: 127^2 K is just below 2^31."""
    K, N = 131072, 48
    codes = torch.full((M, K), 127, dtype=torch.int8, device=DEV)
    codes[::2] = -127
    w = torch.full((N, K), 127, dtype=torch.int8, device=DEV)
    one = torch.ones(max(M, N), device=DEV)
    y = P.matmul_int8(codes, one[:M], w, one[:N], K, torch.float32)
    want = torch.full((M, N), float(127 * 127 * K), dtype=torch.float32)
    want[::2] *= -1
    assert torch.equal(y.cpu(), want)


@gpu
@pytest.mark.parametrize("M,N,K", [(5, 300, 4096), (150, 601, 528), (700, 1030, 256)])
def test_out_bias_types_and_rows_of_one_input(M, N, K):
    """``out`` at an odd place of a larger buffer, guarded on both sides; a bias of another
    type; rows quantised once for two products."""
    x, w, sw, b, want, mag = _case(M, N, K, torch.float16, True)
    buf = torch.full((M * N + 6,), 5.0, dtype=torch.float16, device=DEV)
    out = buf[3:3 + M * N].view(M, N)
    assert P.matmul_w8a8(x, w, sw, bias=b, out=out) is out
    _check(out, want, mag, torch.float16)
    assert (buf[:3] == 5).all() and (buf[3 + M * N:] == 5).all()
    codes, s = P.quantize_rows(x)
    assert torch.equal(P.matmul_int8(codes, s, w, sw, K, torch.float16, bias=b), out)
    assert torch.equal(P.matmul_w8a8(x, w, sw, bias=b.float()), out)
    with pytest.raises(AssertionError):
        P.matmul_w8a8(x, w[:, :-16], sw)
    with pytest.raises(AssertionError):
        P.matmul_w8a8(x, w, sw[:-1])
    with pytest.raises(AssertionError):
        P.matmul_w8a8(x, w, sw, bias=b[:-1])
    with pytest.raises(RuntimeError):
        P.matmul_w8a8(x, w, sw.cpu())


@gpu
@pytest.mark.parametrize("bias", [True, False])
def test_int8_linear(bias):
    """The module beside the layer it was made from: each weight is off by at most half its
    channel's code, each activation by half its token's."""
    lin = nn.Linear(520, 330, bias=bias).to(DEV)
    q = P.Int8Linear.from_linear(lin)
    x = _rows(6, 520, torch.float32, 3).view(2, 3, 520).to(DEV)
    y = q(x)
    assert y.shape == (2, 3, 330) and y.dtype == torch.float32
    w = lin.weight.detach().double().cpu()
    xd = x.double().cpu()
    sw, sx = w.abs().amax(1) / 254, xd.abs().amax(-1, keepdim=True) / 254
    tol = (xd.abs() + sx).sum(-1, keepdim=True) * sw + sx * w.abs().sum(1) + 1e-5
    want = xd @ w.t() + (lin.bias.detach().double().cpu() if bias else 0)
    assert ((y.double().cpu() - want).abs() <= tol * 1.0001).all()
    again = P.Int8Linear(torch.empty_like(q.weight), torch.empty_like(q.scale), 520,
                         torch.empty(330, device=DEV) if bias else None)
    again.load_state_dict(q.state_dict())
    assert torch.equal(again(x), y)
    cpu = P.Int8Linear.from_weight(lin.weight.detach().cpu())
    assert cpu.weight.device.type == "cpu" and torch.equal(cpu.weight, q.weight.cpu())


def _codes(N, K, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-127, 128, (N, -(-K // 16) * 16), generator=g, dtype=torch.int8), torch.rand(N, generator=g) * 1e-5


def test_scales_stay_fp32_when_the_module_changes_type():
    """``half()`` and ``to(dtype)`` of a model convert the bias; the scales, which fp16 would
    round or lose, and the codes stay."""
    for convert in (lambda m: m.half(), lambda m: m.to(torch.bfloat16), lambda m: m.double(),
                    lambda m: nn.Sequential(m).half()[0]):
        codes, scale = _codes(5, 32)
        m = convert(P.Int8Linear(codes, scale, 32, torch.ones(5)))
        assert m.scale.dtype == torch.float32 and torch.equal(m.scale, scale)
        assert m.weight.dtype == torch.int8 and torch.equal(m.weight, codes)
        assert m.bias.dtype != torch.float32
        assert m.state_dict()["scale"].dtype == torch.float32


@gpu
def test_a_converted_module_gives_the_same():
    lin = nn.Linear(256, 40).half().to(DEV)
    m = P.Int8Linear.from_linear(lin)
    x = _rows(3, 256, torch.float16, 1).to(DEV)
    want = m(x)
    assert torch.equal(m.half()(x), want) and torch.equal(nn.Sequential(m).to(torch.float16)(x), want)


def test_the_bias_is_no_leaf_to_train():
    """The product has no backward pass, so no optimizer is offered the bias."""
    codes, scale = _codes(5, 32)
    m = P.Int8Linear(codes, scale, 32, torch.ones(5))
    assert not any(p.requires_grad for p in m.parameters())


@gpu
def test_an_input_that_needs_a_gradient_is_refused():
    m = P.Int8Linear.from_linear(nn.Linear(64, 8).to(DEV))
    x = torch.randn(2, 64, device=DEV, requires_grad=True)
    with pytest.raises(RuntimeError, match="gradient"):
        m(x)
    with torch.no_grad():
        y = m(x)
    assert torch.equal(m(x.detach()), y)
    with torch.inference_mode():
        assert torch.equal(m(x), y)


def test_models_with_int8_layers_are_saved_and_loaded(tmp_path):
    """``save_quantized`` and ``load_quantized`` of a model that holds both kinds of layer: the
    codes come back as codes, not as the float weight of what stood there."""
    config = P.QuantConfig(bits=4, scheme="rtn", group_size=32)
    g = torch.Generator().manual_seed(0)

    def four(n, k):
        return P.QuantizedLinear(torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8),
                                 torch.rand(n, k // 32, 1, generator=g), torch.full((n, k // 32, 1), 8.0), config, None, k, n)

    def eight(n, k, bias):
        return P.Int8Linear(*_codes(n, k, n), k, torch.randn(n, generator=g) if bias else None)

    model = nn.ModuleDict({"a": four(64, 64), "b": eight(48, 64, True), "c": nn.ModuleDict({"d": eight(32, 40, False)}),
                           "e": nn.Linear(8, 8)})
    with pytest.warns(UserWarning, match="8-bit"):
        P.save_quantized(model, tmp_path)
    for other in (nn.ModuleDict({"a": nn.Linear(64, 64), "b": nn.Linear(64, 48),
                                 "c": nn.ModuleDict({"d": nn.Linear(40, 32, bias=False)}), "e": nn.Linear(8, 8)}),
                  nn.ModuleDict({"a": four(64, 64), "b": eight(48, 64, True),
                                 "c": nn.ModuleDict({"d": eight(32, 40, False)}), "e": nn.Linear(8, 8)})):
        got = P.load_quantized(other, tmp_path)
        assert isinstance(got["b"], P.Int8Linear) and isinstance(got["c"]["d"], P.Int8Linear)
        assert got["c"]["d"].in_features == 40 and got["c"]["d"].out_features == 32 and got["c"]["d"].bias is None
        assert isinstance(got["a"], P.QuantizedLinear) and isinstance(got["e"], nn.Linear)
        have, want = got.state_dict(), model.state_dict()
        assert have.keys() == want.keys()
        assert all(have[n].dtype == want[n].dtype and torch.equal(have[n], want[n]) for n in want)
    # 8-bit layers alone
    alone = nn.ModuleDict({"b": eight(48, 64, True)})
    with pytest.warns(UserWarning, match="8-bit"):
        P.save_quantized(alone, tmp_path / "alone")
    got = P.load_quantized(nn.ModuleDict({"b": nn.Linear(64, 48)}), tmp_path / "alone")
    assert torch.equal(got["b"].weight, alone["b"].weight)
    with pytest.raises(ValueError):
        P.save_quantized(nn.Linear(4, 4), tmp_path / "none")


@gpu
@pytest.mark.parametrize("M,N,K,dtype,bias", [
    # 256 x 256 tiles, two or three a workgroup, ragged on both sides
    (300, 70001, 144, torch.bfloat16, True), (1100, 33001, 272, torch.float16, False),
    (520, 33003, 400, torch.float32, True),
    # 128 x 128 tiles, two a workgroup
    (130, 64900, 272, torch.float16, True), (129, 60001, 128, torch.float32, False),
    # up to 64 rows with 32 and 64 weight rows a workgroup
    (1, 5200, 1040, torch.float16, True), (6, 5200, 528, torch.bfloat16, False), (16, 12400, 1040, torch.float16, True),
    (17, 5200, 1040, torch.bfloat16, True), (17, 12401, 528, torch.float16, False), (40, 5201, 528, torch.float32, True),
    (40, 12400, 1040, torch.bfloat16, False), (64, 5200, 528, torch.float16, True), (64, 12403, 1040, torch.float16, True)])
def test_matmul_of_every_tile(M, N, K, dtype, bias):
    """The forms that only wide products take."""
    x, w, sw, b, want, mag = _case(M, N, K, dtype, bias)
    y = P.matmul_w8a8(x, w, sw, bias=b)
    assert y.isfinite().all()
    _check(y, want, mag, dtype)
    assert torch.equal(y, P.matmul_w8a8(x, w, sw, bias=b))
