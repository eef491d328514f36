"""GPU: the W8A8 linear layer with bias, activation and residual (``s8b_linear_w8a8``) against
the same formula in 64 bits.

The int32 sums are exact. The epilogue is binary32 (a few roundings of 2^-24 on terms no larger
than |v| + |bias| + |residual|; exp, erf and the divisions below 1e-5 relative), then one
rounding to the output type, at most half a step: eps / 2 relative."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _case(M, N, K, dtype, bias, residual, seed=0):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    codes = lambda *s: torch.randint(-127, 128, s, generator=g, device=DEV, dtype=torch.int8)  # noqa: E731
    xq, w = codes(M, K), codes(N, K)
    xs = 0.01 + 0.03 * torch.rand(M, generator=g, device=DEV)
    ws = (0.5 + torch.rand(N, generator=g, device=DEV)) / (73 * math.sqrt(K))
    b = torch.randn(N, generator=g, device=DEV).to(dtype) if bias else None
    r = torch.randn(M, N, generator=g, device=DEV).to(dtype) if residual else None
    return xq, xs, w, ws, b, r


def _exact(xq, xs, w, ws, b, r, act):
    v = (xq.double() @ w.double().T) * xs.double()[:, None] * ws.double()
    size = v.abs()
    if b is not None:
        v = v + b.double()
        size = size + b.double().abs()
    if act == "silu":
        v = v * torch.sigmoid(v)
    elif act == "gelu":
        v = v * 0.5 * torch.erfc(-v / math.sqrt(2))
    elif act == "gelu_tanh":
        v = 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))
    elif act == "relu":
        v = v.clamp(min=0)
    if r is not None:
        v = v + r.double()
        size = size + r.double().abs()
    return v, size


def _near(y, v, size):
    tol = torch.finfo(y.dtype).eps / 2 * v.abs() + 2e-5 * size + torch.finfo(y.dtype).tiny
    bad = ((y.double() - v).abs() > tol) | ~torch.isfinite(y.double())
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, first {bad.nonzero()[0].tolist()}"


@pytest.mark.parametrize("M,N,K", [
    (1, 64, 128), (1, 7, 16), (3, 129, 272), (16, 512, 256), (255, 100, 384), (256, 96, 128),
    (257, 256, 128), (300, 264, 144), (129, 513, 1040), (640, 1000, 2064), (2050, 264, 512),
])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_linear_sizes(M, N, K, dtype):
    from superl8_serve_b200 import ops

    xq, xs, w, ws, b, r = _case(M, N, K, dtype, True, True, seed=M + N)
    y = ops.linear_w8a8(xq, xs, w, ws, bias=b, activation="silu", residual=r, out_dtype=dtype)
    _near(y, *_exact(xq, xs, w, ws, b, r, "silu"))


@pytest.mark.parametrize("M,N,K", [(5, 260, 256), (300, 260, 256), (300, 261, 80)])
@pytest.mark.parametrize("act", [None, "silu", "gelu", "gelu_tanh", "relu"])
@pytest.mark.parametrize("bias,residual", [(False, False), (True, False), (False, True)])
def test_linear_epilogues(M, N, K, act, bias, residual):
    from superl8_serve_b200 import ops

    xq, xs, w, ws, b, r = _case(M, N, K, torch.bfloat16, bias, residual, seed=7)
    xs = xs * 40  # pre-activations far into both tails
    y = ops.linear_w8a8(xq, xs, w, ws, bias=b, activation=act, residual=r)
    _near(y, *_exact(xq, xs, w, ws, b, r, act))


@pytest.mark.parametrize("M,N,K", [(1, 256, 128), (40, 260, 512), (256, 1024, 256),
                                   (257, 1024, 256), (700, 777, 640), (4096, 512, 4096)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_linear_without_epilogue_is_the_gemm(M, N, K, dtype):
    """Neither bias, activation nor residual: bit for bit the framework's other W8A8 products."""
    from superl8_serve_b200 import ops

    xq, xs, w, ws, _, _ = _case(M, N, K, dtype, False, False, seed=3)
    y = ops.linear_w8a8(xq, xs, w, ws, out_dtype=dtype)
    assert torch.equal(y, ops.gemm_w8a8_tc(xq, xs, w, ws, out_dtype=dtype))
    if M <= 256:
        assert torch.equal(y, ops.gemm_w8a8(xq, xs, w, ws, out_dtype=dtype))


def test_linear_extreme_values():
    """Largest sums, infinite and NaN scales and addends reach their own outputs only."""
    from superl8_serve_b200 import ops

    M, N, K = 300, 136, 4096
    xq = torch.full((M, K), 127, dtype=torch.int8, device=DEV)
    w = torch.full((N, K), 127, dtype=torch.int8, device=DEV)
    w[1] = -127
    xs = torch.full((M,), 1e-3, device=DEV)
    ws = torch.full((N,), 1e-4, device=DEV)
    xs[5], ws[9] = float("nan"), float("inf")
    r = torch.zeros(M, N, dtype=torch.bfloat16, device=DEV)
    r[7, 11] = float("-inf")
    y = ops.linear_w8a8(xq, xs, w, ws, residual=r).float()
    assert y[5].isnan().all() and y[7, 11] == float("-inf")
    keep = torch.ones(M, N, dtype=torch.bool, device=DEV)
    keep[5], keep[:, 9], keep[7, 11] = False, False, False
    assert (y[torch.arange(M, device=DEV) != 5, 9] == float("inf")).all()
    want = torch.full((M, N), 127 * 127 * K * 1e-7, device=DEV)
    want[:, 1] *= -1
    assert ((y - want).abs()[keep] <= want.abs()[keep] * 2 ** -8).all()
    s = ops.linear_w8a8(xq, xs * 1e4, w, ws, activation="silu").float()
    assert (s[keep & (want < 0)] == 0).all()


def test_linear_in_place_residual_leading_shape_and_reuse():
    from superl8_serve_b200 import ops

    for M in (6, 384):
        xq, xs, w, ws, b, r = _case(M, 200, 256, torch.bfloat16, True, True, seed=11)
        space = ops.linear_workspace(M, 200, 256, DEV)
        want = ops.linear_w8a8(xq, xs, w, ws, bias=b, residual=r, workspace=space)
        got = r.clone().view(2, M // 2, 200)
        out = ops.linear_w8a8(xq.view(2, M // 2, 256), xs.view(2, M // 2), w, ws, bias=b,
                              residual=got, out=got, workspace=space)
        assert out is got and torch.equal(got.view(M, 200), want)
        assert int(space[:4].view(torch.int32)) == 0
    empty = ops.linear_w8a8(xq[:0], xs[:0], w, ws)
    assert empty.shape == (0, 200)


@pytest.mark.parametrize("M", [9, 500])
def test_linear_unaligned_output_rows(M):
    """Outputs, bias and residual that start off a 16-byte boundary."""
    from superl8_serve_b200 import ops

    xq, xs, w, ws, b, r = _case(M, 264, 256, torch.bfloat16, True, True, seed=13)
    want = ops.linear_w8a8(xq, xs, w, ws, bias=b, residual=r)
    buf = torch.full((M * 264 + 8,), 9.0, dtype=torch.bfloat16, device=DEV)
    b2 = torch.zeros(265, dtype=torch.bfloat16, device=DEV)
    b2[1:] = b
    y = ops.linear_w8a8(xq, xs, w, ws, bias=b2[1:], residual=r, out=buf[3:3 + M * 264].view(M, 264))
    assert torch.equal(y, want) and (buf[:3] == 9).all() and (buf[3 + M * 264:] == 9).all()


@pytest.mark.parametrize("M", [12, 600])
def test_linear_graph_and_side_stream(M):
    from superl8_serve_b200 import ops

    xq, xs, w, ws, b, r = _case(M, 256, 256, torch.bfloat16, True, True, seed=17)
    want = ops.linear_w8a8(xq, xs, w, ws, bias=b, activation="gelu", residual=r)
    space = ops.linear_workspace(M, 256, 256, DEV)
    out = torch.empty_like(want)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        ops.linear_w8a8(xq, xs, w, ws, bias=b, activation="gelu", residual=r, out=out,
                        workspace=space)
    st.synchronize()
    assert torch.equal(out, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        ops.linear_w8a8(xq, xs, w, ws, bias=b, activation="gelu", residual=r, out=out,
                        workspace=space)
    out.zero_()
    xq2, *_ = _case(M, 256, 256, torch.bfloat16, True, True, seed=18)
    xq.copy_(xq2)
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, ops.linear_w8a8(xq, xs, w, ws, bias=b, activation="gelu", residual=r))


@pytest.mark.parametrize("M", [1, 8, 64, 256, 300])
@pytest.mark.parametrize("epilogue", [False, True])
def test_linear_weights_quantized_just_before(M, epilogue):
    """The weights come from kernels that the launch may overlap with, directly before or before the
    activations' own quantization: the product is that of the new weights."""
    from superl8_serve_b200 import _lib, ops

    N, K = 1184, 4096
    g = torch.Generator(device=DEV)
    g.manual_seed(M)
    ws_in = [torch.randn(N, K, generator=g, device=DEV).bfloat16() for _ in range(2)]
    x = torch.randn(M, K, generator=g, device=DEV).bfloat16()
    r = torch.randn(M, N, generator=g, device=DEV).bfloat16() if epilogue else None
    space = ops.linear_workspace(M, N, K, DEV)
    w, ws = ops.quant_rows(ws_in[0])
    xq, xs = ops.quant_rows(x)
    out = torch.empty(M, N, dtype=torch.bfloat16, device=DEV)
    want = []
    for t in ws_in:
        qw, qs = ops.quant_rows(t)
        torch.cuda.synchronize()
        want.append(ops.linear_w8a8(xq, xs, qw, qs, residual=r))
    torch.cuda.synchronize()

    def quantize(src, q, s):
        _lib.call("s8b_quant_rows", src.data_ptr(), 0, q.data_ptr(), s.data_ptr(), src.shape[0], K,
                  _lib.stream(src.device))

    for i in range(40):
        for both in (False, True):
            quantize(ws_in[i % 2], w, ws)
            if both:
                quantize(x, xq, xs)
            ops.linear_w8a8(xq, xs, w, ws, residual=r, out=out, workspace=space)
            assert torch.equal(out, want[i % 2])


@pytest.mark.parametrize("M", [9, 257])
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_activation_tails(M, act, dtype):
    """Relative to the activation's own value, however small. v has two roundings (2^-23 relative), which
    the tails multiply by |v f'(v) / f(v)|: below v^2 + 1 <= 200 for GELU down to binary32's smallest
    values, 100 for SiLU: 2.4e-5. The argument's own rounding counts the same again, exp, erfc and the
    division below 2e-5. Together below 1e-4, then half a step of the output. Below binary32's normal
    range (2^-126, times |v| < 2^7) steps are coarser; fp16's own end at 2^-24."""
    from superl8_serve_b200 import ops

    K, N = 128, 254
    xq = torch.zeros(M, K, dtype=torch.int8, device=DEV)
    w = torch.zeros(N, K, dtype=torch.int8, device=DEV)
    xq[:, 5] = 1 + torch.arange(M, device=DEV) % 9
    w[:, 5] = torch.cat([torch.arange(-127, 0), torch.arange(1, 128)]).to(DEV)
    xs = 0.25 + torch.rand(M, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    ws = torch.full((N,), 0.1, device=DEV)
    v = (xq.double() @ w.double().T) * xs.double()[:, None] * ws.double()
    assert v.min() < -100 and v.max() > 100 and v.abs().min() < 0.1
    if act == "silu":
        want = v * torch.sigmoid(v)
    elif act == "gelu":
        want = v * 0.5 * torch.erfc(-v / math.sqrt(2))
    else:
        want = v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))
    y = ops.linear_w8a8(xq, xs, w, ws, activation=act, out_dtype=dtype).double()
    least = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -118
    tol = (torch.finfo(dtype).eps / 2 + 1e-4) * want.abs() + least
    bad = (y - want).abs() > tol
    assert not bad.any(), (v[bad][:4].tolist(), y[bad][:4].tolist(), want[bad][:4].tolist())


@pytest.mark.parametrize("M", [16, 17, 40, 96, 128, 129, 200, 256])
@pytest.mark.parametrize("N,K", [(264, 256), (1025, 1024), (20000, 256), (4096, 512)])
def test_both_forms_with_one_workspace(M, N, K):
    """A workspace made for 256 rows serves every smaller call, whichever form it takes."""
    from superl8_serve_b200 import ops

    xq, xs, w, ws, b, r = _case(M, N, K, torch.bfloat16, True, True, seed=M + N)
    space = ops.linear_workspace(256, N, K, DEV)
    y = ops.linear_w8a8(xq, xs, w, ws, bias=b, activation="silu", residual=r, workspace=space)
    _near(y, *_exact(xq, xs, w, ws, b, r, "silu"))
    y = ops.linear_w8a8(xq, xs, w, ws, workspace=space)
    assert torch.equal(y, ops.gemm_w8a8(xq, xs, w, ws))
    assert int(space[:4].view(torch.int32)) == 0


@pytest.mark.parametrize("M,N,K", [(1, 7, 128), (5, 261, 256), (16, 1001, 384), (3, 129, 4096),
                                   (60, 515, 512)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_few_rows_of_odd_width(M, N, K, dtype):
    """The streamed form's scalar epilogue (N not a multiple of 4)."""
    from superl8_serve_b200 import ops

    xq, xs, w, ws, b, r = _case(M, N, K, dtype, True, True, seed=M + N)
    assert ops.linear_workspace(M, N, K, DEV).numel() > 256
    y = ops.linear_w8a8(xq, xs, w, ws, bias=b, activation="gelu", residual=r, out_dtype=dtype)
    _near(y, *_exact(xq, xs, w, ws, b, r, "gelu"))
    assert torch.equal(ops.linear_w8a8(xq, xs, w, ws, out_dtype=dtype),
                       ops.gemm_w8a8(xq, xs, w, ws, out_dtype=dtype))
