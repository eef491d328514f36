"""CPU: what the linear, chunk-attention and few-token MoE entry points refuse, at the C ABI
(before anything is dereferenced or launched) and in the tensor wrappers."""

import pytest
import torch

from superl8_serve_b200 import ops

OK = 4096  # a non-null, well-aligned address: validation comes before any dereference


def _linear(lib, **kw):
    a = dict(xq=OK, xs=OK, w=OK, ws=OK, bias=None, act=0, res=None, y=OK, M=4, N=64, K=128, dt=0,
             space=OK, size=1 << 30)
    a.update(kw)
    return lib.s8b_linear_w8a8(*a.values(), None)


@pytest.mark.parametrize("kw,code", [
    ({"xq": None}, -8), ({"xs": None}, -8), ({"w": None}, -8), ({"ws": None}, -8),
    ({"y": None}, -8), ({"act": 5}, -8), ({"act": -1}, -8), ({"dt": 2}, -2), ({"M": -1}, -1),
    ({"N": 0}, -1), ({"K": 0}, -1), ({"K": 136}, -1), ({"K": 131072}, -1), ({"xq": OK + 8}, -3),
    ({"w": OK + 4}, -3), ({"xs": OK + 2}, -3), ({"y": OK + 1}, -3), ({"bias": OK + 1}, -3),
    ({"res": OK + 1}, -3), ({"space": None}, -7), ({"size": 255}, -7), ({"space": OK + 16}, -3),
    ({"M": 0}, 0),
])
def test_linear_refusals(lib, kw, code):
    assert _linear(lib, **kw) == code


def test_linear_workspace(lib):
    assert lib.s8b_linear_workspace_size(257, 4096, 4096) == 256  # tiled: the status word only
    assert lib.s8b_linear_workspace_size(4, 4096, 144) == 256
    n = lib.s8b_linear_workspace_size(4, 4096, 4096)
    assert n > 256 and (n - 256) % (4 * 4096 * 4) == 0
    assert _linear(lib, M=4, N=4096, K=4096, size=n - 1) == -7


def test_linear_wrapper_refusals():
    z = torch.zeros
    xq, xs, w, ws = z(2, 64, dtype=torch.int8), z(2), z(8, 64, dtype=torch.int8), z(8)
    with pytest.raises(ValueError, match="unknown activation"):
        ops.linear_w8a8(xq, xs, w, ws, activation="swish")
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ops.linear_w8a8(xq, xs, w, ws)
    with pytest.raises(ValueError, match=r"w \[N, K\]"):
        ops.linear_w8a8(xq, xs, w[0], ws)


def _chunk(lib, **kw):
    a = dict(q=OK, qs=OK, kc=OK, ks=OK, vc=OK, vs=OK, bt=OK, ctx=OK, cu=OK, out=OK, T=8, S=2, Hq=8,
             Hkv=2, D=128, bs=16, maxb=4, nb=9, scale=0.1, space=OK, size=1 << 30, dt=0)
    a.update(kw)
    return lib.s8b_paged_chunk_q8(*a.values(), None)


@pytest.mark.parametrize("kw,code", [
    *[({n: None}, -8) for n in ("q", "qs", "kc", "ks", "vc", "vs", "bt", "ctx", "cu", "out")],
    ({"scale": 0.0}, -8), ({"scale": -1.0}, -8), ({"scale": float("nan")}, -8),
    ({"scale": float("inf")}, -8), ({"dt": 2}, -2), ({"T": -1}, -1), ({"S": -1}, -1),
    ({"S": 1025}, -1), ({"Hq": 9}, -1), ({"Hkv": 0}, -1), ({"Hq": 258}, -1), ({"D": 64}, -1),
    ({"bs": 12}, -1), ({"bs": 512}, -1), ({"bs": 0}, -1), ({"maxb": 0}, -1), ({"nb": 0}, -1),
    ({"nb": 2 ** 31 - 1}, -1), ({"T": 2 ** 30}, -1), ({"q": OK + 8}, -3), ({"kc": OK + 4}, -3),
    ({"out": OK + 2}, -3), ({"ks": OK + 2}, -3), ({"cu": OK + 1}, -3), ({"space": None}, -7),
    ({"size": 1024}, -7), ({"space": OK + 16}, -3), ({"T": 0}, 0), ({"S": 0}, 0),
])
def test_chunk_refusals(lib, kw, code):
    assert _chunk(lib, **kw) == code


def test_chunk_wrapper_refusals():
    z = torch.zeros
    q, qs = z(4, 8, 128, dtype=torch.int8), z(4, 8)
    kc, ks = z(3, 2, 16, 128, dtype=torch.int8), z(3, 2, 16)
    bt, ctx, cu = (z(s, dtype=torch.int32) for s in ((1, 2), (1,), (2,)))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ops.paged_chunk_q8(q, qs, kc, ks, kc, ks, bt, ctx, cu, 0.1)


def _moe(lib, **kw):
    a = dict(y=OK, xq=OK, xs=OK, gate=OK, gu_w=OK, gu_s=OK, d_w=OK, d_s=OK, out=OK, T=4, H=256,
             F=128, E=16, k=4, norm=1, scaling=1.0, space=OK, size=1 << 30, dt=0)
    a.update(kw)
    return lib.s8b_moe_layer(*a.values(), None)


@pytest.mark.parametrize("kw,code", [
    *[({n: None}, -8) for n in ("y", "xq", "xs", "gate", "gu_w", "gu_s", "d_w", "d_s", "out")],
    ({"dt": 2}, -2), ({"T": -1}, -1), ({"T": 17}, -1), ({"H": 264}, -1), ({"F": 120}, -1),
    ({"H": 0}, -1), ({"H": 8208}, -1), ({"E": 0}, -1), ({"E": 257}, -1), ({"k": 0}, -1),
    ({"k": 17, "E": 20}, -1), ({"k": 5, "E": 4}, -1), ({"F": 16384, "k": 10}, -1),
    ({"y": OK + 8}, -3), ({"gu_w": OK + 8}, -3), ({"d_w": OK + 4}, -3), ({"gate": OK + 4}, -3),
    ({"xs": OK + 2}, -3), ({"out": OK + 1}, -3), ({"space": None}, -7), ({"size": 256}, -7),
    ({"space": OK + 64}, -3), ({"T": 0}, 0),
])
def test_moe_layer_refusals(lib, kw, code):
    assert _moe(lib, **kw) == code


def test_moe_layer_rows():
    assert ops.moe_layer_max_rows(2048, 768, 8) == 16
    assert ops.moe_layer_max_rows(256, 16384, 8) == 1  # codes of one row of eight experts
    assert 0 < ops.moe_layer_max_rows(8192, 1024, 16) < 16
    assert ops.moe_layer_max_rows(256, 16384, 16) == 0
    assert ops.moe_layer_max_rows(100, 128, 2) == 0
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        z = torch.zeros
        ops.moe_layer(z(1, 32), z(1, 32, dtype=torch.int8), z(1), z(2, 32),
                      z(2, 32, 32, dtype=torch.int8), z(2, 32), z(2, 32, 16, dtype=torch.int8),
                      z(2, 32), 1)


def test_chunk_sequences():
    from superl8_serve_b200.engine import chunk_sequences

    lens = [5, 1, 9]
    seq = [i for i, n in enumerate(lens) for _ in range(n)]
    pos = [p for n in lens for p in range(n)]
    got = chunk_sequences(seq, pos, 4)
    assert got == [([0], [4], [0, 4]), ([0, 1, 2], [5, 1, 2], [0, 1, 2, 4]), ([2], [6], [0, 4]),
                   ([2], [9], [0, 3])]
    for seqs, ctx, cu in got:
        assert len(seqs) == len(ctx) == len(cu) - 1


def test_pipeline_options_are_checked():
    from superl8_serve_b200.engine import DecodePipeline

    with pytest.raises(ValueError, match="prefill_attention"):
        DecodePipeline([], batch=1, prefill_attention="tiles")
