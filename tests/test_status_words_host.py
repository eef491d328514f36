"""CPU: the pipeline reads the status words of its runners' workspaces and raises on them."""

import pytest
import torch

from superl8_serve_b200._lib import ERR_TIMEOUT, S8BError
from superl8_serve_b200.engine import DecodePipeline
from superl8_serve_b200.runtime import StageRunner


def _runner(m=4, fused=False, chunk=False):
    r = StageRunner.__new__(StageRunner)
    ws = lambda: torch.full((512,), 7, dtype=torch.uint8)  # noqa: E731
    r.m, r.fused_moe = m, fused
    r.chunk_ws, r.tc_ws, r.moe_buf = ws() if chunk else None, ws(), {"layer_ws": ws()}
    for w in (r.chunk_ws, r.tc_ws, r.moe_buf["layer_ws"]):
        if w is not None:
            w[:256].zero_()
    return r


def _pipe(*runners):
    p = DecodePipeline.__new__(DecodePipeline)
    p.models, p.runners = [], list(runners)
    return p


def test_workspaces_that_are_read():
    names = lambda r: [n for n, _ in r.status_workspaces()]  # noqa: E731
    assert names(_runner()) == []
    assert names(_runner(chunk=True)) == ["s8b_paged_chunk_q8"]
    assert names(_runner(fused=True)) == ["s8b_moe_layer"]
    assert names(_runner(m=257)) == ["s8b_linear_w8a8"]
    assert names(_runner(m=300, fused=True, chunk=True)) == ["s8b_paged_chunk_q8", "s8b_moe_layer",
                                                             "s8b_linear_w8a8"]


@pytest.mark.parametrize("name,code", [("chunk_ws", -8), ("tc_ws", ERR_TIMEOUT),
                                       ("layer_ws", ERR_TIMEOUT)])
def test_a_word_that_is_set_raises_once(name, code):
    good, r = _runner(chunk=True), _runner(m=300, fused=True, chunk=True)
    pipe = _pipe(good, r)
    pipe.synchronize()
    ws = r.moe_buf["layer_ws"] if name == "layer_ws" else getattr(r, name)
    ws[:4].view(torch.int32).fill_(code)
    ws[64:72].view(torch.int64).fill_(1000)  # the MoE layer's barrier counter, half way
    with pytest.raises(S8BError, match="invalid") as e:
        pipe.synchronize()
    assert e.value.code == code
    assert not ws[:256].any() and (ws[256:] == 7).all()  # zeroed: the next launch may use it
    pipe.synchronize()
    with pytest.raises(S8BError):
        ws[:4].view(torch.int32).fill_(code)
        pipe.check_status([r])
    ws[:4].view(torch.int32).fill_(code)
    pipe.check_status([good])
