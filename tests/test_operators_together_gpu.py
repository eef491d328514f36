"""GPU: the linear, chunk-attention and few-row MoE operators as the layers, the stage runner
and the pipeline use them, and one after another as a decoder layer does."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _weight(g, n, k):
    w = torch.randint(-127, 128, (n, k), generator=g, device=DEV, dtype=torch.int8)
    return w, (0.5 + torch.rand(n, generator=g, device=DEV)) / (73 * math.sqrt(k))


# ------------------------------------------------------------------------------- layers ----
@pytest.mark.parametrize("M", [1, 2, 37, 300])
@pytest.mark.parametrize("bias", [False, True])
def test_linear_layer_keeps_its_results(M, bias):
    """Without activation and residual: the dp4a product (and the bias added after it), bit for
    bit as before."""
    from superl8_serve_b200 import ops
    from superl8_serve_b200.layers import LinearW8A8
    from superl8_serve_b200.weights import QTensor

    g = _gen(M)
    w, ws = _weight(g, 260, 272)
    b = torch.randn(260, generator=g, device=DEV).bfloat16() if bias else None
    lin = LinearW8A8(QTensor(w, ws, "per_row_i8"), b)
    x = torch.randn(M, 272, generator=g, device=DEV).bfloat16()
    q, s = ops.quant_rows(x)
    want = ops.gemm_w8a8(q, s, w, ws)
    assert torch.equal(lin(x), want if b is None else want + b)
    assert torch.equal(lin(x.view(1, M, 272))[0], lin(x))
    r = torch.randn(M, 260, generator=g, device=DEV).bfloat16()
    assert torch.equal(lin(x, activation="gelu", residual=r),
                       ops.linear_w8a8(q, s, w, ws, bias=b, activation="gelu", residual=r))


# ------------------------------------------------------------- one after another ----------
def test_a_sparse_layer_over_a_chunk_of_draft_rows():
    """Three sequences bring 4, 1 and 7 new rows: keys and values go to the pages, the chunk
    attends over them, the output projection adds the residual, the MoE layer follows. Each step
    is checked against 64 bits on what the step before it gave."""
    from superl8_serve_b200 import ops
    from superl8_serve_b200.layers import rope_tables
    from test_chunk_attention_gpu import Case
    from test_linear_gpu import _exact, _near
    from test_moe_layer_gpu import Layer

    H, Hq, Hkv, bs = 512, 8, 2, 16
    lens = [(4, 150), (1, 33), (7, 7)]
    g = _gen(5)
    c = Case(lens, Hq, Hkv, bs, seed=5)
    T = c.T
    seq = torch.tensor([i for i, (n, _) in enumerate(lens) for _ in range(n)], device=DEV)
    pos = torch.cat([torch.arange(m - n, m) for n, m in lens]).to(torch.int32).to(DEV)
    cos, sin = (t.to(DEV) for t in rope_tables(128, 256))
    gain = torch.ones(128, dtype=torch.bfloat16, device=DEV)
    qkv = torch.randn(T, (Hq + 2 * Hkv) * 128, generator=g, device=DEV).bfloat16()
    before = c.kc.clone()
    c.q, c.qs, _ = ops.qkv_post(qkv, pos, cos, sin, gain, gain, 1e-6, Hq, Hkv, c.kc, c.ks, c.vc,
                                c.vs, block_table=c.bt[seq].contiguous())
    slot = c.bt[seq, (pos // bs).long()].long(), (pos % bs).long()
    same = torch.ones(c.kc.shape[0], bs, dtype=torch.bool, device=DEV)
    same[slot] = False
    assert torch.equal(c.kc.transpose(1, 2)[same], before.transpose(1, 2)[same])
    attn = c.run()
    c.check(attn)

    w, ws = _weight(g, H, Hq * 128)
    res = torch.randn(T, H, generator=g, device=DEV).bfloat16()
    aq, asc = ops.quant_rows(attn)
    h = ops.linear_w8a8(aq, asc, w, ws, residual=res)
    _near(h, *_exact(aq, asc, w, ws, None, res, None))

    L = Layer(T, H, 128, 16, 4, seed=6)
    _, L.xq, L.xs, L.y = ops.rmsnorm_quant(h, None, torch.ones(H, dtype=torch.bfloat16, device=DEV),
                                           1e-6, y_out=True)
    L.check(L.run())


# ----------------------------------------------------------------------------- pipeline ----
def _models(cfg, stages=1, seed=3):
    from superl8_serve_b200.runtime import StageModel
    from superl8_serve_b200.weights import random_state_dict

    sd = random_state_dict(cfg, seed, w_std=0.1)
    n = cfg.num_hidden_layers
    cut = [i * n // stages for i in range(stages + 1)]
    return [StageModel.from_state_dict(cfg, sd, cut[s], cut[s + 1], DEV, first=s == 0,
                                       last=s == stages - 1) for s in range(stages)]


def _prompts(lens, vocab, seed=0):
    g = torch.Generator()
    g.manual_seed(seed)
    return [torch.randint(0, vocab, (n,), generator=g).tolist() for n in lens]


@pytest.mark.parametrize("stages", [1, 2])
def test_wide_prefill_chunks_give_the_same_bits(stages):
    from superl8_serve_b200.config import tiny
    from superl8_serve_b200.engine import DecodePipeline

    cfg = tiny()
    models = _models(cfg, stages)
    prompts = _prompts([300, 7, 411], cfg.vocab_size)
    got = []
    for chunk in (256, 700):
        pipe = DecodePipeline(models, batch=3, max_len=512)
        pipe.prefill_chunk = chunk
        got.append(pipe.prefill(prompts, keep_logits=True))
    assert got[0][0] == got[1][0]
    for a, b in zip(got[0][1], got[1][1]):
        assert torch.equal(a, b)


@pytest.mark.parametrize("chunk", [64, 256, 1000])
def test_chunk_attention_in_the_prefill(chunk):
    """One layer, so that both kinds of attention see the same queries and pages: the last chunk's
    attention rows differ by the two forms' roundings of the weights, 2^-8 and below 2^-9 of the
    average of |v|, itself at most the largest |v| of the pool, and the outputs' roundings."""
    from superl8_serve_b200.config import tiny
    from superl8_serve_b200.engine import DecodePipeline

    cfg = tiny(num_hidden_layers=1)
    models = _models(cfg)
    prompts = _prompts([300, 1, 411, 90], cfg.vocab_size)
    rows, pools = [], []
    for kind in ("rows", "chunk"):
        pipe = DecodePipeline(models, batch=4, max_len=512, prefill_attention=kind)
        pipe.prefill_chunk = chunk
        first = pipe.prefill(prompts)
        n = (300 + 1 + 411 + 90 - 1) % chunk + 1  # rows of the last chunk
        rows.append(pipe._pf[0][0].attn[:n].double())
        pools.append(pipe.pools[0])
        assert len(first) == 4 and all(0 <= t < cfg.vocab_size for t in first)
        ws = pipe._pf[0][0].chunk_ws
        assert (ws is None) == (kind == "rows")
        assert ws is None or int(ws[:4].view(torch.int32)) == 0
    assert torch.equal(pools[0].vc, pools[1].vc) and torch.equal(pools[0].kc, pools[1].kc)
    top = (pools[0].vc.float().abs() * pools[0].vs[..., None]).max().item()
    assert (rows[0] - rows[1]).abs().max().item() <= (2 ** -8 + 2 ** -9 + 2 * 2 ** -8) * top
    assert (rows[0] - rows[1]).norm() < 2 ** -7 * rows[0].norm()


def test_generation_with_chunk_attention_and_continuation():
    from superl8_serve_b200.config import tiny
    from superl8_serve_b200.engine import DecodePipeline

    cfg = tiny()
    pipe = DecodePipeline(_models(cfg, 2), batch=3, max_len=512, prefill_attention="chunk")
    outs = pipe.generate(_prompts([40, 3, 130], cfg.vocab_size, 1), 5, prefill=True)
    assert [len(o) for o in outs] == [5, 5, 5]
    assert all(0 <= t < cfg.vocab_size for o in outs for t in o)
    with pytest.raises(ValueError, match="native"):
        pipe.set_native()


@pytest.mark.parametrize("batch", [1, 5, 16])
def test_fused_moe_in_the_decode_step(batch):
    """One sparse layer: its output against the general path's on the same rows, within that
    path's own roundings to dtype (16 steps of at most 2^-8 each)."""
    from superl8_serve_b200.config import tiny_moe
    from superl8_serve_b200.engine import DecodePipeline

    cfg = tiny_moe(num_hidden_layers=1)
    models = _models(cfg)
    h = []
    for fused in (False, True):
        pipe = DecodePipeline(models, batch=batch, max_len=64, fused_moe=fused)
        pipe.add_sequences()
        pipe.set_state([0] * batch, list(range(3, 3 + batch)), reserve=4)
        pipe.step()
        pipe.synchronize()
        h.append(pipe.runners[0].h[:batch].double().clone())
        pipe.capture()
        for _ in range(3):
            pipe.step()
        pipe.synchronize()
        assert int(pipe.runners[0].moe_buf["layer_ws"][:4].view(torch.int32)) == 0
        toks = pipe.tokens().tolist()
        assert all(0 <= t < cfg.vocab_size for t in toks)
    assert ((h[0] - h[1]).norm() / h[0].norm()).item() < 16 * 2 ** -8
    assert not torch.equal(h[0], h[1]) or batch == 1


def test_linear_layer_takes_scales_as_a_column():
    """As the dp4a product does, which took several rows before the tensor cores took over."""
    from superl8_serve_b200 import ops
    from superl8_serve_b200.layers import LinearW8A8
    from superl8_serve_b200.weights import QTensor

    g = _gen(3)
    w, ws = _weight(g, 24, 272)
    lin = LinearW8A8(QTensor(w, ws[:, None], "per_row_i8"))
    x = torch.randn(3, 272, generator=g, device=DEV).bfloat16()
    q, s = ops.quant_rows(x)
    assert torch.equal(lin(x), ops.gemm_w8a8(q, s, w, ws))


def test_status_words_end_a_step_and_a_prefill():
    """A word left in a workspace, as by a wait that gave up, raises at the next synchronisation;
    afterwards the pipeline gives what it gave before."""
    from superl8_serve_b200._lib import ERR_TIMEOUT, S8BError
    from superl8_serve_b200.config import tiny_moe
    from superl8_serve_b200.engine import DecodePipeline

    cfg = tiny_moe()
    prompts = _prompts([20, 3], cfg.vocab_size, 2)
    pipe = DecodePipeline(_models(cfg), batch=2, max_len=64, prefill_attention="chunk",
                          fused_moe=True)
    want = pipe.generate(prompts, 4, prefill=True)
    for ws in (pipe._pf[0][0].chunk_ws, pipe.runners[0].moe_buf["layer_ws"]):
        ws[:4].view(torch.int32).fill_(ERR_TIMEOUT)
        with pytest.raises(S8BError, match="invalid"):
            pipe.generate(prompts, 4, prefill=True)
        assert pipe.generate(prompts, 4, prefill=True) == want


@pytest.mark.parametrize("M,N,K", [(2, 260, 256), (3, 260, 256), (8, 24, 272), (9, 24, 272),
                                   (64, 1000, 512), (256, 264, 1024), (257, 264, 1024)])
def test_linear_layer_keeps_its_bits_in_every_form(M, N, K):
    from superl8_serve_b200 import ops
    from superl8_serve_b200.layers import LinearW8A8
    from superl8_serve_b200.weights import QTensor

    g = _gen(M + K)
    w, ws = _weight(g, N, K)
    lin = LinearW8A8(QTensor(w, ws, "per_row_i8"))
    x = torch.randn(M, K, generator=g, device=DEV).bfloat16()
    q, s = ops.quant_rows(x)
    want = ops.gemm_w8a8(q, s, w, ws)
    assert torch.equal(lin(x), want)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        y = lin(x)
    y.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want) and ops.linear_status(DEV) == 0


def test_linear_layer_needs_no_more_than_its_output():
    """256 rows of a head with 40,000 columns: no partial sums in memory beside the result."""
    from superl8_serve_b200.layers import LMHead
    from superl8_serve_b200.weights import QTensor

    g = _gen(8)
    w, ws = _weight(g, 40000, 1024)
    head = LMHead(QTensor(w, ws, "per_row_i8"))
    x = torch.randn(256, 1024, generator=g, device=DEV).bfloat16()
    y = head(x)
    out = y.numel() * 2
    del y
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    y = head(x)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before <= out + (1 << 20)


def test_status_word_of_calls_without_a_workspace():
    from superl8_serve_b200 import _lib, ops

    assert ops.linear_status(DEV) == 0
    ops._status[0][:4].view(torch.int32).fill_(_lib.ERR_TIMEOUT)
    assert ops.linear_status("cuda") == _lib.ERR_TIMEOUT
    assert ops.linear_status(torch.device(DEV)) == 0


def test_linear_layer_refuses_rows_of_another_length():
    from superl8_serve_b200.layers import LinearW8A8
    from superl8_serve_b200.weights import QTensor

    g = _gen(4)
    w, ws = _weight(g, 24, 256)
    for M in (1, 3, 300):
        with pytest.raises(ValueError, match="rows of 272"):
            LinearW8A8(QTensor(w, ws, "per_row_i8"))(torch.zeros(M, 272, device=DEV).bfloat16())


@pytest.mark.parametrize("moe", [False, True])
@pytest.mark.parametrize("stages", [1, 2])
def test_wide_chunks_in_every_kind_of_stage_step(moe, stages):
    """Prefill chunks above 256 rows, launch by launch and as native stage steps, dense and sparse: the
    bits of 256-row chunks, without partial sums for more than 256 rows in memory."""
    from superl8_serve_b200 import _lib
    from superl8_serve_b200.config import tiny, tiny_moe
    from superl8_serve_b200.engine import DecodePipeline

    cfg = tiny_moe() if moe else tiny()
    models = _models(cfg, stages)
    prompts = _prompts([300, 7, 411], cfg.vocab_size)
    got = []
    for native, chunk in ((False, 256), (False, 700), (True, 256), (True, 700)):
        pipe = DecodePipeline(models, batch=3, max_len=512)
        pipe.prefill_chunk = chunk
        if native:
            pipe.set_native()
        got.append(pipe.prefill(prompts, keep_logits=True))
        for r in pipe._pf[0]:
            most = max(_lib.load().s8b_gemm_tc_split_count(256, *w.shape) * w.shape[0]
                       for L in r.model.layers for w in L.matrices())
            assert r.m == chunk and r.part.numel() == 256 * most
    for toks, logits in got[1:]:
        assert toks == got[0][0]
        for a, b in zip(logits, got[0][1]):
            assert torch.equal(a, b)


@pytest.mark.parametrize("batch", [1, 5, 16])
def test_the_pipelines_fused_layer_is_the_operator(batch):
    """What the stage leaves is, bit for bit, ``ops.moe_layer`` of the layer's normalised rows."""
    from superl8_serve_b200 import ops
    from superl8_serve_b200.config import tiny_moe
    from superl8_serve_b200.engine import DecodePipeline

    cfg = tiny_moe(num_hidden_layers=1)
    models = _models(cfg)
    pipe = DecodePipeline(models, batch=batch, max_len=64, fused_moe=True)
    pipe.add_sequences()
    pipe.set_state([0] * batch, list(range(3, 3 + batch)), reserve=4)
    pipe.step()
    pipe.synchronize()
    r, mw = pipe.runners[0], models[0].layers[0].moe
    y = r.moe_buf["y"][:batch].clone()
    q, s = ops.quant_rows(y)
    want = ops.moe_layer(y, q, s, mw.router, mw.gu_w, mw.gu_s, mw.d_w, mw.d_s, mw.top_k,
                         norm_topk_prob=mw.norm_topk_prob, scaling=mw.scaling)
    assert torch.equal(r.h[:batch], want)


def test_status_word_made_in_inference_mode():
    """The device's word, first asked for by a layer under inference_mode, can be cleared outside of it."""
    from superl8_serve_b200 import _lib, ops
    from superl8_serve_b200.layers import LinearW8A8
    from superl8_serve_b200.weights import QTensor

    kept = ops._status.pop(0, None)
    try:
        g = _gen(2)
        w, ws = _weight(g, 64, 128)
        x = torch.randn(5, 128, generator=g, device=DEV).bfloat16()
        with torch.inference_mode():
            LinearW8A8(QTensor(w, ws, "per_row_i8"))(x)
        ops._status[0][:4].view(torch.int32).fill_(_lib.ERR_TIMEOUT)
        assert ops.linear_status(DEV) == _lib.ERR_TIMEOUT and ops.linear_status(DEV) == 0
    finally:
        if kept is not None:
            ops._status[0] = kept
