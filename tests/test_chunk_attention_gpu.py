"""GPU: attention of a chunk of new tokens over the paged cache (``s8b_paged_chunk_q8``)
against the formula in 64 bits.

Tolerance of one output value o_d = sum_j p_j vs_j v_jd / l: each weight p_j vs_j is rounded to
bf16 (half a step, 2^-8 relative), so o_d moves by at most 2^-8 A_d, A_d = sum_j p_j vs_j |v_jd| /
l. The exponents t (at most a few hundred here) carry binary32 roundings of a few 2^-24 |t|,
and the sums binary32 roundings: below 2e-4 A_d together. Then one rounding to the output type."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


class Case:
    def __init__(self, lens, Hq, Hkv, bs, seed=0, sharp=1.0, extra=0, tail=0):
        """lens: (new rows, context) per sequence; extra: unused block-table columns; tail: rows
        of q behind the last sequence."""
        g = torch.Generator(device=DEV)
        g.manual_seed(seed)
        codes = lambda *s: torch.randint(-127, 128, s, generator=g, device=DEV, dtype=torch.int8)  # noqa: E731
        uni = lambda lo, hi, *s: lo + (hi - lo) * torch.rand(s, generator=g, device=DEV)  # noqa: E731
        self.lens, self.Hq, self.Hkv, self.bs = lens, Hq, Hkv, bs
        S = len(lens)
        need = [-(-max(c, 0) // bs) for _, c in lens]
        nb = sum(need) + 2
        perm = torch.randperm(nb, generator=g, device=DEV).to(torch.int32)
        self.bt = torch.full((S, max(max(need), 1) + extra), 0, dtype=torch.int32, device=DEV)
        at = 0
        for i, n in enumerate(need):
            self.bt[i, :n] = perm[at:at + n]
            at += n
        self.free = perm[at:]  # pages of no sequence
        self.kc, self.vc = codes(nb, Hkv, bs, 128), codes(nb, Hkv, bs, 128)
        self.ks, self.vs = uni(0.01, 0.03, nb, Hkv, bs), uni(0.01, 0.05, nb, Hkv, bs)
        self.T = sum(n for n, _ in lens)
        self.q = codes(self.T + tail, Hq, 128)
        self.qs = uni(0.002, 0.01, self.T + tail, Hq) * sharp
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
        self.ctx = i32([c for _, c in lens])
        self.cu = i32([sum(n for n, _ in lens[:i]) for i in range(S + 1)])
        self.scale = 128 ** -0.5

    def run(self, dtype=torch.bfloat16, **kw):
        from superl8_serve_b200 import ops

        ws = kw.pop("workspace", None)
        ws = ops.chunk_workspace(DEV) if ws is None else ws
        out = ops.paged_chunk_q8(self.q, self.qs, self.kc, self.ks, self.vc, self.vs, self.bt,
                                 self.ctx, self.cu, self.scale, workspace=ws, dtype=dtype, **kw)
        torch.cuda.synchronize()
        assert int(ws[:4].view(torch.int32)) == 0
        return out

    def exact(self):
        """(o, A) in 64 bits, [T, Hq, 128] each."""
        o = torch.zeros(self.T, self.Hq, 128, dtype=torch.float64, device=DEV)
        A = torch.zeros_like(o)
        r0, G = 0, self.Hq // self.Hkv
        for i, (n, c) in enumerate(self.lens):
            pos = torch.arange(max(c, 0), device=DEV)
            blk, off = self.bt[i].long()[pos // self.bs], pos % self.bs
            hide = pos > c - n + torch.arange(n, device=DEV)[:, None]
            for g in range(self.Hkv):
                k = self.kc[blk, g, off].double() * self.ks[blk, g, off].double()[:, None]
                v = self.vc[blk, g, off].double() * self.vs[blk, g, off].double()[:, None]
                for h in range(g * G, (g + 1) * G):
                    q = self.q[r0:r0 + n, h].double() * self.qs[r0:r0 + n, h].double()[:, None]
                    p = torch.softmax((q @ k.T * self.scale).masked_fill(hide, float("-inf")), -1)
                    p = p.masked_fill(hide, 0.0)
                    o[r0:r0 + n, h] = p @ torch.where(hide.all(0)[:, None], 0.0, v)
                    A[r0:r0 + n, h] = p @ torch.where(hide.all(0)[:, None], 0.0, v.abs())
            r0 += n
        return o, A

    def check(self, out, rows=None, weights=2 ** -8):
        o, A = self.exact()
        out = out[:self.T].view(self.T, self.Hq, 128)
        # below a type's normal range its steps are those of the range's lower end: 2^-24 in fp16
        # (a value that ought to be 1e-15 becomes 0), so half a step is 2^-25 there; bf16 has
        # binary32's range
        least = 2.0 ** -25 if out.dtype == torch.float16 else 1e-30
        tol = (weights + 2e-4) * A + torch.finfo(out.dtype).eps / 2 * o.abs() + least
        bad = ~((out.double() - o).abs() <= tol)
        if rows is not None:
            bad = bad[rows]
        assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} off; first {bad.nonzero()[0].tolist()}, "
                               f"rows {bad.any(-1).any(-1).nonzero().flatten()[:8].tolist()}")


@pytest.mark.parametrize("n,c", [(1, 1), (1, 2), (1, 128), (1, 129), (2, 127), (5, 37), (31, 31),
                                 (32, 32), (33, 33), (64, 64), (65, 65), (64, 200), (100, 1000),
                                 (129, 129), (300, 300), (7, 5000), (257, 3001)])
def test_one_sequence(n, c):
    Case([(n, c)], 8, 2, 16, seed=n + c).check(Case([(n, c)], 8, 2, 16, seed=n + c).run())


@pytest.mark.parametrize("Hq,Hkv", [(4, 4), (4, 2), (21, 3), (32, 8), (40, 8), (12, 2), (32, 4),
                                    (24, 2), (16, 1), (33, 1), (128, 1)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_head_groups(Hq, Hkv, dtype):
    c = Case([(70, 70), (3, 140), (150, 400)], Hq, Hkv, 16, seed=Hq)
    c.check(c.run(dtype))


@pytest.mark.parametrize("bs", [1, 2, 4, 8, 16, 32, 64, 128, 256])
def test_block_sizes(bs):
    c = Case([(40, 300), (1, 7), (130, 131)], 8, 2, bs, seed=bs, extra=3)
    c.check(c.run())


def test_scales_off_a_16_byte_boundary():
    """Scale arrays that bulk copies cannot read give the same result."""
    c = Case([(40, 300), (130, 131)], 8, 2, 16, seed=61)
    want = c.run()
    for name in ("ks", "vs"):
        t = getattr(c, name)
        buf = torch.zeros(t.numel() + 1, device=DEV)
        buf[1:] = t.flatten()
        setattr(c, name, buf[1:].view(t.shape))
        assert torch.equal(c.run(), want)


def test_ragged_batch_with_idle_sequences():
    lens = [(0, 50), (5, 5), (0, 0), (1, 700), (40, 90), (0, 1), (128, 128), (2, 257), (0, 9)]
    c = Case(lens, 32, 8, 16, seed=5)
    c.check(c.run())


def test_many_short_sequences_and_split_items():
    c = Case([(4, 100 + 37 * i) for i in range(200)], 8, 2, 16, seed=9)
    c.check(c.run())


@pytest.mark.parametrize("S", [1, 3])
def test_long_context_is_split_over_ctas(S):
    c = Case([(3 + 7 * i, 20000 + 777 * i) for i in range(S)], 16, 2, 16, seed=S)
    c.check(c.run(torch.float16))


def test_sharp_softmax_moves_the_reference():
    """Scores of hundreds, growing along the context: the running maximum moves at many tiles."""
    c = Case([(70, 1500)], 8, 2, 16, seed=3, sharp=40.0)
    ramp = torch.linspace(0.05, 3.0, 1500, device=DEV)
    pos = torch.arange(1500, device=DEV)
    c.ks[c.bt[0].long()[pos // 16], :, pos % 16] *= ramp[:, None]
    c.check(c.run())


@pytest.mark.parametrize("n", [3, 70])
def test_jumps_beyond_the_reference(n):
    """Single keys far into the context whose scores lie hundreds above all before them: the
    weights of the tile overflow against the last reference."""
    c = Case([(n, 1400)], 8, 2, 16, seed=17)
    for pos, k in ((300, 40.0), (777, 120.0), (778, 119.0), (1250, 300.0)):
        c.ks[int(c.bt[0, pos // 16]), :, pos % 16] = k * 0.02
    c.check(c.run())
    c.check(c.run(torch.float16))


def test_rows_that_see_nothing():
    """More new rows than context: the first rows see no key and give zeros."""
    c = Case([(50, 20), (10, 0), (300, 7)], 8, 2, 16, seed=4)
    out = c.run()
    c.check(out)
    o = out.view(-1, 8, 128)
    assert (o[:30] == 0).all() and (o[50:60] == 0).all() and (o[60:353] == 0).all()
    assert (o[353:].abs().sum(-1) > 0).all()


def test_masked_places_may_hold_anything():
    """NaN and infinite scales of pages behind the context and of keys that a row does not see
    leave that row alone."""
    c = Case([(40, 200), (6, 30)], 8, 2, 16, seed=6)
    want = c.run()
    bad = torch.tensor([float("nan"), float("inf"), float("-inf"), 3e38], device=DEV)
    for page in c.free:
        c.ks[page] = bad[0]
        c.vs[page] = bad[1]
    for i, (_, n) in enumerate(c.lens):  # the rest of each last page
        page = int(c.bt[i, n // 16])
        c.ks[page, :, n % 16:] = bad[0]
        c.vs[page, :, n % 16:] = bad[0]
    assert torch.equal(c.run(), want)
    # the last new key of sequence 0: only the last row sees it
    page = int(c.bt[0, 199 // 16])
    for b in bad:
        c.vs[page, :, 199 % 16] = b
        c.ks[page, :, 199 % 16] = b if b != bad[3] else 1.0
        got = c.run()
        assert torch.equal(got[:39], want[:39]) and torch.equal(got[40:], want[40:])
        assert not torch.isfinite(got[39]).all()


def test_extreme_value_scales():
    """Value scales across binary32's range in one tile: nothing overflows or vanishes."""
    c = Case([(4, 256)], 4, 2, 16, seed=8)
    pos = torch.arange(256, device=DEV)
    c.vs[c.bt[0].long()[pos // 16], :, pos % 16] = torch.where(pos % 2 == 0, 1e-30, 1e-34)[:, None]
    o, A = c.exact()
    from superl8_serve_b200 import ops

    out = ops.paged_chunk_q8(c.q, c.qs, c.kc, c.ks, c.vc, c.vs, c.bt, c.ctx, c.cu, c.scale)
    err = (out.view(4, 4, 128).double() - o).abs()
    assert (err <= (2 ** -8 + 2e-4) * A + 2 ** -8 * o.abs()).all() and out.abs().max() > 0


def test_rows_behind_the_last_sequence_stay():
    c = Case([(9, 30), (4, 4)], 8, 2, 16, seed=12, tail=5)
    out = torch.full((18, 8 * 128), 7.0, dtype=torch.bfloat16, device=DEV)
    assert c.run(out=out) is out
    c.check(out)
    assert (out[13:] == 7.0).all()


def test_equals_the_prefill_rows_within_rounding():
    """The same rows through the framework's prefill attention: both are within rounding of the
    exact result, so within the sum of the two tolerances of each other."""
    from superl8_serve_b200 import ops

    lens = [(90, 90), (17, 300)]
    c = Case(lens, 32, 8, 16, seed=21)
    out = c.run()
    bt = torch.cat([c.bt[i:i + 1].expand(n, -1) for i, (n, _) in enumerate(lens)]).contiguous()
    ctx = torch.cat([torch.arange(m - n + 1, m + 1) for n, m in lens]).to(torch.int32).to(DEV)
    R = ops.prefill_block_rows(32, 8)
    rb = torch.tensor(ops.prefill_row_blocks([n for n, _ in lens], R), dtype=torch.int32, device=DEV)
    ref = ops.paged_prefill_q8(c.q, c.qs, c.kc, c.ks, c.vc, c.vs, bt, ctx, rb, 300, c.scale)
    _, A = c.exact()
    assert ((out.double() - ref.double()).abs() <= (3 * 2 ** -8) * A.view(c.T, -1)).all()


def test_same_on_every_run_and_workspace_reuse():
    from superl8_serve_b200 import ops

    ws = ops.chunk_workspace(DEV)
    a = Case([(64, 5000), (1, 3000)], 32, 8, 16, seed=1)
    b = Case([(300, 300)], 4, 2, 32, seed=2)
    ra, rb = a.run(workspace=ws), b.run(workspace=ws)
    for _ in range(5):
        assert torch.equal(a.run(workspace=ws), ra) and torch.equal(b.run(workspace=ws), rb)


def test_graph_replays_with_other_lengths():
    from superl8_serve_b200 import ops

    c = Case([(20, 400), (30, 500)], 8, 2, 16, seed=31)
    ws = ops.chunk_workspace(DEV)
    out = torch.zeros(50, 8 * 128, dtype=torch.bfloat16, device=DEV)
    args = (c.q, c.qs, c.kc, c.ks, c.vc, c.vs, c.bt, c.ctx, c.cu, c.scale)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        ops.paged_chunk_q8(*args, out=out, workspace=ws)
    st.synchronize()
    c.check(out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        ops.paged_chunk_q8(*args, out=out, workspace=ws)
    c.lens = [(45, 310), (5, 77)]
    c.ctx.copy_(torch.tensor([310, 77], dtype=torch.int32))
    c.cu.copy_(torch.tensor([0, 45, 50], dtype=torch.int32))
    for _ in range(2):
        out.zero_()
        g.replay()
    torch.cuda.synchronize()
    c.check(out)


def test_two_streams_with_their_own_workspaces():
    from superl8_serve_b200 import ops

    cs = [Case([(200, 900)], 8, 2, 16, seed=i) for i in (40, 41)]
    want = [c.run() for c in cs]
    sts = [torch.cuda.Stream() for _ in cs]
    wss = [ops.chunk_workspace(DEV) for _ in cs]
    torch.cuda.synchronize()
    outs = [None, None]
    for _ in range(4):
        for i, c in enumerate(cs):
            with torch.cuda.stream(sts[i]):
                outs[i] = ops.paged_chunk_q8(c.q, c.qs, c.kc, c.ks, c.vc, c.vs, c.bt, c.ctx, c.cu,
                                             c.scale, workspace=wss[i])
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w)


def test_bad_pages_and_lengths_are_reported():
    """Block ids, contexts and row ranges outside the tensors set the status word; nothing
    outside is read or written, and the other sequences are right."""
    from superl8_serve_b200 import _lib, ops

    c = Case([(8, 60), (8, 60)], 8, 2, 16, seed=51)
    want = c.run()

    def status(**kw):
        ws = ops.chunk_workspace(DEV)
        a = {"bt": c.bt, "ctx": c.ctx, "cu": c.cu, **kw}
        out = ops.paged_chunk_q8(c.q, c.qs, c.kc, c.ks, c.vc, c.vs, a["bt"], a["ctx"], a["cu"],
                                 c.scale, workspace=ws)
        torch.cuda.synchronize()
        return int(ws[:4].view(torch.int32)), out

    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    for page in (c.kc.shape[0], -1, 2 ** 31 - 1):
        bt = c.bt.clone()
        bt[0, 1] = page
        code, out = status(bt=bt)
        assert code == -8 and torch.equal(out[8:], want[8:])
    for ctx in (65, 2 ** 31 - 1, -5):
        code, out = status(ctx=i32(ctx, 60))
        assert code == -8 and torch.equal(out[8:], want[8:])
    assert status(cu=i32(0, 8, 17))[0] == -8
    assert status(cu=i32(-1, 8, 16))[0] == -8
    assert status(cu=i32(8, 4, 16))[0] == -8
    assert status()[0] == 0
    assert _lib.strerror(-8) == "null pointer or invalid argument"


@pytest.mark.parametrize("lens,dtype", [
    ([(5, 37)], torch.bfloat16), ([(1, 1), (256, 256), (7, 200)], torch.bfloat16),
    ([(40, 129), (3, 3)], torch.float16), ([(130, 700)], torch.float16),
])
def test_weights_of_two_terms(lens, dtype):
    """Tables of up to 256 keys, and fp16 results at any length: a weight is p1 + p2 in bf16, p2 what
    rounding to p1 left over (at most 2^-8 of it), itself off by at most 2^-8: 2^-16 in all."""
    c = Case(lens, 8, 2, 16)
    assert dtype == torch.float16 or c.bt.shape[1] * c.bs <= 256
    c.check(c.run(dtype=dtype), weights=2 ** -16)


def test_tables_on_both_sides_of_256_keys():
    """The same context behind a table of 256 and of 272 positions."""
    for extra in (0, 1):
        c = Case([(33, 250)], 4, 2, 16, seed=9, extra=extra)
        assert c.bt.shape[1] == 16 + extra
        c.check(c.run())


@pytest.mark.parametrize("Hq,Hkv,edge", [(4, 4, 32), (8, 4, 16), (6, 2, 8), (8, 2, 8), (10, 2, 4),
                                         (8, 1, 4), (9, 1, 0)])
def test_items_of_few_tokens(Hq, Hkv, edge):
    """On both sides of 32 / G tokens (each softmax warp has 8 rows, 8 / G whole tokens), alone and
    as a long sequence's rest, in one piece and cut over CTAs."""
    G = Hq // Hkv
    whole = 2 * (128 // G)
    lens = [(max(edge, 1), 70), (edge + 1, 300), (max(edge - 1, 1), 2000), (1, 1),
            (whole + max(edge, 1), whole + 150), (whole + edge + 1, whole + 400), (2, 5000)]
    c = Case(lens, Hq, Hkv, 16, seed=Hq)
    c.check(c.run())
    c.check(c.run(dtype=torch.float16), weights=2 ** -16)


def test_cuts_next_to_an_items_start():
    """Many items of one and two key tiles: cuts fall before, among and behind their first units."""
    c = Case([(1 + i % 5, 1 + 37 * i % 260 + 5) for i in range(70)], 8, 4, 16, seed=4)
    c.check(c.run())


def test_pieces_of_one_tile_between_longer_ones():
    """The groups of a piece of one key tile do not both work: the order between pieces has to hold
    however the runs fall in time."""
    from superl8_serve_b200 import ops

    c = Case([(1 + (i * 7) % 40, 41 + 97 * i % 900) for i in range(60)], 8, 2, 16, seed=5)
    ws = ops.chunk_workspace(DEV)
    want = c.run(workspace=ws)
    c.check(want)
    for _ in range(50):
        assert torch.equal(ops.paged_chunk_q8(c.q, c.qs, c.kc, c.ks, c.vc, c.vs, c.bt, c.ctx,
                                              c.cu, c.scale, workspace=ws), want)


@pytest.mark.parametrize("lens", [[(5, 37)], [(1, 1), (3, 3), (40, 41)], [(33, 250)], [(70, 2100)]])
def test_weights_keep_16_bits_behind_any_table(lens):
    """bf16 results too, and where rows see few of the keys that the table reaches: a weight is p1 + p2
    in bf16, off by at most 2^-16 of it, so that the output's own rounding is what remains."""
    for extra in (0, 1, 200):
        c = Case(lens, 8, 2, 16, seed=71, extra=extra)
        c.check(c.run(), weights=2 ** -16)


def test_the_tables_width_does_not_show():
    """The same sequences behind tables of other widths: the same bits."""
    want = Case([(33, 250), (5, 37)], 8, 2, 16, seed=72).run()
    for extra in (1, 2, 113):
        assert torch.equal(Case([(33, 250), (5, 37)], 8, 2, 16, seed=72, extra=extra).run(), want)


def test_no_sequence_brings_a_row():
    """All chunks empty: nothing is written, and the workspace serves the next call."""
    from superl8_serve_b200 import ops

    c = Case([(9, 300), (4, 70)], 8, 2, 16, seed=81)
    ws = ops.chunk_workspace(DEV)
    want = c.run(workspace=ws)
    out = torch.full_like(want, 7.0)
    ops.paged_chunk_q8(c.q, c.qs, c.kc, c.ks, c.vc, c.vs, c.bt, c.ctx, torch.zeros_like(c.cu), c.scale,
                       out=out, workspace=ws)
    assert (out == 7.0).all() and int(ws[:4].view(torch.int32)) == 0
    assert torch.equal(c.run(workspace=ws), want)
