"""GPU: the few-row MoE layer (``s8b_moe_layer``) against its definition in 64 bits.

Tolerance. Integer products are exact. The act row a is binary32 (exp within 1e-6 relative), so
its codes are those of the exact row except where a / step lies within about 1e-4 of a half
(127 codes, 1e-6 relative): such a code is one step off. At most a few of a row's F codes are, so
one row's share of out moves by |w| step ds |d_w| <= 127 |w| as ds for each of them; the test
allows two per row. All else is binary32 (below 1e-5 of the sum of magnitudes), then one rounding to the
output type."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


class Layer:
    def __init__(self, T, H, F, E, k, dtype=torch.bfloat16, seed=0, spread=1.0):
        g = torch.Generator(device=DEV)
        g.manual_seed(seed)
        codes = lambda *s: torch.randint(-127, 128, s, generator=g, device=DEV, dtype=torch.int8)  # noqa: E731
        self.k, self.F = k, F
        self.y = torch.randn(T, H, generator=g, device=DEV).to(dtype)
        self.quantize()
        self.gate = spread * torch.randn(E, H, generator=g, device=DEV) / math.sqrt(H)
        self.gu_w, self.d_w = codes(E, 2 * F, H), codes(E, H, F)
        self.gu_s = (0.5 + torch.rand(E, 2 * F, generator=g, device=DEV)) / (73 * math.sqrt(H))
        self.d_s = (0.5 + torch.rand(E, H, generator=g, device=DEV)) / (73 * math.sqrt(F))

    def quantize(self):
        from superl8_serve_b200 import ops

        self.xq, self.xs = ops.quant_rows(self.y)

    def run(self, **kw):
        from superl8_serve_b200 import ops

        ws = kw.pop("workspace", None)
        ws = ops.moe_layer_workspace(self.k, self.F, DEV) if ws is None else ws
        out = ops.moe_layer(self.y, self.xq, self.xs, self.gate, self.gu_w, self.gu_s, self.d_w,
                            self.d_s, self.k, workspace=ws, **kw)
        torch.cuda.synchronize()
        assert int(ws[:4].view(torch.int32)) == 0
        return out

    def exact(self, norm=True, scaling=1.0):
        """(out, tolerance before the output's rounding), 64 bits."""
        T, H = self.y.shape
        p = torch.softmax(self.y.double() @ self.gate.double().T, -1)
        w, e = torch.sort(p, dim=-1, descending=True, stable=True)
        w, e = w[:, :self.k], e[:, :self.k]
        if norm:
            w = w / w.sum(-1, keepdim=True).clamp(min=1e-9)
        w = w * scaling
        out = torch.zeros(T, H, dtype=torch.float64, device=DEV)
        tol = torch.zeros_like(out)
        for t in range(T):
            for j in range(self.k):
                i = int(e[t, j])
                gu = (self.gu_w[i].double() @ self.xq[t].double()) * self.xs[t].double() * self.gu_s[i].double()
                a = gu[:self.F] * torch.sigmoid(gu[:self.F]) * gu[self.F:]
                step = a.abs().max() / 127
                q = torch.round(a / step) if step > 0 else torch.zeros_like(a)
                d = self.d_w[i].double()
                out[t] += w[t, j] * step * self.d_s[i].double() * (d @ q)
                tol[t] += w[t, j].abs() * step * self.d_s[i].double() * (2 * 127 + 1e-5 * (d.abs() @ q.abs()))
        return out, tol

    def check(self, out, **kw):
        ref, tol = self.exact(**kw)
        tol = tol + torch.finfo(out.dtype).eps / 2 * ref.abs() + torch.finfo(out.dtype).tiny
        bad = ~((out.double() - ref).abs() <= tol)
        assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, first {bad.nonzero()[0].tolist()}"
        rel = ((out.double() - ref).norm() / ref.norm()).item()
        assert rel < torch.finfo(out.dtype).eps  # flipped codes are few


@pytest.mark.parametrize("T,H,F,E,k", [
    (1, 16, 16, 1, 1), (1, 256, 128, 16, 4), (2, 64, 48, 8, 8), (3, 272, 80, 5, 2),
    (5, 512, 144, 33, 3), (7, 1040, 272, 20, 3), (16, 256, 128, 16, 4), (16, 256, 512, 4, 4),
    (16, 528, 1040, 7, 1), (4, 4112, 96, 64, 6), (1, 2048, 768, 128, 8), (8, 2048, 768, 128, 8),
    (16, 2048, 768, 128, 8), (9, 128, 64, 256, 16), (2, 8192, 256, 6, 2),
])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_sizes(T, H, F, E, k, dtype):
    L = Layer(T, H, F, E, k, dtype, seed=T + H + E)
    L.check(L.run())


@pytest.mark.parametrize("norm,scaling", [(True, 2.5), (False, 1.0), (False, 0.3)])
def test_weights(norm, scaling):
    L = Layer(6, 256, 128, 16, 4, seed=3, spread=3.0)
    L.check(L.run(norm_topk_prob=norm, scaling=scaling), norm=norm, scaling=scaling)


def test_all_rows_choose_the_same_experts():
    L = Layer(16, 512, 256, 32, 3, seed=5)
    L.y[:] = L.y[0]
    L.quantize()
    out = L.run()
    L.check(out)
    assert (out == out[0]).all()


def test_equal_logits_go_to_the_lowest_experts():
    L = Layer(3, 256, 128, 12, 4, seed=7)
    L.gate[:] = L.gate[0]
    out = L.run()
    sub = Layer(3, 256, 128, 12, 4, seed=7)
    for n in ("gate", "gu_w", "gu_s", "d_w", "d_s"):
        setattr(sub, n, getattr(L, n)[:4].contiguous())
    assert torch.equal(out, sub.run())


def test_equals_the_general_path_within_its_roundings():
    """Route, grouped GEMMs and combine round to dtype after every step: 2^-8 each on gate, up,
    silu, the product, the down row, its weight, the weighting and up to k additions."""
    from superl8_serve_b200 import ops

    T, H, F, E, k = 8, 512, 256, 32, 4
    L = Layer(T, H, F, E, k, seed=9)
    out = L.run()
    r = ops.moe_route(L.y, L.gate, k)
    gu = ops.moe_gemm_grouped(L.xq, L.xs, L.gu_w, L.gu_s, r["offsets"], row_index=r["sorted_token"],
                              A=T * k)
    aq, asc, _ = ops.silu_mul_quant(gu)
    part = ops.moe_gemm_grouped(aq, asc, L.d_w, L.d_s, r["offsets"], A=T * k)
    old = ops.moe_combine(part, r["topw"], r["topi"], r["assign_pos"])
    assert ((out.double() - old.double()).norm() / old.double().norm()).item() < 16 * 2 ** -8


def test_zero_rows_and_non_finite_rows():
    """A row of zeros gives zeros; a NaN row gives its own NaN and leaves the others alone."""
    L = Layer(5, 256, 128, 16, 4, seed=11)
    L.y[1] = 0
    L.quantize()
    want = L.run()
    assert (want[1] == 0).all()
    L.y[3] = float("nan")
    got = L.run()
    keep = [0, 1, 2, 4]
    assert torch.equal(got[keep], want[keep])
    L.xs[2] = float("inf")
    got = L.run()
    assert torch.equal(got[[0, 1, 4]], want[[0, 1, 4]]) and not torch.isfinite(got[2]).any()


def test_same_on_every_run_and_workspace_reuse():
    from superl8_serve_b200 import ops

    ws = ops.moe_layer_workspace(8, 768, DEV)
    a, b = Layer(16, 1024, 768, 64, 8, seed=1), Layer(2, 256, 128, 16, 4, seed=2)
    ra, rb = a.run(workspace=ws), b.run(workspace=ws)
    for _ in range(20):
        assert torch.equal(a.run(workspace=ws), ra) and torch.equal(b.run(workspace=ws), rb)


def test_graph_and_out():
    from superl8_serve_b200 import ops

    L = Layer(4, 256, 128, 16, 4, seed=13)
    ws = ops.moe_layer_workspace(4, 128, DEV)
    out = torch.full((6, 256), 5.0, dtype=torch.bfloat16, device=DEV)
    args = (L.y, L.xq, L.xs, L.gate, L.gu_w, L.gu_s, L.d_w, L.d_s, 4)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(st):
        ops.moe_layer(*args, out=out[1:5], workspace=ws)
    st.synchronize()
    assert torch.equal(out[1:5], L.run())
    with torch.cuda.graph(g, stream=st):
        ops.moe_layer(*args, out=out[1:5], workspace=ws)
    M = Layer(4, 256, 128, 16, 4, seed=14)
    L.y.copy_(M.y)
    L.xq.copy_(M.xq)
    L.xs.copy_(M.xs)
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    L.check(out[1:5])
    assert (out[0] == 5).all() and (out[5] == 5).all()


def test_two_streams_with_their_own_workspaces():
    """Each launch needs every SM for its barriers: launches of two streams take turns."""
    from superl8_serve_b200 import ops

    Ls = [Layer(16, 1024, 512, 32, 4, seed=21), Layer(3, 512, 256, 8, 2, seed=22)]
    want = [L.run() for L in Ls]
    sts = [torch.cuda.Stream() for _ in Ls]
    wss = [ops.moe_layer_workspace(L.k, L.F, DEV) for L in Ls]
    outs = [[], []]
    torch.cuda.synchronize()
    for _ in range(10):
        for i, L in enumerate(Ls):
            with torch.cuda.stream(sts[i]):
                outs[i].append(ops.moe_layer(L.y, L.xq, L.xs, L.gate, L.gu_w, L.gu_s, L.d_w,
                                             L.d_s, L.k, workspace=wss[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert int(wss[i][:4].view(torch.int32)) == 0
        assert all(torch.equal(o, want[i]) for o in outs[i])


def test_a_workspace_whose_wait_gave_up_is_not_used():
    """What a launch that gave up leaves (status word, counter with its top bit and some arrivals): later
    launches write nothing and do not wait; after the header is zeroed, results are right again."""
    from superl8_serve_b200 import _lib, ops

    L = Layer(5, 256, 128, 16, 4, seed=31)
    ws = ops.moe_layer_workspace(4, 128, DEV)
    want = L.run(workspace=ws)
    for count in (0, 1, 147, 2 ** 40 + 5):
        ws[:4].view(torch.int32).fill_(_lib.ERR_TIMEOUT)
        ws[64:72].view(torch.int64).fill_(count - 2 ** 63)
        out = torch.full_like(want, 3.0)
        for _ in range(3):
            ops.moe_layer(L.y, L.xq, L.xs, L.gate, L.gu_w, L.gu_s, L.d_w, L.d_s, 4, out=out,
                          workspace=ws)
        torch.cuda.synchronize()
        assert (out == 3.0).all()
        assert int(ws[:4].view(torch.int32)) == _lib.ERR_TIMEOUT
        assert int(ws[64:72].view(torch.int64)) < 0
        ws[:256].zero_()
        assert torch.equal(L.run(workspace=ws), want)
