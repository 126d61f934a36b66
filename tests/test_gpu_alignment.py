"""-m gpu: cross attention (forward, backward, attention mass) and per-utterance group norm against their definitions in
float64, with element-wise bounds counted from the arithmetic: u = 2^-24 per fp32 operation, h = half a step of the output's
type (bf16 2^-8, fp32 2^-24)."""
import math

import numpy as np
import pytest
import torch
import torch.nn.functional as F

from fastspeech2_amd import hip
from fastspeech2_amd.hip import call, ptr, stream
from tests.test_gpu_dropout import drop_mul

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
LOG2E = math.log2(math.e)
HALF = {"fp32": 2.0 ** -24, "bf16": 2.0 ** -8}
TDT = {"fp32": torch.float32, "bf16": torch.bfloat16}
CODE = {"fp32": 0, "bf16": 1}


def _cu(lens):
    return torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device=DEV)


def _bytes(name, *args):
    n = int(getattr(hip.load(), name)(*args))
    return torch.full((max(n, 16),), 0xFF, dtype=torch.uint8, device=DEV)        # NaN wherever it is read before it is written


class Problem:
    """Packed q [Mq + 3, ldq], fused k | v [Mk + 3, ldk] with NaN behind the last utterance, on CPU (float64) and device."""

    def __init__(self, lq, lk, H, KV, dk, dtype, seed=0, pad=0, scale=1.0):
        g = torch.Generator().manual_seed(seed * 7919 + sum(lq) * 31 + sum(lk) + 17 * H + KV + dk)
        self.lq, self.lk, self.H, self.KV, self.dk, self.dtype = list(lq), list(lk), H, KV, dk, dtype
        self.B, self.Mq, self.Mk = len(lq), sum(lq) + 3, sum(lk) + 3
        self.ldq, self.ldk = H * dk + pad, 2 * KV * dk + pad
        t = TDT[dtype]

        def make(rows, cols, s=1.0):
            x = (torch.randn(rows, cols, generator=g) * s).to(t)
            x[-3:] = math.nan
            return x
        self.q, self.kv = make(self.Mq, self.ldq, scale), make(self.Mk, self.ldk)
        self.dctx = make(self.Mq, self.ldq, 0.5)
        self.cq, self.ck = [0] + list(np.cumsum(lq)), [0] + list(np.cumsum(lk))
        self.d = {k: getattr(self, k).to(DEV) for k in ("q", "kv", "dctx")}
        self.cu_q, self.cu_k = _cu(lq), _cu(lk)
        self.max_q, self.max_k = max(lq), max(lk)
        self.half = KV * dk * self.kv.element_size()

    def forward(self, drop=(0, 0, 0.0), ws=None, ctx=None, lse=None, want_lse=True):
        t = TDT[self.dtype]
        ctx = torch.full((self.Mq, self.ldq), 7.0, dtype=t, device=DEV) if ctx is None else ctx
        lse = torch.full((self.H, self.Mq), 7.0, device=DEV) if lse is None else lse
        if ws is None:
            ws = _bytes("fs2_cross_attention_workspace", self.B, self.max_q, self.max_k, self.Mq, self.H, self.KV, self.dk,
                        CODE[self.dtype])
        kv = ptr(self.d["kv"])
        call("fs2_cross_attention", ptr(self.d["q"]), kv, kv + self.half, ptr(ctx), ptr(lse) if want_lse else None, ptr(self.cu_q),
             ptr(self.cu_k), ptr(ws), self.B, self.max_q, self.max_k, self.Mq, self.Mk, self.H, self.KV, self.dk, self.ldq, self.ldk,
             self.ldk, self.ldq, CODE[self.dtype], *drop, stream())
        return ctx, lse

    def backward(self, ctx, lse, drop=(0, 0, 0.0), ws=None, dq=None, dkv=None):
        t = TDT[self.dtype]
        dq = torch.full((self.Mq, self.ldq), 7.0, dtype=t, device=DEV) if dq is None else dq
        dkv = torch.full((self.Mk, self.ldk), 7.0, dtype=t, device=DEV) if dkv is None else dkv
        if ws is None:
            ws = _bytes("fs2_cross_attention_bwd_workspace", self.B, self.max_q, self.max_k, self.Mq, self.Mk, self.H, self.KV,
                        self.dk, CODE[self.dtype])
        kv = ptr(self.d["kv"])
        call("fs2_cross_attention_bwd", ptr(self.d["q"]), kv, kv + self.half, ptr(ctx), ptr(self.d["dctx"]), ptr(lse), ptr(dq),
             ptr(dkv), ptr(dkv) + self.half, ptr(self.cu_q), ptr(self.cu_k), ptr(ws), self.B, self.max_q, self.max_k, self.Mq, self.Mk,
             self.H, self.KV, self.dk, self.ldq, self.ldk, self.ldk, self.ldq, CODE[self.dtype], *drop, stream())
        return dq, dkv

    def mass(self, lse, ws=None):
        out = torch.full((self.H, self.Mk), 7.0, device=DEV)
        if ws is None:
            ws = _bytes("fs2_cross_attention_mass_workspace", self.B, self.max_q, self.max_k, self.Mk, self.H, self.KV, self.dk,
                        CODE[self.dtype])
        call("fs2_cross_attention_mass", ptr(self.d["q"]), ptr(self.d["kv"]), ptr(lse), ptr(out), ptr(self.cu_q), ptr(self.cu_k),
             ptr(ws), self.B, self.max_q, self.max_k, self.Mq, self.Mk, self.H, self.KV, self.dk, self.ldq, self.ldk,
             CODE[self.dtype], stream())
        return out

    def pairs(self):
        for b in range(self.B):
            for h in range(self.H):
                j = h // (self.H // self.KV)
                yield (b, h, slice(self.cq[b], self.cq[b + 1]), slice(self.ck[b], self.ck[b + 1]),
                       slice(h * self.dk, (h + 1) * self.dk), slice(j * self.dk, (j + 1) * self.dk),
                       slice((self.KV + j) * self.dk, (self.KV + j + 1) * self.dk))

    def exact(self, drop=(0, 0, 0.0)):
        """results and bounds, everything float64.  Scores: dk products and sums, the scaling and the subtraction of the maximum
        or lse, dS = (dk + 4) u sum|q||k| / sqrt(dk).  A probability: twice that (numerator and sum), exp2 and its argument
        (|S| u each, two units of the last place), the sum of n terms: rP = 2 dS + (2 n + 16) u + 4 |S|max u.
        ctx: sum P|v| (rP + n u + half a step where bf16 rounds P), then half a step of the result."""
        q, kv, do = self.q.double(), self.kv.double(), self.dctx.double()
        ctx, lse = torch.zeros(self.Mq, self.H * self.dk, dtype=torch.float64), torch.full((self.H, self.Mq), -math.inf, dtype=torch.float64)
        dq, dkv = torch.zeros_like(ctx), torch.zeros(self.Mk, 2 * self.KV * self.dk, dtype=torch.float64)
        mass = torch.zeros(self.H, self.Mk, dtype=torch.float64)
        tol = {k: torch.zeros_like(v) for k, v in dict(ctx=ctx, lse=lse, dq=dq, dkv=dkv, mass=mass).items()}
        hp = HALF[self.dtype] if self.dtype == "bf16" else 0.0
        ho = HALF[self.dtype]
        s = self.dk ** -0.5
        for b, h, rq, rk, hc, kc, vc in self.pairs():
            n, nq = rk.stop - rk.start, rq.stop - rq.start
            if n == 0 or nq == 0:
                continue
            Q, K, V, D = q[rq, hc], kv[rk, kc], kv[rk, vc], do[rq, hc]
            S = Q @ K.T * s
            P = torch.softmax(S, 1)
            M = drop_mul(drop[0], drop[1] + h, nq, n, drop[2], rq.start) if drop[2] else torch.ones_like(P)
            dS = (self.dk + 4) * U * (Q.abs() @ K.abs().T) * s
            dmax = dS.max(1, keepdim=True).values
            rP = dS + dmax + (2 * n + 16) * U + 4 * U * LOG2E * S.abs().max(1, keepdim=True).values
            O = (P * M) @ V
            ctx[rq, hc] = O
            eO = (P * M * (rP + n * U + 2 * U + hp)) @ V.abs() + 2 * U * O.abs()
            tol["ctx"][rq, hc] = eO + ho * (O.abs() + eO)
            lse[h, rq] = torch.logsumexp(S, 1) * LOG2E
            tol["lse"][h, rq] = (dmax[:, 0] + (n + 8) * U) * LOG2E + 8 * U * (1 + lse[h, rq].abs())
            rB = rP + 8 * U * (1 + lse[h, rq].abs())[:, None]                # P again, from the stored lse
            dP = (D @ V.T) * M
            delta = (D * O).sum(1, keepdim=True)
            eD = (D.abs() * (tol["ctx"][rq, hc] + self.dk * U * O.abs())).sum(1, keepdim=True)
            G = P * (dP - delta)
            eG = rB * G.abs() + P * ((self.dk + 2) * U * (D.abs() @ V.abs().T) * M + eD + 4 * U * (dP.abs() + delta.abs()))
            eG = eG + hp * (G.abs() + eG)
            dq[rq, hc] = G @ K * s
            tol["dq"][rq, hc] = (eG + n * U * G.abs()) @ K.abs() * s
            g = self.H // self.KV
            dkv[rk, kc] += G.T @ Q * s
            tol["dkv"][rk, kc] += (eG + (g * nq + 40) * U * G.abs()).T @ Q.abs() * s
            PM = P * M
            dkv[rk, vc] += PM.T @ D
            tol["dkv"][rk, vc] += (PM * (rB + (g * nq + 40) * U + hp)).T @ D.abs()
            mass[h, rk] = P.sum(0)
            tol["mass"][h, rk] = (P * (rB + (nq + 8) * U)).sum(0)
        for k, v in (("dq", dq), ("dkv", dkv)):
            tol[k] += ho * (v.abs() + tol[k]) + 2 * U * v.abs()
        return dict(ctx=ctx, lse=lse, dq=dq, dkv=dkv, mass=mass), tol


def _near(got, want, tol, rows, what):
    """got (device, rows of a matrix) within tol of want on `rows`; every row behind them still 7"""
    got = got.cpu().double()
    cols = want.shape[1]
    off = (got[:rows, :cols] - want[:rows]).abs()
    bad = off > tol[:rows] + 1e-30
    assert not bad.any() and not torch.isnan(off).any(), \
        "%s: %d of %d outside, worst %.3g of its bound" % (what, int(bad.sum()), bad.numel(), float((off / (tol[:rows] + 1e-30)).max()))
    assert (got[rows:] == 7.0).all(), what + ": rows behind the last utterance were written"
    if got.shape[1] > cols:
        assert (got[:, cols:] == 7.0).all(), what + ": columns behind the heads were written"


def _near_heads(got, want, tol, rows, what):
    got = got.cpu().double()
    w, g = want[:, :rows], got[:, :rows]
    assert torch.equal(torch.isinf(w), torch.isinf(g)), what
    off = torch.where(torch.isinf(w), 0.0, g - w).abs()
    bad = off > torch.where(torch.isinf(w), 0.0, tol[:, :rows]) + 1e-30
    assert not bad.any() and not torch.isnan(off).any(), "%s: %d outside, worst %.3g" % (what, int(bad.sum()), float(off.max()))
    assert (got[:, rows:] == 7.0).all(), what + ": rows behind the last utterance were written"


SHAPES = [
    # lq, lk, H, KV, dk, pad
    ([1], [1], 1, 1, 32, 0),                                       # one query, one key
    ([1] * 6, [3, 64, 1, 120, 33, 0], 2, 2, 128, 0),               # one frame each, one utterance without keys
    ([1, 0, 1, 1], [31, 32, 33, 65], 8, 2, 64, 8),                 # shared heads, an utterance without a frame
    ([2, 1, 2], [100, 7, 260], 8, 1, 96, 0),                       # all heads share one key head, 16 packed rows
    ([1], [1500], 2, 1, 128, 0),                                   # keys over several workgroups
    ([3, 1], [1900, 0], 4, 2, 32, 0),                              # ... and an utterance with none
    ([5, 17, 64, 65, 1, 130], [64, 65, 1, 63, 200, 2], 2, 2, 128, 0),
    ([129, 0, 40], [0, 9, 77], 4, 2, 96, 0),                       # no keys, no queries
    ([33, 70], [129, 191], 6, 2, 64, 16),                          # three heads to a key head
    ([300, 211], [12, 90], 4, 1, 32, 0),
    ([40], [900], 2, 2, 64, 0),                                    # few rows, long keys: split and merged
    ([17, 30, 0], [0, 1030, 5], 4, 4, 128, 0),
    ([700], [301], 2, 1, 128, 8),
    ([2, 1], [20000, 17], 2, 1, 96, 0),                            # more than 32 key ranges for a few rows
]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("lq,lk,H,KV,dk,pad", SHAPES)
def test_cross_attention(lq, lk, H, KV, dk, pad, dtype):
    p = Problem(lq, lk, H, KV, dk, dtype, pad=pad, scale=1.5)
    want, tol = p.exact()
    ctx, lse = p.forward()
    _near(ctx, want["ctx"], tol["ctx"], sum(lq), "ctx")
    _near_heads(lse, want["lse"], tol["lse"], sum(lq), "lse")
    again, none = p.forward(want_lse=False)
    assert torch.equal(again, ctx) and (none == 7.0).all()
    m = p.mass(lse)
    _near_heads(m, want["mass"], tol["mass"], sum(lk), "mass")
    assert torch.equal(p.mass(lse), m)
    dq, dkv = p.backward(ctx, lse)
    _near(dq, want["dq"], tol["dq"], sum(lq), "dq")
    _near(dkv, want["dkv"], tol["dkv"], sum(lk), "dk, dv")
    dq2, dkv2 = p.backward(ctx, lse)
    assert torch.equal(dq, dq2) and torch.equal(dkv, dkv2)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("lq,lk,H,KV,dk", [([90, 33], [70, 40], 4, 2, 64), ([1, 1], [40, 100], 4, 1, 128), ([30], [700], 2, 2, 96),
                                           ([400, 3], [301, 9], 4, 2, 128), ([1, 2], [1500, 40], 4, 2, 32)])
def test_cross_attention_dropout(lq, lk, H, KV, dk, dtype):
    drop = (12345, 9, 0.25)
    p = Problem(lq, lk, H, KV, dk, dtype, seed=4)
    want, tol = p.exact(drop)
    ctx, lse = p.forward(drop)
    _near(ctx, want["ctx"], tol["ctx"], sum(lq), "ctx")
    _near_heads(lse, want["lse"], tol["lse"], sum(lq), "lse")
    dq, dkv = p.backward(ctx, lse, drop)
    _near(dq, want["dq"], tol["dq"], sum(lq), "dq")
    _near(dkv, want["dkv"], tol["dkv"], sum(lk), "dk, dv")


def test_cross_attention_gradient_against_differences():
    """d <ctx, dctx> along a direction = central difference of two forwards.  fp32, step 1/64: the cubic term is step^2 / 6 of a
    third derivative that the sizes here keep below ~50 |derivative scale|, the noise of a forward ~1e-6 |ctx||dctx| / step."""
    p = Problem([19, 40], [33, 21], 4, 2, 64, "fp32", seed=9)
    ctx, lse = p.forward()
    dq, dkv = p.backward(ctx, lse)
    g = torch.Generator().manual_seed(1)
    step = 1.0 / 64
    nq, nk = sum(p.lq), sum(p.lk)
    for name, grad, rows in (("q", dq, nq), ("kv", dkv, nk)):
        base = p.d[name].clone()
        u = torch.randn(base.shape, generator=g).to(DEV)
        u[rows:] = 0
        want = float((grad[:rows].double() * u[:rows].double()).sum())
        vals = []
        for sgn in (1, -1):
            p.d[name] = base + sgn * step * u
            vals.append(float((p.forward()[0][:nq].double() * p.d["dctx"][:nq].double()).sum()))
        p.d[name] = base
        norm = float(grad[:rows].double().norm()) * math.sqrt(grad.shape[1] * rows) ** 0.5
        assert abs((vals[0] - vals[1]) / (2 * step) - want) <= 5e-3 * max(abs(want), norm), name


def test_infinite_and_nan_neighbours_stay_where_they_are():
    """an utterance of NaN keys and values, and one of infinities, change no other utterance"""
    lq, lk = [20, 33, 5, 1], [64, 65, 3, 40]
    for dtype in ("fp32", "bf16"):
        p = Problem(lq, lk, 2, 2, 64, dtype, seed=2)
        clean = p.forward()
        cleanb = p.backward(*clean)
        p.d["kv"][p.ck[1]:p.ck[2]] = math.nan
        p.d["kv"][p.ck[2]:p.ck[3]] = math.inf
        dirty = p.forward()
        dirtyb = p.backward(*dirty)
        for b in (0, 3):
            rq, rk = slice(p.cq[b], p.cq[b + 1]), slice(p.ck[b], p.ck[b + 1])
            assert torch.equal(clean[0][rq], dirty[0][rq]) and torch.equal(clean[1][:, rq], dirty[1][:, rq])
            assert torch.equal(cleanb[0][rq], dirtyb[0][rq]) and torch.equal(cleanb[1][rk], dirtyb[1][rk])
        assert torch.isnan(dirty[0][p.cq[1]:p.cq[2]]).all()


def test_batch_row_equals_the_utterance_alone():
    """the same kernel form for both: bit-equal"""
    lq, lk = [200, 150, 256], [90, 64, 120]
    p = Problem(lq, lk, 2, 2, 128, "bf16", seed=6)
    ctx, _ = p.forward()
    for b in range(3):
        one = Problem(lq[b:b + 1], lk[b:b + 1], 2, 2, 128, "bf16")
        for name, c in (("q", p.cq), ("kv", p.ck)):
            one.d[name][:c[b + 1] - c[b]] = p.d[name][c[b]:c[b + 1]]
        assert torch.equal(one.forward()[0][:lq[b]], ctx[p.cq[b]:p.cq[b + 1]])


def test_keys_beyond_32_bit_offsets():
    """an utterance whose keys lie more than 2^31 elements behind the pointer (and 2^32 bytes)"""
    rows, n, dk = 17_000_000, 70, 64
    kv = torch.zeros(rows, 2 * dk, dtype=torch.bfloat16, device=DEV)
    assert (rows - n) * 2 * dk > 2 ** 31
    small = Problem([20, 1], [n, 0], 1, 1, dk, "bf16")
    kv[-n:] = small.d["kv"][:n]
    lq = 20
    ctx, lse = torch.empty(lq, dk, dtype=torch.bfloat16, device=DEV), torch.empty(1, lq, device=DEV)
    dq, dkv = torch.empty_like(ctx), torch.empty(rows, 2 * dk, dtype=torch.bfloat16, device=DEV)
    mass = torch.empty(1, rows, device=DEV)
    cu_q, cu_k = _cu([lq]), torch.tensor([rows - n, rows], dtype=torch.int32, device=DEV)
    ws = _bytes("fs2_cross_attention_bwd_workspace", 1, lq, n, lq, rows, 1, 1, dk, 1)
    s = stream()
    for nq in (lq, 1):              # the rows kernel and the few-rows kernel
        q_cu = _cu([nq])
        call("fs2_cross_attention", ptr(small.d["q"]), ptr(kv), ptr(kv) + 2 * dk, ptr(ctx), ptr(lse), ptr(q_cu), ptr(cu_k), None, 1, nq,
             n, lq, rows, 1, 1, dk, dk, 2 * dk, 2 * dk, dk, 1, 0, 0, 0.0, s)
        want = small.forward()[0]
        if nq == lq:
            assert torch.equal(ctx, want[:lq])
            call("fs2_cross_attention_bwd", ptr(small.d["q"]), ptr(kv), ptr(kv) + 2 * dk, ptr(ctx), ptr(small.d["dctx"]), ptr(lse),
                 ptr(dq), ptr(dkv), ptr(dkv) + 2 * dk, ptr(cu_q), ptr(cu_k), ptr(ws), 1, lq, n, lq, rows, 1, 1, dk, dk, 2 * dk,
                 2 * dk, dk, 1, 0, 0, 0.0, s)
            w = _bytes("fs2_cross_attention_mass_workspace", 1, lq, n, rows, 1, 1, dk, 1)
            call("fs2_cross_attention_mass", ptr(small.d["q"]), ptr(kv), ptr(lse), ptr(mass), ptr(cu_q), ptr(cu_k), ptr(w), 1, lq, n, lq,
                 rows, 1, 1, dk, dk, 2 * dk, 1, s)
            exact, tol = small.exact()
            assert ((dkv[-n:].cpu().double() - exact["dkv"][:n]).abs() <= tol["dkv"][:n]).all()
            assert ((mass[:, -n:].cpu().double() - exact["mass"][:, :n]).abs() <= tol["mass"][:, :n]).all()
        else:
            assert ((ctx[:1].cpu().double() - exact["ctx"][:1]).abs() <= tol["ctx"][:1]).all()


def test_offsets_outside_the_matrices_touch_nothing():
    """cu arrays that point outside [0, M) are clamped: no row of the outputs' guard is written, nothing faults"""
    p = Problem([20, 30], [40, 50], 2, 2, 64, "bf16")
    p.cu_q = torch.tensor([-5, 30, 1000], dtype=torch.int32, device=DEV)
    p.cu_k = torch.tensor([60, 20, 1 << 30], dtype=torch.int32, device=DEV)
    p.max_q, p.max_k = 30, 50
    guard = torch.full((p.Mq + 64, p.ldq), 7.0, dtype=torch.bfloat16, device=DEV)
    ctx, lse = p.forward(ctx=guard)
    assert (guard[p.Mq:] == 7.0).all()
    dkv = torch.full((p.Mk + 64, p.ldk), 7.0, dtype=torch.bfloat16, device=DEV)
    p.backward(ctx, lse, dkv=dkv)
    assert (dkv[p.Mk:] == 7.0).all()


@pytest.mark.parametrize("lq,lk", [([70, 20], [50, 33]), ([1, 1], [3000, 40]), ([30, 50], [900, 700])])
def test_rows_in_front_of_the_first_utterance(lq, lk):
    """offsets that begin behind row 0: the rows in front of them keep their values, the others the results of a batch without them"""
    p = Problem(lq, lk, 2, 2, 64, "bf16", seed=3)
    lead = Problem([5] + lq, [7] + lk, 2, 2, 64, "bf16", seed=3)
    for name, n in (("q", 5), ("kv", 7), ("dctx", 5)):
        lead.d[name][n:] = p.d[name]
        lead.d[name][:n] = math.nan
    lead.cu_q, lead.cu_k, lead.B, lead.max_q, lead.max_k = lead.cu_q[1:].clone(), lead.cu_k[1:].clone(), 2, max(lq), max(lk)
    ctx, lse = p.forward()
    got, glse = lead.forward()
    assert torch.equal(got[5:], ctx) and torch.equal(glse[:, 5:], lse) and (got[:5] == 7.0).all() and (glse[:, :5] == 7.0).all()
    dq, dkv = p.backward(ctx, lse)
    gq, gkv = lead.backward(got, glse)
    assert torch.equal(gq[5:], dq) and torch.equal(gkv[7:], dkv) and (gq[:5] == 7.0).all() and (gkv[:7] == 7.0).all()
    m, gm = p.mass(lse), lead.mass(glse)
    assert torch.equal(gm[:, 7:], m) and (gm[:, :7] == 7.0).all()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("lq,lk,H,KV,dk", [([70, 33], [50, 90], 4, 2, 64), ([2, 1], [300, 5], 2, 1, 96)])
def test_every_matrix_has_its_own_leading_dim(lq, lk, H, KV, dk, dtype):
    """q, k, v and ctx as views of wider matrices, each of another width: the bits of the packed call"""
    p = Problem(lq, lk, H, KV, dk, dtype, seed=11)
    ctx, lse = p.forward()
    dq, dkv = p.backward(ctx, lse)
    m = p.mass(lse)
    t, nk, nv = TDT[dtype], KV * dk, 2 * KV * dk

    def wide(x, extra, left):
        w = torch.full((x.shape[0], x.shape[1] + extra), 7.0, dtype=t, device=DEV)
        v = w[:, left:left + x.shape[1]]
        v.copy_(x)
        return w, v
    bufs = [wide(x, e, l) for x, e, l in ((p.d["q"], 40, 16), (p.d["kv"][:, :nk], 8, 8), (p.d["kv"][:, nk:nv], 24, 0),
                                          (torch.full_like(ctx, 7.0), 56, 32), (p.d["dctx"], 56, 32))]
    grads = [wide(torch.full_like(b[1], 7.0), b[0].shape[1] - b[1].shape[1], l) for b, l in zip(bufs[:3], (16, 8, 0))]
    ldq, ldk, ldv, ldo = (b[0].shape[1] for b in bufs[:4])
    q, k, v, o, do = (b[1].data_ptr() for b in bufs)
    gq, gk, gv = (b[1].data_ptr() for b in grads)
    n = (p.B, p.max_q, p.max_k, p.Mq, p.Mk)
    l2 = torch.full_like(lse, 7.0)
    m2 = torch.full_like(m, 7.0)
    ws = _bytes("fs2_cross_attention_workspace", *n[:4], H, KV, dk, CODE[dtype])
    call("fs2_cross_attention", q, k, v, o, ptr(l2), ptr(p.cu_q), ptr(p.cu_k), ptr(ws), *n, H, KV, dk, ldq, ldk, ldv, ldo, CODE[dtype], 0, 0,
         0.0, stream())
    ws = _bytes("fs2_cross_attention_bwd_workspace", *n, H, KV, dk, CODE[dtype])
    call("fs2_cross_attention_bwd", q, k, v, o, do, ptr(l2), gq, gk, gv, ptr(p.cu_q), ptr(p.cu_k), ptr(ws), *n, H, KV, dk, ldq, ldk, ldv, ldo,
         CODE[dtype], 0, 0, 0.0, stream())
    ws = _bytes("fs2_cross_attention_mass_workspace", *n[:3], p.Mk, H, KV, dk, CODE[dtype])
    call("fs2_cross_attention_mass", q, k, ptr(l2), ptr(m2), ptr(p.cu_q), ptr(p.cu_k), ptr(ws), *n, H, KV, dk, ldq, ldk, CODE[dtype], stream())
    assert torch.equal(bufs[3][1], ctx) and torch.equal(l2, lse) and torch.equal(m2, m)
    assert torch.equal(grads[0][1], dq) and torch.equal(grads[1][1], dkv[:, :nk]) and torch.equal(grads[2][1], dkv[:, nk:nv])
    for (w, v_), left in zip([bufs[3]] + grads, (32, 16, 8, 0)):
        assert (w[:, :left] == 7.0).all() and (w[:, left + v_.shape[1]:] == 7.0).all()


def test_two_calls_at_once():
    """two streams, a workspace each, many calls under way together: the bits of the calls alone"""
    probs = [Problem([1, 1], [5000, 700], 2, 2, 64, "bf16", seed=1), Problem([700], [301], 4, 2, 96, "fp32", seed=2)]
    norm = Norm([300, 120], 256, 16, "tanh", "fp32", seed=3)
    want = []
    for p in probs:
        c, l = p.forward()
        want.append([c, l, *p.backward(c, l), p.mass(l)])
    ny, nst = norm.forward("bf16")
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for p, st in zip(probs, streams):
            with torch.cuda.stream(st):
                c, l = p.forward()
                got.append([c, l, *p.backward(c, l), p.mass(l), *norm.forward("bf16")])
    for st in streams:
        st.synchronize()
    for k, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, want[k % 2] + [ny, nst]))


def test_utterances_longer_than_announced_are_cut():
    """max_q, max_k below the longest: what is computed is that of the cut utterances, no other row is touched"""
    full = Problem([100, 60], [80, 30], 4, 2, 64, "bf16", seed=5)
    full.max_q, full.max_k = 60, 30
    cut = Problem([60, 60], [30, 30], 4, 2, 64, "bf16", seed=5)
    for name, c, n in (("q", full.cq, 60), ("kv", full.ck, 30), ("dctx", full.cq, 60)):
        for b in range(2):
            cut.d[name][b * n:(b + 1) * n] = full.d[name][c[b]:c[b] + n]
    ctx, lse = cut.forward()
    dq, dkv = cut.backward(ctx, lse)
    got, glse = full.forward()
    gq, gkv = full.backward(got, glse)
    m, gm = cut.mass(lse), full.mass(glse)
    for b in range(2):
        rq, sq = slice(b * 60, b * 60 + 60), slice(full.cq[b], full.cq[b] + 60)
        rk, sk = slice(b * 30, b * 30 + 30), slice(full.ck[b], full.ck[b] + 30)
        assert torch.equal(got[sq], ctx[rq]) and torch.equal(glse[:, sq], lse[:, rq]) and torch.equal(gq[sq], dq[rq])
        assert torch.equal(gkv[sk], dkv[rk]) and torch.equal(gm[:, sk], m[:, rk])
    assert (got[60:100] == 7.0).all() and (gq[60:100] == 7.0).all() and (gkv[30:80] == 7.0).all() and (gm[:, 30:80] == 7.0).all()


@pytest.mark.parametrize("H,nq,nk", [(8, 1, 3), (1, 17, 2)])
def test_as_many_utterances_as_one_call_takes(H, nq, nk):
    """65535 utterances: the last one's results, and a sum over all, against float64 on the device"""
    B, dk = 65535, 32
    g = torch.Generator(device=DEV).manual_seed(H)
    q, do = (torch.randn(B * nq, H * dk, generator=g, device=DEV) for _ in range(2))
    k, v = (torch.randn(B * nk, H * dk, generator=g, device=DEV) for _ in range(2))
    cu_q = torch.arange(B + 1, device=DEV, dtype=torch.int32) * nq
    cu_k = torch.arange(B + 1, device=DEV, dtype=torch.int32) * nk
    ctx, dq, dk_, dv = torch.empty_like(q), torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    lse, mass = torch.empty(H, B * nq, device=DEV), torch.empty(H, B * nk, device=DEV)
    ld = H * dk
    n = (B, nq, nk, B * nq, B * nk)
    ws = _bytes("fs2_cross_attention_workspace", *n[:4], H, H, dk, 0)
    call("fs2_cross_attention", ptr(q), ptr(k), ptr(v), ptr(ctx), ptr(lse), ptr(cu_q), ptr(cu_k), ptr(ws), *n, H, H, dk, ld, ld, ld, ld, 0,
         0, 0, 0.0, stream())
    ws = _bytes("fs2_cross_attention_bwd_workspace", *n, H, H, dk, 0)
    call("fs2_cross_attention_bwd", ptr(q), ptr(k), ptr(v), ptr(ctx), ptr(do), ptr(lse), ptr(dq), ptr(dk_), ptr(dv), ptr(cu_q), ptr(cu_k),
         ptr(ws), *n, H, H, dk, ld, ld, ld, ld, 0, 0, 0, 0.0, stream())
    ws = _bytes("fs2_cross_attention_mass_workspace", *n[:3], B * nk, H, H, dk, 0)
    call("fs2_cross_attention_mass", ptr(q), ptr(k), ptr(lse), ptr(mass), ptr(cu_q), ptr(cu_k), ptr(ws), *n, H, H, dk, ld, ld, 0, stream())
    Q, D = (t.double().view(B, nq, 1, H, dk) for t in (q, do))
    K, V = (t.double().view(B, 1, nk, H, dk) for t in (k, v))
    P = torch.softmax((Q * K).sum(-1) * dk ** -0.5, 2)
    O = (P[..., None] * V).sum(2)
    dS = P * ((D * V).sum(-1) - (D[:, :, 0] * O).sum(-1)[:, :, None]) * dk ** -0.5
    for got, want in ((ctx, O), (dq, (dS[..., None] * K).sum(2)), (dk_, (dS[..., None] * Q).sum(1)), (dv, (P[..., None] * D).sum(1)),
                      (mass.t(), P.sum(1))):
        got, want = got.double().reshape(B, -1), want.reshape(B, -1)
        # 2 dk fp32 operations behind an element of size ~10, at most
        assert (got - want).abs().max() <= 64 * U * 10 * 4 and (got[-1] - want[-1]).abs().max() <= 64 * U * 10 * 4


def test_mass_of_a_broken_query_is_nan():
    p = Problem([20, 9], [30, 12], 2, 2, 64, "fp32", seed=4)
    clean = p.mass(p.forward()[1])
    p.d["q"][3] = math.nan
    m = p.mass(p.forward()[1])
    assert torch.isnan(m[:, :30]).all() and torch.equal(m[:, 30:42], clean[:, 30:42])


# ---------------------------------------------------------------------------------------------------------- group norm
ACTS = {"none": lambda z: z, "relu": torch.relu, "tanh": torch.tanh, "silu": F.silu}
ACT_CODE = {"none": 0, "relu": 1, "tanh": 2, "silu": 3}
EPS = 1e-5


class Norm:
    def __init__(self, lens, C, G, act, xt, seed=0, pad=0, level=1.0):
        g = torch.Generator().manual_seed(seed + C * 13 + G + sum(lens))
        self.lens, self.C, self.G, self.act, self.xt = list(lens), C, G, act, xt
        self.M, self.B, self.ld = sum(lens) + 3, len(lens), C + pad
        self.x = (torch.randn(self.M, self.ld, generator=g) * (0.5 + torch.rand(self.ld, generator=g))
                  + level * torch.randn(self.ld, generator=g)).to(TDT[xt])
        self.x[-3:] = math.nan
        self.gamma, self.beta = 1 + 0.2 * torch.randn(C, generator=g), 0.2 * torch.randn(C, generator=g)
        self.dout = torch.randn(self.M, self.ld, generator=g) * 0.5
        self.cu = _cu(lens)
        self.xd, self.gd, self.bd = self.x.to(DEV), self.gamma.to(DEV), self.beta.to(DEV)

    def forward(self, ot, drop=(0, 0, 0.0), ws=None):
        y = torch.full((self.M, self.ld), 7.0, dtype=TDT[ot], device=DEV)
        stats = torch.full((self.B, self.G, 2), 7.0, device=DEV)
        ws = _bytes("fs2_group_norm_workspace", self.B, max(self.lens), self.C, self.G) if ws is None else ws
        call("fs2_group_norm", ptr(self.xd), ptr(self.cu), ptr(self.gd), ptr(self.bd), ptr(y), ptr(stats), ptr(ws), self.B,
             max(self.lens), self.M, self.C, self.G, self.ld, self.ld, EPS, ACT_CODE[self.act], CODE[self.xt], CODE[ot], *drop, stream())
        return y, stats

    def backward(self, stats, dt, gt, drop=(0, 0, 0.0)):
        d = self.dout.to(TDT[dt]).to(DEV)
        dx = torch.full((self.M, self.ld), 7.0, dtype=TDT[gt], device=DEV)
        dg, db = torch.full((self.C,), 7.0, device=DEV), torch.full((self.C,), 7.0, device=DEV)
        ws = _bytes("fs2_group_norm_bwd_workspace", self.B, max(self.lens), self.C, self.G)
        call("fs2_group_norm_bwd", ptr(self.xd), ptr(stats), ptr(self.cu), ptr(self.gd), ptr(self.bd), ptr(d), ptr(dx), ptr(dg), ptr(db),
             ptr(ws), self.B, max(self.lens), self.M, self.C, self.G, self.ld, self.ld, self.ld, ACT_CODE[self.act], CODE[self.xt],
             CODE[dt], CODE[gt], *drop, stream())
        return dx, dg, db

    def exact(self, dt, drop=(0, 0, 0.0)):
        """values and bounds, float64.  k = number of additions behind a sum here (rows of a thread, the two stages over the
        workgroup, channels of the group, chunks): at most 300 at these sizes.  mean: dm = k u mean|x|; centred squares: the
        error of the mean enters squared, var relative (k + 4) u + dm^2 / var; xhat: dm rstd + |xhat| (that / 2 + 4 u).
        tanh, silu and their slopes: 4e-7 absolute (times 1 + |z| for silu), and slope <= 1.1."""
        C, G, k = self.C, self.G, 300
        n = self.M - 3
        cu = [0] + list(np.cumsum(self.lens))
        x = self.x.double()[:n, :C]
        do = self.dout.to(TDT[dt]).double()[:n, :C]
        mul = drop_mul(drop[0], drop[1], n, C, drop[2]) if drop[2] else torch.ones(n, C, dtype=torch.float64)
        ga, be = self.gamma.double(), self.beta.double()
        out = dict(y=torch.zeros(n, C, dtype=torch.float64), stats=torch.zeros(self.B, G, 2, dtype=torch.float64),
                   dx=torch.zeros(n, C, dtype=torch.float64), dgamma=torch.zeros(C, dtype=torch.float64),
                   dbeta=torch.zeros(C, dtype=torch.float64))
        tol = {key: torch.zeros_like(v) for key, v in out.items()}
        for b in range(self.B):
            r = slice(cu[b], cu[b + 1])
            L = cu[b + 1] - cu[b]
            if L == 0:
                out["stats"][b, :, 1] = EPS ** -0.5
                tol["stats"][b, :, 1] = 4 * U * EPS ** -0.5
                continue
            w = x[r].view(L, G, C // G)
            mean = w.mean((0, 2), keepdim=True)
            var = ((w - mean) ** 2).mean((0, 2), keepdim=True)
            rstd = (var + EPS) ** -0.5
            dm = k * U * w.abs().mean((0, 2), keepdim=True)
            rv = ((k + 4) * U * var + dm ** 2) / (var + EPS)
            xh = ((w - mean) * rstd)
            ex = (dm * rstd + U * w.abs() * rstd + xh.abs() * (rv / 2 + 4 * U)).reshape(L, C)
            out["stats"][b, :, 0], out["stats"][b, :, 1] = mean.flatten(), rstd.flatten()
            tol["stats"][b, :, 0], tol["stats"][b, :, 1] = dm.flatten() + U * mean.abs().flatten(), (rstd * (rv / 2 + 4 * U)).flatten()
            xh, rs = xh.reshape(L, C), rstd.expand(1, G, C // G).reshape(1, C)
            z = (xh * ga + be).requires_grad_(True)
            ez = (ga.abs() * ex + 3 * U * (xh.abs() * ga.abs() + be.abs())).detach()
            y = ACTS[self.act](z)
            slope, = torch.autograd.grad(y.sum(), z)
            y, z = y.detach(), z.detach()
            extra = 0.0 if self.act in ("none", "relu") else 4e-7 * (1 + z.abs())
            out["y"][r] = y * mul[r]
            tol["y"][r] = (1.1 * ez + extra) * mul[r] + 2 * U * y.abs() * mul[r]
            es = 0.0 if self.act in ("none", "relu") else ez + extra
            u = do[r] * mul[r]
            dz = u * slope
            edz = u.abs() * es + 3 * U * dz.abs()
            dh, edh = dz * ga, edz * ga.abs() + U * (dz * ga).abs()

            def mean_of(v):
                return v.view(L, G, C // G).mean((0, 2), keepdim=True).expand(1, G, C // G).reshape(1, C)
            m1, m2 = mean_of(dh), mean_of(dh * xh)
            e1 = mean_of(edh) + k * U * mean_of(dh.abs())
            e2 = mean_of(edh * xh.abs() + dh.abs() * ex) + k * U * mean_of((dh * xh).abs())
            body = dh - m1 - xh * m2
            out["dx"][r] = rs * body
            rr = mean_of((rv / 2 + 4 * U).expand(L, G, C // G))
            tol["dx"][r] = rs * (edh + e1 + ex * m2.abs() + xh.abs() * e2 + 6 * U * (dh.abs() + m1.abs() + (xh * m2).abs())) + rr * (rs * body).abs()
            out["dgamma"] += (dz * xh).sum(0)
            out["dbeta"] += dz.sum(0)
            tol["dgamma"] += (edz * xh.abs() + dz.abs() * ex + k * U * (dz * xh).abs()).sum(0)
            tol["dbeta"] += (edz + k * U * dz.abs()).sum(0)
        return out, tol


NORMS = [
    # lens, C, G, act
    ([1], 8, 8, "none"),                                 # one row, one channel to a group: xhat = 0
    ([1, 2, 5], 80, 16, "tanh"),                         # groups of five channels
    ([130, 0, 64, 7], 256, 16, "tanh"),                  # an utterance without rows
    ([33, 300], 256, 1, "silu"),                         # one group of all channels
    ([200, 150], 384, 32, "relu"),                       # twelve channels
    ([700, 10], 96, 4, "silu"),
    ([900], 80, 2, "none"),
    ([2100, 40], 64, 4, "tanh"),                         # chunks for the backward
    ([9000, 3], 40, 8, "silu"),                          # chunks both ways
    ([40, 3], 1024, 2, "none"),
    ([70], 1024, 1024, "tanh"),
    ([180, 0] + [3] * 254, 256, 1, "tanh"),              # 256 workgroups of up to 16 rows a thread, both ways and types
]


def _half(t, want, tol):
    return tol + HALF[t] * (want.abs() + tol)


@pytest.mark.parametrize("xt,ot,dt,gt", [("fp32", "fp32", "fp32", "fp32"), ("fp32", "bf16", "fp32", "bf16"),
                                         ("bf16", "bf16", "bf16", "bf16"), ("bf16", "fp32", "fp32", "bf16"),
                                         ("fp32", "fp32", "bf16", "fp32")])
@pytest.mark.parametrize("lens,C,G,act", NORMS)
def test_group_norm(lens, C, G, act, xt, ot, dt, gt):
    p = Norm(lens, C, G, act, xt, pad=8)
    want, tol = p.exact(dt)
    y, stats = p.forward(ot)
    n = sum(lens)
    _near(y, want["y"], _half(ot, want["y"], tol["y"]), n, "y")
    off = (stats.cpu().double() - want["stats"]).abs()
    assert (off <= tol["stats"]).all(), float((off - tol["stats"]).max())
    if act == "relu":                # the kink: no gradient where the sign of z is not certain
        xh = ((p.x.double()[:n, :C].view(n, G, -1) - 0) * 1)
        b = torch.bucketize(torch.arange(n), torch.tensor(np.cumsum(lens)), right=True)
        xh = (xh - want["stats"][b, :, :1]) * want["stats"][b, :, 1:]
        z = xh.reshape(n, C) * p.gamma.double() + p.beta.double()
        p.dout[:n, :C][z.abs() < 1e-3] = 0
        want, tol = p.exact(dt)
    dx, dg, db = p.backward(stats, dt, gt)
    _near(dx, want["dx"], _half(gt, want["dx"], tol["dx"]), n, "dx")
    for name, got in (("dgamma", dg), ("dbeta", db)):
        off = (got.cpu().double() - want[name]).abs()
        assert (off <= tol[name] + HALF["fp32"] * want[name].abs() + 1e-30).all(), (name, float((off / (tol[name] + 1e-30)).max()))
    again = p.backward(stats, dt, gt)
    assert all(torch.equal(u, v) for u, v in zip(again, (dx, dg, db)))


def test_group_norm_far_from_zero():
    """levels a thousand times the spread: the centred squares lose nothing that the inputs hold"""
    p = Norm([500, 3000], 64, 4, "none", "fp32", level=0.0)
    p.x[:, :] += 1000.0
    p.xd = p.x.to(DEV)
    want, tol = p.exact("fp32")
    y, stats = p.forward("fp32")
    _near(y, want["y"], _half("fp32", want["y"], tol["y"]), 3500, "y")
    assert ((stats.cpu().double() - want["stats"]).abs() <= tol["stats"]).all()


def test_group_norm_dropout_and_differences():
    drop = (77, 5, 0.5)
    p = Norm([60, 21], 80, 16, "tanh", "fp32")
    want, tol = p.exact("fp32", drop)
    y, stats = p.forward("fp32", drop)
    _near(y, want["y"], _half("fp32", want["y"], tol["y"]), 81, "y")
    dx, dg, db = p.backward(stats, "fp32", "fp32", drop)
    _near(dx, want["dx"], _half("fp32", want["dx"], tol["dx"]), 81, "dx")
    # central difference of <y, dout> along a direction, step 1/128: noise 1e-6 / step, curvature step^2
    g = torch.Generator().manual_seed(3)
    u = torch.randn(p.M, p.ld, generator=g)
    u[-3:] = 0
    base, step, vals = p.xd.clone(), 1.0 / 128, []
    for sgn in (1, -1):
        p.xd = base + sgn * step * u.to(DEV)
        vals.append(float((p.forward("fp32", drop)[0][:81].cpu().double() * p.dout[:81].double()).sum()))
    got = float((dx[:81].cpu().double() * u[:81].double()).sum())
    assert abs((vals[0] - vals[1]) / (2 * step) - got) <= 5e-3 * max(abs(got), float(dx[:81].double().norm()))


# ------------------------------------------------------------------------------------------- streams, graphs, together
def test_other_stream_and_two_graphs():
    """calls on a side stream; two captured graphs with a workspace each, replayed in turn with eager work between"""
    probs = [Problem([1, 1], [1800, 700], 2, 2, 64, "bf16", seed=1), Problem([150, 40], [33, 200], 4, 2, 64, "bf16", seed=2)]
    want = []
    for p in probs:
        c, l = p.forward()
        want.append([c, l, *p.backward(c, l), p.mass(l)])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c, l = probs[0].forward()
        got = [c, l, *probs[0].backward(c, l), probs[0].mass(l)]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    graphs = []
    for p in probs:
        args = (p.B, p.max_q, p.max_k)
        ws = [_bytes("fs2_cross_attention_workspace", *args, p.Mq, p.H, p.KV, p.dk, 1),
              _bytes("fs2_cross_attention_bwd_workspace", *args, p.Mq, p.Mk, p.H, p.KV, p.dk, 1),
              _bytes("fs2_cross_attention_mass_workspace", *args, p.Mk, p.H, p.KV, p.dk, 1)]
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            c, l = p.forward(ws=ws[0])
            dq, dkv = p.backward(c, l, ws=ws[1])
            m = p.mass(l, ws=ws[2])
        graphs.append((gr, [c, l, dq, dkv, m], ws))
    for _ in range(3):
        for (gr, outs, _), w, p in zip(graphs, want, probs):
            for o in outs:
                o.fill_(7.0)
            gr.replay()
            p.forward()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, w))


@pytest.mark.parametrize("lens", [[70, 0, 33], [9000, 20]])
def test_group_norm_in_a_graph(lens):
    """the forms that hold an utterance and that cut it into chunks: captured, replayed with eager calls between; rows in front of the
    first utterance and behind an announced length keep their values"""
    p = Norm(lens, 64, 4, "silu", "bf16", seed=2)
    p.dout = p.dout.to(DEV)                      # (no copy from the host while capturing)
    drop = (5, 6, 0.1)
    y, st = p.forward("bf16", drop)
    want = [y, st, *p.backward(st, "bf16", "bf16", drop)]
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        y, st = p.forward("bf16", drop)
        out = [y, st, *p.backward(st, "bf16", "bf16", drop)]
    for _ in range(3):
        for o in out:
            o.fill_(3.0)
        gr.replay()
        p.forward("bf16")
        torch.cuda.synchronize()
        for got, w in zip(out, want):
            assert torch.equal(got[:sum(lens)], w[:sum(lens)]) if got.shape[0] == p.M else torch.equal(got, w)


def test_group_norm_rows_of_nobody():
    """offsets that begin behind row 0 and an utterance longer than announced"""
    p = Norm([50, 40], 96, 4, "tanh", "fp32", seed=1)
    cut = Norm([40, 40], 96, 4, "tanh", "fp32", seed=1)
    p.xd = torch.cat([torch.full((4, p.ld), math.nan, device=DEV), p.xd])
    p.dout = torch.cat([torch.full((4, p.ld), math.nan), p.dout])
    cut.gd, cut.bd = p.gd, p.bd
    cut.xd[:40], cut.xd[40:80] = p.xd[4:44], p.xd[54:94]
    cut.dout[:40], cut.dout[40:80] = p.dout[4:44], p.dout[54:94]
    p.cu, p.M, p.lens = p.cu + 4, p.M + 4, [40, 40]
    y, st = p.forward("fp32")
    w, wst = cut.forward("fp32")
    assert torch.equal(st, wst) and torch.equal(y[4:44], w[:40]) and torch.equal(y[54:94], w[40:80])
    dx, dg, db = p.backward(st, "fp32", "fp32")
    wx, wg, wb = cut.backward(wst, "fp32", "fp32")
    assert torch.equal(dg, wg) and torch.equal(db, wb) and torch.equal(dx[4:44], wx[:40]) and torch.equal(dx[54:94], wx[40:80])
    for t in (y, dx):
        assert (t[:4] == 7.0).all() and (t[44:54] == 7.0).all() and (t[94:] == 7.0).all()


def test_aligner_step_end_to_end():
    """What they are for, in one chain on packed rows: conv outputs of frames -> group norm + tanh -> queries of a cross
    attention to phone states -> loss, its backward through both; then the attention mass as durations for the length
    regulator.  Against autograd in float64 over the same (fp32) data."""
    lq, lk, C, G, H, dk = [57, 120, 33], [9, 21, 5], 128, 16, 2, 64
    n = Norm(lq, C, G, "tanh", "fp32", seed=8)
    y, stats = n.forward("fp32")
    p = Problem(lq, lk, H, H, dk, "fp32", seed=8)
    p.d["q"] = y
    ctx, lse = p.forward()
    dq, dkv = p.backward(ctx, lse)
    n.dout = dq.cpu()
    dx, dg, db = n.backward(stats, "fp32", "fp32")
    mass = p.mass(lse)
    # float64
    x = n.x[:sum(lq)].double().requires_grad_(True)
    kv = p.kv[:sum(lk)].double().requires_grad_(True)
    ga = n.gamma.double().requires_grad_(True)
    loss, masses = 0.0, []
    for b in range(3):
        rq, rk = slice(p.cq[b], p.cq[b + 1]), slice(p.ck[b], p.ck[b + 1])
        yy = torch.tanh(F.group_norm(x[rq].t()[None], G, ga, n.beta.double(), EPS))[0].t()
        for h in range(H):
            c, v = slice(h * dk, (h + 1) * dk), slice((H + h) * dk, (H + h + 1) * dk)
            P = torch.softmax(yy[:, c] @ kv[rk, c].T / math.sqrt(dk), 1)
            loss = loss + ((P @ kv[rk, v]) * p.dctx[rq, c].double()).sum()
            masses.append(P.sum(0).detach())
    loss.backward()
    for got, want in ((dx[:sum(lq)], x.grad), (dkv[:sum(lk)], kv.grad), (dg, ga.grad)):
        assert (got.cpu().double() - want).norm() <= 3e-6 * want.norm()
    total = mass[:, :sum(lk)].cpu().double()
    for b in range(3):
        rk = slice(p.ck[b], p.ck[b + 1])
        for h in range(H):
            assert (total[h, rk] - masses[b * H + h]).abs().max() <= 1e-4
            assert abs(float(total[h, rk].sum()) - lq[b]) <= 1e-3
    # durations of the first head through the framework's own length regulator
    dur = mass[0, :sum(lk)].round().to(torch.int32).contiguous()
    used, cum = torch.empty_like(dur), torch.empty_like(dur)
    olens, cu_f = torch.empty(3, dtype=torch.int32, device=DEV), torch.empty(4, dtype=torch.int32, device=DEV)
    call("fs2_lr_plan", ptr(dur), ptr(p.cu_k), 1.0, ptr(used), ptr(cum), ptr(olens), ptr(cu_f), 3, stream())
    assert all(abs(int(o) - q) <= k / 2 + 1 for o, q, k in zip(olens.tolist(), lq, lk))
