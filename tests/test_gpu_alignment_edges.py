"""-m gpu: the alignment operators where they are easily wrong: roundings beyond that of the result, infinities next to a tile's end,
sides without rows, long chunked utterances.  Bounds are counted as in test_gpu_alignment.py: u = 2^-24 per fp32 operation,
h = half a step of the output's type."""
import math

import numpy as np
import pytest
import torch

from fastspeech2_amd import hip
from fastspeech2_amd.hip import call, ptr, stream
from tests import test_gpu_alignment as base
from tests.test_gpu_alignment import ACT_CODE, CODE, DEV, EPS, HALF, LOG2E, TDT, U, Norm, Problem, _bytes, _cu, _half, _near
from tests.test_gpu_dropout import drop_mul

pytestmark = pytest.mark.gpu


def _weights_and_bounds(p, drop):
    """(utterance, head, rows, keys, dropped probabilities, relative error of one) in float64, the error as fp32 arithmetic makes it:
    scores dS = (dk + 4) u sum|q||k| / sqrt(dk), exp2 and its argument, the sum of n terms (Problem.exact), and 2^-15 for a probability
    held as the sum of two bf16 numbers (the first off by less than 2^-7 of it, what is left rounded to half a step)"""
    q, kv = p.q.double(), p.kv.double()
    s = p.dk ** -0.5
    for b, h, rq, rk, hc, kc, vc in p.pairs():
        n, nq = rk.stop - rk.start, rq.stop - rq.start
        if n == 0 or nq == 0:
            continue
        Q, K = q[rq, hc], kv[rk, kc]
        S = Q @ K.T * s
        dS = (p.dk + 4) * U * (Q.abs() @ K.abs().T) * s
        rP = dS + dS.max(1, keepdim=True).values + (2 * n + 16) * U + 4 * U * LOG2E * S.abs().max(1, keepdim=True).values
        P = torch.softmax(S, 1)
        if drop[2]:
            P = P * drop_mul(drop[0], drop[1] + h, nq, n, drop[2], rq.start)
        lse = torch.logsumexp(S, 1, keepdim=True).abs() * LOG2E
        yield rq, rk, hc, vc, P, rP + (n + 2) * U + 2.0 ** -15, rP + 8 * U * (1 + lse) + 2.0 ** -15, nq


@pytest.mark.parametrize("lq,lk,H,KV,dk,drop", [
    ([200, 33], [120, 70], 2, 2, 128, 0.0),          # many rows
    ([300, 64], [65, 200], 4, 2, 64, 0.1),
    ([40], [900], 2, 2, 64, 0.0),                    # keys over several workgroups
    ([1, 1, 2], [120, 33, 700], 4, 1, 96, 0.0),      # few rows
    ([1], [1500], 2, 2, 32, 0.1),                    # ... over several workgroups
])
def test_bf16_results_are_rounded_once(lq, lk, H, KV, dk, drop):
    """ctx and dv in bf16 are off by half a step of the RESULT and fp32 errors: the probabilities lose nothing on the way to the
    matrix pipe (an element whose terms cancel shows it: rounding them to 2^-8 moves it by far more than its own half step)"""
    p = Problem(lq, lk, H, KV, dk, "bf16", seed=21)
    drop = (99, 3, drop)
    ctx, lse = p.forward(drop)
    _, dkv = p.backward(ctx, lse, drop)
    V, D = p.kv.double(), p.dctx.double()
    want, tol = torch.zeros(p.Mq, H * dk, dtype=torch.float64), torch.zeros(p.Mq, H * dk, dtype=torch.float64)
    wv, tv = torch.zeros(p.Mk, KV * dk, dtype=torch.float64), torch.zeros(p.Mk, KV * dk, dtype=torch.float64)
    for rq, rk, hc, vc, P, r, rb, nq in _weights_and_bounds(p, drop):
        O = P @ V[rk, vc]
        e = (P * r) @ V[rk, vc].abs() + 2 * U * O.abs()
        want[rq, hc], tol[rq, hc] = O, e + HALF["bf16"] * (O.abs() + e)
        out = slice(vc.start - KV * dk, vc.stop - KV * dk)
        wv[rk, out] += P.T @ D[rq, hc]
        tv[rk, out] += (P * (rb + (H // KV * nq + 40) * U)).T @ D[rq, hc].abs()
    tv += HALF["bf16"] * (wv.abs() + tv)
    _near(ctx, want, tol, sum(lq), "ctx")
    _near(dkv[:, KV * dk:].contiguous(), wv, tv, sum(lk), "dv")


@pytest.mark.parametrize("drop", [0.0, 0.2])
@pytest.mark.parametrize("lq,lk,H,KV,dk", [
    ([100, 33], [2, 1], 2, 2, 64), ([70, 7], [8, 31], 4, 2, 32), ([1, 1, 40], [5, 32, 17], 4, 1, 128), ([300], [16], 2, 2, 96),
    ([100, 65], [33, 64], 2, 2, 64), ([40, 1], [50, 61], 4, 2, 128)])
def test_bf16_score_gradients_of_few_keys_are_rounded_once(lq, lk, H, KV, dk, drop):
    """up to 64 keys dq, up to 32 dk as well take delta = sum P dP from what is at hand and not from the rounded ctx, whose rounding weighs
    most where few keys share it.  dP: (dk + 2) u sum|dO||V|; delta: that and P's own error, n u of its terms; dS = P (dP - delta) held to
    2^-16 by two numbers; then half a step of the result"""
    p = Problem(lq, lk, H, KV, dk, "bf16", seed=23)
    drop = (77, 4, drop)
    ctx, lse = p.forward(drop)
    dq, dkv = p.backward(ctx, lse, drop)
    q, kv, do, s = p.q.double(), p.kv.double(), p.dctx.double(), dk ** -0.5
    wq, tq = torch.zeros(p.Mq, H * dk, dtype=torch.float64), torch.zeros(p.Mq, H * dk, dtype=torch.float64)
    wk, tk = torch.zeros(p.Mk, KV * dk, dtype=torch.float64), torch.zeros(p.Mk, KV * dk, dtype=torch.float64)
    for b, h, rq, rk, hc, kc, vc in p.pairs():
        n, nq = rk.stop - rk.start, rq.stop - rq.start
        Q, K, V, D = q[rq, hc], kv[rk, kc], kv[rk, vc], do[rq, hc]
        S = Q @ K.T * s
        P = torch.softmax(S, 1)
        M = drop_mul(drop[0], drop[1] + h, nq, n, drop[2], rq.start) if drop[2] else torch.ones_like(P)
        dS = (dk + 4) * U * (Q.abs() @ K.abs().T) * s
        rP = dS + dS.max(1, keepdim=True).values + (2 * n + 16) * U + 4 * U * LOG2E * S.abs().max(1, keepdim=True).values
        rP = rP + 8 * U * (1 + torch.logsumexp(S, 1, keepdim=True).abs() * LOG2E)
        dP = (D @ V.T) * M
        eP = (dk + 2) * U * (D.abs() @ V.abs().T) * M + 2 * U * dP.abs()
        delta = (P * dP).sum(1, keepdim=True)
        eD = (P * (eP + (rP + (n + 2) * U) * dP.abs())).sum(1, keepdim=True)
        G = P * (dP - delta)
        eG = rP * G.abs() + P * (eP + eD + 4 * U * (dP.abs() + delta.abs())) + 2.0 ** -16 * G.abs()
        wq[rq, hc] = G @ K * s
        tq[rq, hc] = (eG + (n + 2) * U * G.abs()) @ K.abs() * s
        wk[rk, kc] += G.T @ Q * s
        tk[rk, kc] += (eG + (H // KV * nq + 40) * U * G.abs()).T @ Q.abs() * s
    tq += HALF["bf16"] * (wq.abs() + tq)
    tk += HALF["bf16"] * (wk.abs() + tk)
    _near(dq, wq, tq, sum(lq), "dq")
    if max(lk) <= 32:
        _near(dkv[:, :KV * dk].contiguous(), wk, tk, sum(lk), "dk")


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("lq,H,KV", [([70, 3, 129], 4, 2), ([1, 1], 2, 2)])
def test_a_batch_without_keys(lq, H, KV, dtype):
    """ctx = 0, lse = -inf, dq = 0, with no key matrix and the 16 bytes of workspace that the query asks for"""
    p = Problem(lq, [0] * len(lq), H, KV, 64, dtype, seed=5)
    assert p.max_k == 0
    n = int(hip.load().fs2_cross_attention_bwd_workspace(p.B, p.max_q, 0, p.Mq, p.Mk, H, KV, 64, CODE[dtype]))
    ws = torch.full((n,), 0xFF, dtype=torch.uint8, device=DEV)
    rows = sum(lq)
    ctx, lse = p.forward()
    assert (ctx[:rows, :H * 64] == 0).all() and (ctx[rows:] == 7).all()
    assert (lse[:, :rows] == -math.inf).all() and (lse[:, rows:] == 7).all()
    dq, dkv = p.backward(ctx, lse, ws=ws)
    assert (dq[:rows, :H * 64] == 0).all() and (dq[rows:] == 7).all() and (dkv == 7).all()
    assert (p.mass(lse) == 7).all()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("lk", [[90, 5, 33], [700]])
def test_a_batch_without_queries(lk, dtype):
    """dk = dv = 0 and no key receives anything; nothing of the query side is touched"""
    p = Problem([0] * len(lk), lk, 4, 2, 64, dtype, seed=6)
    assert p.max_q == 0
    ctx, lse = p.forward()
    assert (ctx == 7).all() and (lse == 7).all()
    dq, dkv = p.backward(ctx, lse)
    rows = sum(lk)
    assert (dq == 7).all() and (dkv[:rows, :256] == 0).all() and (dkv[rows:] == 7).all()
    m = p.mass(lse)
    assert (m[:, :rows] == 0).all() and (m[:, rows:] == 7).all()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("lq,H,KV", [(40, 2, 2), (33, 4, 2), (1, 2, 2), (64, 2, 1)])
@pytest.mark.parametrize("lk", [1, 31, 32, 33, 63, 64, 65, 120])
def test_an_infinite_last_value_row(lk, lq, H, KV, dtype):
    """an infinite element of the last value row is infinite in its column of ctx, whether or not a tile ends there (fp32: NaN, as
    announced), and nothing else changes a bit"""
    p = Problem([lq, 7], [lk, 20], H, KV, 64, dtype, seed=8)
    clean = p.forward()[0][:lq + 7].float()
    col = KV * 64 + 3                                      # element 3 of shared head 0
    p.d["kv"][p.ck[1] - 1, col] = -math.inf
    got = p.forward()[0][:lq + 7].float()
    hit = [h * 64 + 3 for h in range(H // KV)]             # the query heads that read it
    want = clean.clone()
    want[:lq, hit] = math.nan if dtype == "fp32" else -math.inf
    assert torch.equal(torch.nan_to_num(got, nan=5.0, neginf=-9.0), torch.nan_to_num(want, nan=5.0, neginf=-9.0))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("lq", [1, 31, 32, 33, 64, 100, 250])
@pytest.mark.parametrize("H,KV", [(2, 2), (2, 1)])
def test_an_infinite_last_gradient_row(H, KV, lq, dtype):
    """an infinite element of the last row of dctx in the same way in dv (dq of that row and dk are no numbers, dP - delta being none)"""
    p = Problem([lq, 9], [50, 20], H, KV, 64, dtype, seed=9)
    ctx, lse = p.forward()
    clean = p.backward(ctx, lse)[1].float()
    p.d["dctx"][lq - 1, (H - 1) * 64 + 5] = math.inf       # the last head's: the last of the packed rows
    dq, got = p.backward(ctx, lse)
    got, v = got.float(), slice(KV * 64, 2 * KV * 64)
    want = clean[:, v].clone()
    want[:50, (KV - 1) * 64 + 5] = math.nan if dtype == "fp32" else math.inf
    rows = 70
    assert torch.equal(torch.nan_to_num(got[:rows, v], nan=5.0, posinf=9.0), torch.nan_to_num(want[:rows], nan=5.0, posinf=9.0))
    assert torch.equal(got[50:rows], clean[50:rows])       # the other utterance


@pytest.mark.parametrize("lq", [1, 20])                    # the few-rows and the rows kernel
def test_fp32_scores_are_products_of_fp32(lq):
    """one key and one element of q and k other than zero: lse = x y log2(e) / 8 shows a single product.  It may be off by 2^-24 of the
    six products' missing terms, by two roundings of the matrix pipe's sum (one, or a truncation), by those of log2(e), of its
    multiplication and of the last addition: 6.1 * 2^-24.  Significands whose lower half is all ones, where planes that are cut off
    leave 2^-21, and random ones."""
    B, dk = 64, 64
    p = Problem([lq] * B, [1] * B, 1, 1, dk, "fp32")
    rng = np.random.default_rng(5)

    def some(n):
        bits = (0x42000000 + (rng.integers(0, 16, n).astype(np.uint32) << 16) + 0xFFFF)
        x = bits.astype(np.uint32).view(np.float32)
        other = (32 * (1 + rng.random(n))).astype(np.float32)
        return torch.from_numpy(np.where(rng.random(n) < 0.5, x, other).astype(np.float32))
    x, y = some(B * lq), some(B)
    p.d["q"].zero_()
    p.d["kv"].zero_()
    p.d["q"][:B * lq, 7] = x.to(DEV)
    p.d["kv"][:B, 7] = y.to(DEV)
    lse = p.forward()[1][0, :B * lq].cpu().double()
    want = x.double() * y.double().repeat_interleave(lq) * LOG2E / 8
    assert float(((lse - want).abs() / want).max()) <= 6.1 * U


def test_fp32_values_pass_whole():
    """weights of exactly one: ctx is v, bit by bit, up to the largest fp32 numbers (beyond bf16's) and down to small ones"""
    top = torch.finfo(torch.float32).max
    v = torch.tensor([top, -top, 3.3895e38, 3.396e38, -3.397e38, 1e-30, -1e-28, 0.0, 1 / 3, 65535.0 / 65536, 2 - 2 ** -23])
    for lq in (1, 40):
        p = Problem([lq], [1], 1, 1, 32, "fp32")
        p.d["q"].zero_()
        p.d["kv"][0, 32:32 + v.numel()] = v.to(DEV)
        ctx = p.forward()[0][:lq, :v.numel()].cpu()
        assert torch.equal(ctx, v.expand(lq, -1))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("lq,lk,H,KV", [([1], [5000], 2, 2), ([3, 1], [1900, 0], 4, 2), ([40, 7], [900, 30], 2, 2), ([700, 64], [33, 40], 4, 1)])
def test_workspaces_hold_what_their_queries_say(lq, lk, H, KV, dtype):
    """few utterances in the middle of large matrices: the bits of the call on matrices of their own, nothing behind a workspace written"""
    p = Problem(lq, lk, H, KV, 64, dtype, seed=12)
    want = p.forward()
    want = [*want, *p.backward(*want), p.mass(want[1])]
    front, behind = 3000, 2000
    big = Problem(lq, lk, H, KV, 64, dtype, seed=12)
    for name, n in (("q", front), ("kv", front), ("dctx", front)):
        t = big.d[name]
        big.d[name] = torch.cat([torch.full((n, t.shape[1]), math.nan, dtype=t.dtype, device=DEV), t,
                                 torch.full((behind, t.shape[1]), math.nan, dtype=t.dtype, device=DEV)])
    big.cu_q, big.cu_k = big.cu_q + front, big.cu_k + front
    big.Mq, big.Mk = big.Mq + front + behind, big.Mk + front + behind

    def guarded(name, *args):
        n = int(getattr(hip.load(), name)(*args))
        return torch.full((n + 4096,), 0xAB, dtype=torch.uint8, device=DEV), n
    n = (p.B, p.max_q, p.max_k)
    ws = [guarded("fs2_cross_attention_workspace", *n, big.Mq, H, KV, 64, CODE[dtype]),
          guarded("fs2_cross_attention_bwd_workspace", *n, big.Mq, big.Mk, H, KV, 64, CODE[dtype]),
          guarded("fs2_cross_attention_mass_workspace", *n, big.Mk, H, KV, 64, CODE[dtype])]
    ctx, lse = big.forward(ws=ws[0][0])
    dq, dkv = big.backward(ctx, lse, ws=ws[1][0])
    m = big.mass(lse, ws=ws[2][0])
    rq, rk = slice(front, front + sum(lq)), slice(front, front + sum(lk))
    for got, w, rows in ((ctx, want[0], rq), (dq, want[2], rq), (dkv, want[3], rk)):
        assert torch.equal(got[rows], w[:rows.stop - rows.start])
        assert (got[:rows.start] == 7).all() and (got[rows.stop:] == 7).all()
    for got, w, rows in ((lse, want[1], rq), (m, want[4], rk)):
        assert torch.equal(got[:, rows], w[:, :rows.stop - rows.start])
    assert all((t[k:] == 0xAB).all() for t, k in ws)


@pytest.mark.parametrize("nq", [1, 17])
def test_as_many_heads_of_utterances_as_one_call_takes(nq):
    """B * n_heads = 2^19: every result against float64.  2 dk fp32 operations behind an element of size ~10, at most"""
    B, H, nk, dk = 32768, 16, 2, 32
    g = torch.Generator(device=DEV).manual_seed(nq)
    q = torch.randn(B * nq, H * dk, generator=g, device=DEV)
    k, v = (torch.randn(B * nk, H * dk, generator=g, device=DEV) for _ in range(2))
    cu_q, cu_k = (torch.arange(B + 1, device=DEV, dtype=torch.int32) * n for n in (nq, nk))
    ctx, lse, mass = torch.empty_like(q), torch.empty(H, B * nq, device=DEV), torch.empty(H, B * nk, device=DEV)
    ld, n = H * dk, (B, nq, nk, B * nq, B * nk)
    call("fs2_cross_attention", ptr(q), ptr(k), ptr(v), ptr(ctx), ptr(lse), ptr(cu_q), ptr(cu_k), None, *n, H, H, dk, ld, ld, ld, ld, 0, 0, 0,
         0.0, stream())
    call("fs2_cross_attention_mass", ptr(q), ptr(k), ptr(lse), ptr(mass), ptr(cu_q), ptr(cu_k), None, *n, H, H, dk, ld, ld, 0, stream())
    Q, K, V = q.double().view(B, nq, H, dk), k.double().view(B, nk, H, dk), v.double().view(B, nk, H, dk)
    S = torch.stack([(Q * K[:, j, None]).sum(-1) * dk ** -0.5 for j in range(nk)], -1)           # [B, nq, H, nk]
    P = torch.softmax(S, -1)
    O = sum(P[..., j, None] * V[:, j, None] for j in range(nk))
    assert (ctx.double().view(B, nq, H, dk) - O).abs().max() <= 64 * U * 10 * 4
    assert (mass.double().view(H, B, nk) - P.sum(1).permute(1, 0, 2)).abs().max() <= 64 * U * 10 * 4


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("lq,lk", [([57, 120, 33], [9, 21, 5]), ([1, 800, 13, 7], [3, 120, 1, 40])])
def test_durations_of_the_mass_fill_the_frames(lq, lk, dtype):
    """from the mass to the length regulator: durations are differences of the rounded running sum, so every utterance gets its frames back, every phone within one frame of
    its mass (rounding both ends of its span)"""
    p = Problem(lq, lk, 2, 2, 64, dtype, seed=13)
    mass, cu_p, B = p.mass(p.forward()[1]), p.cu_k, len(lq)
    lens = (cu_p[1:] - cu_p[:-1]).long()
    run = torch.cat([mass.new_zeros(1, dtype=torch.float64), mass[:, :cu_p[-1]].double().mean(0).cumsum(0)])
    start = run[cu_p[:-1].long()].repeat_interleave(lens)
    dur = ((run[1:] - start).round() - (run[:-1] - start).round()).int()
    used, cum = torch.empty_like(dur), torch.empty_like(dur)
    olens, cu_f = torch.empty(B, dtype=torch.int32, device=DEV), torch.empty(B + 1, dtype=torch.int32, device=DEV)
    call("fs2_lr_plan", ptr(dur), ptr(cu_p), 1.0, ptr(used), ptr(cum), ptr(olens), ptr(cu_f), B, stream())
    assert olens.tolist() == lq and torch.equal(used, dur) and (dur >= 0).all()
    assert (dur - mass[:, :sum(lk)].double().mean(0)).abs().max() <= 1 + 1e-3


# ---------------------------------------------------------------------------------------------------------- group norm
@pytest.mark.parametrize("act,xt", [("tanh", "fp32"), ("tanh", "bf16"), ("silu", "fp32"), ("silu", "bf16")])
def test_activations_and_slopes_are_fp32(act, xt):
    """gamma = 0: y is the activation of beta and, with one row and dout = 1, dbeta its slope.  u = 2^-24; exp2 and the reciprocal are
    good to one unit of the last place, 2 u.  tanh = z P / Q: 2 u for the reciprocal, 5 u for the fit and the other operations (an
    evaluation of the quotient in fp32, rounded each time, is off by 6.6 u at worst with its reciprocal one unit off).  Its slope
    4 e / (1 + e)^2 with e = exp(-2|z|) off by (2.5 |z| + 2) u: (4 |z| + 10) u.  Sigmoid of either sign 8 u, so silu 9 u; its slope
    s (1 + z s') 12 u of s (1 + |z| s')."""
    rng = np.random.default_rng(7)
    C = 1024
    z = np.concatenate([rng.standard_normal(400) * 2, np.exp(rng.uniform(-12, 4.3, 616)) * rng.choice([-1, 1], 616),
                        [0.0, 8.0, -8.000001, 0.0625, 7.99999, 1e-30, -80.0, 60.0]]).astype(np.float32)
    if act == "tanh":
        z = np.clip(z, -40, 40)
    p = Norm([1], C, 4, act, xt)
    p.gd.zero_()
    p.bd = torch.from_numpy(z).to(DEV)
    p.dout = torch.ones(p.M, p.ld)
    y, stats = p.forward("fp32")
    _, _, slope = p.backward(stats, "fp32", "fp32")
    Z = torch.from_numpy(z).double()
    if act == "tanh":
        want, ws = torch.tanh(Z), torch.cosh(Z) ** -2
        ty, ts = 7 * U * want.abs(), (4 * Z.abs() + 10) * U * ws
    else:
        g, h = torch.sigmoid(Z), torch.sigmoid(-Z)
        want, ws = Z * g, g * (1 + Z * h)
        ty, ts = 9 * U * want.abs(), 12 * U * g * (1 + Z.abs() * h)
    off, offs = (y[0, :C].cpu().double() - want).abs(), (slope.cpu().double() - ws).abs()
    assert (off <= ty + 1e-37).all(), ("value", float((off / (ty + 1e-37)).max()))
    assert (offs <= ts + 1e-37).all(), ("slope", float((offs / (ts + 1e-37)).max()))


def test_activations_of_infinities():
    for act, up, down in (("tanh", 1.0, -1.0), ("silu", math.inf, 0.0), ("relu", math.inf, 0.0)):
        p = Norm([3], 8, 2, act, "fp32")
        p.gd.zero_()
        p.bd = torch.tensor([math.inf, -math.inf, math.nan, 3e38, -3e38, 100.0, -100.0, 0.0], device=DEV)
        y = p.forward("fp32")[0][0].cpu()
        assert y[0] == up and y[1] == down and math.isnan(y[2]) and abs(float(y[4])) <= (1 if act == "tanh" else 0) and y[7] == 0


@pytest.mark.parametrize("types", [("fp32", "fp32", "fp32", "fp32"), ("fp32", "bf16", "bf16", "bf16"), ("bf16", "fp32", "fp32", "bf16")])
@pytest.mark.parametrize("lens,C,G,act", [
    ([700, 0, 35], 512, 1, "silu"),                  # a row takes more than a wave, 16 rows to a chunk
    ([300, 9], 1024, 1, "tanh"),                     # ... 8 rows
    ([100, 4], 1024, 2, "none"),
    ([2500], 512, 1, "none"),                        # 157 chunks of one group
    ([600, 0, 1], 768, 3, "relu"),                   # a strip is one of three groups
    ([5000, 17, 90], 24, 8, "tanh"),                 # groups of three channels, narrow strips
])
def test_group_norm_of_wide_rows_in_chunks(lens, C, G, act, types):
    base.test_group_norm(lens, C, G, act, *types)


@pytest.mark.parametrize("lens", [[100], [13, 0, 100]])
def test_group_norm_of_rows_that_no_power_of_two_divides(lens):
    """524 channels in 131 groups: a row of 131 lanes, one row at a time in a chunk of 256 threads"""
    base.test_group_norm(lens, 524, 131, "silu", "fp32", "fp32", "fp32", "fp32")


def test_group_norm_of_many_chunks_in_graphs_and_streams():
    """94 chunks: the join is a launch of its own.  Two captured graphs with a workspace each, replayed in turn with eager work between,
    then calls on two streams at once"""
    probs = [Norm([1500, 0, 300], 512, 1, "tanh", "fp32", seed=s) for s in (1, 2)]
    for p in probs:
        p.dout = p.dout.to(DEV)
    run = lambda p: (lambda y, st: [y, st, *p.backward(st, "fp32", "fp32")])(*p.forward("fp32"))
    want = [run(p) for p in probs]
    torch.cuda.synchronize()
    graphs = []
    for p in probs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run(p)
        graphs.append((g, out))
    for _ in range(3):
        for (g, out), w, p in zip(graphs, want, probs):
            for o in out:
                o.fill_(3.0)
            g.replay()
            run(p)
            torch.cuda.synchronize()
            for got, ref in zip(out, w):
                assert torch.equal(got[:1800], ref[:1800]) if got.shape[0] == p.M else torch.equal(got, ref)
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
        for p, st in zip(probs, streams):
            with torch.cuda.stream(st):
                got.append(run(p))
    for st in streams:
        st.synchronize()
    for k, out in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(out, want[k % 2]))
