"""The alignment operators without a GPU: every refusal returns before anything is launched, and the workspace queries are
pure functions of the shape."""
import pytest

from fastspeech2_amd import hip

P = 1 << 20                     # an aligned address nothing reads: the checks run on the host, in front of any launch


def _attend(**kw):
    a = dict(q=P, k=P, v=P, ctx=P, lse=P, cu_q=P, cu_k=P, ws=P, B=2, max_q=8, max_k=9, Mq=16, Mk=18, H=4, KV=2, dk=64, ldq=256,
             ldk=128, ldv=128, ldo=256, dtype=1, seed=0, site=0, rate=0.0)
    assert set(kw) <= set(a)
    a.update(kw)
    return a


def _forward(change):
    hip.call("fs2_cross_attention", *_attend(**change).values(), 0)


def _mass(change):
    a = dict(_attend(**{k: v for k, v in change.items() if k != "mass"}), mass=change.get("mass", P))
    order = ("q", "k", "lse", "mass", "cu_q", "cu_k", "ws", "B", "max_q", "max_k", "Mq", "Mk", "H", "KV", "dk", "ldq", "ldk", "dtype")
    hip.call("fs2_cross_attention_mass", *[a[k] for k in order], 0)


ATTEND_REFUSED = [
    (dict(cu_q=None), "bad args"), (dict(cu_k=None), "bad args"), (dict(B=0), "bad args"), (dict(Mq=-1), "bad args"),
    (dict(max_k=-1), "bad args"), (dict(q=None), "null q or k"), (dict(k=None), "null q or k"), (dict(dtype=2), "dtype=2"),
    (dict(dk=48, ldq=192, ldk=96), "head dim 48"), (dict(KV=3), "4 heads over 3"), (dict(KV=0), "4 heads over 0"),
    (dict(B=65536), "B=65536"), (dict(max_q=17), "max_q=17 > Mq=16"), (dict(max_k=19), "max_k=19 > Mk=18"),
    (dict(ldq=255), "ldq=255"), (dict(ldq=248), "ldq=248"), (dict(ldk=130), "ldk=130"), (dict(q=P + 8), "unaligned q or k"),
    (dict(k=P + 2), "unaligned q or k"),
    (dict(max_q=1 << 25, Mq=1 << 25), "max_q=33554432"), (dict(max_k=(1 << 30) + 1, Mk=(1 << 31) - 1), "max_k=1073741825"),
    (dict(B=60000, max_q=1 << 22, Mq=1 << 24, H=4), "in one launch"),
]


@pytest.mark.parametrize("change,text", ATTEND_REFUSED)
def test_cross_attention_refuses(change, text):
    for refused in (_forward, _back, _mass):
        with pytest.raises(hip.HipError, match=text):
            refused(change)


def _back(change):
    a = _attend(**change)
    tail = [a[k] for k in ("cu_q", "cu_k", "ws", "B", "max_q", "max_k", "Mq", "Mk", "H", "KV", "dk", "ldq", "ldk", "ldv", "ldo", "dtype",
                           "seed", "site", "rate")]
    back = dict(dctx=P, dq=P, dk_=P, dv=P)
    back.update({k: v for k, v in change.items() if k in back})
    hip.call("fs2_cross_attention_bwd", a["q"], a["k"], a["v"], a["ctx"], back["dctx"], a["lse"], back["dq"], back["dk_"], back["dv"],
             *tail, 0)


@pytest.mark.parametrize("change,text", [
    (dict(v=None), "null or unaligned v"), (dict(ctx=P + 4), "null or unaligned v or ctx"), (dict(ldv=120), "ldv=120"),
    (dict(ldo=252), "ldo=252"), (dict(ldo=(1 << 20) + 8), "ldo=1048584"), (dict(rate=1.0), "dropout rate"), (dict(rate=-0.1), "dropout rate"),
    (dict(B=1, max_q=1, Mq=1, max_k=4000, Mk=4000, ws=None), "fs2_cross_attention_workspace bytes"),
    (dict(B=1, max_q=1, Mq=1, max_k=4000, Mk=4000, ws=P + 8), "fs2_cross_attention_workspace bytes"),
])
def test_cross_attention_forward_refuses(change, text):
    with pytest.raises(hip.HipError, match=text):
        _forward(change)


@pytest.mark.parametrize("change,text", [
    (dict(ctx=None), "null argument"), (dict(lse=None), "null argument"), (dict(v=None), "null argument"),
    (dict(ctx=P + 4), "unaligned"), (dict(ldv=120), "ldv=120"), (dict(ldo=1 << 28), "ldo=268435456"), (dict(rate=1.5), "dropout rate"), (dict(ws=None), "workspace bytes"),
    (dict(ws=P + 4), "workspace bytes"), (dict(B=32768, max_q=4096, Mq=1 << 20), "32768 x 4 heads x max_q=4096"),
])
def test_cross_attention_backward_refuses(change, text):
    with pytest.raises(hip.HipError, match=text):
        _back(change)


@pytest.mark.parametrize("change,text", [
    (dict(lse=None), "null lse or mass"), (dict(mass=None), "null lse or mass"),
    (dict(B=1, max_q=3000, Mq=3000, ws=None), "fs2_cross_attention_mass_workspace bytes")])
def test_mass_refuses(change, text):
    with pytest.raises(hip.HipError, match=text):
        _mass(change)


def test_nothing_to_do_is_no_error():
    _forward(dict(Mq=0, max_q=0, q=None, ctx=None))
    _back(dict(Mq=0, max_q=0, Mk=0, max_k=0))


def _norm(**kw):
    a = dict(x=P, cu=P, gamma=P, beta=P, out=P, stats=P, ws=P, B=2, max_len=8, M=16, C=80, G=16, ldx=80, ldo=80, eps=1e-5, act=2,
             x_dtype=0, out_dtype=1, seed=0, site=0, rate=0.0)
    assert set(kw) <= set(a)
    a.update(kw)
    return a


NORM_REFUSED = [
    (dict(cu=None), "bad args"), (dict(gamma=None), "bad args"), (dict(beta=None), "bad args"), (dict(stats=None), "bad args"),
    (dict(x=None), "bad args"), (dict(B=0), "bad args"), (dict(max_len=17), "max_len=17"), (dict(x_dtype=2), "x_dtype=2"),
    (dict(C=82, G=2), "C=82"), (dict(C=84, G=2, x_dtype=1), "C=84"), (dict(C=1040, ldx=1040, ldo=1040), "C=1040"), (dict(G=3), "80 channels in 3"),
    (dict(ldx=76), "ldx=76"), (dict(ldx=82), "ldx=82"), (dict(x=P + 8), "unaligned"), (dict(act=4), "act=4"), (dict(rate=1.0), "dropout"),
    (dict(B=1 << 23), "too many workgroups"),
]


@pytest.mark.parametrize("change,text", NORM_REFUSED + [
    (dict(out=None), "out null"), (dict(ldo=82), "ldo=82"), (dict(out=P + 4), "unaligned"), (dict(out_dtype=3), "out_dtype=3"),
    (dict(eps=0.0), "eps"), (dict(max_len=90000, M=90000, ws=None), "fs2_group_norm_workspace")])
def test_group_norm_refuses(change, text):
    with pytest.raises(hip.HipError, match=text):
        hip.call("fs2_group_norm", *_norm(**change).values(), 0)


@pytest.mark.parametrize("change,text", NORM_REFUSED + [
    (dict(ws=None), "null argument"), (dict(dout=None), "null argument"), (dict(dgamma=None), "null argument"),
    (dict(ldd=78), "ldd=78"), (dict(ldg=70), "ldg=70"), (dict(dx=P + 4), "unaligned"), (dict(dx_dtype=2), "dx_dtype=2")])
def test_group_norm_backward_refuses(change, text):
    extra = dict(dout=P, dx=P, dgamma=P, dbeta=P, ldd=80, ldg=80, dout_dtype=0, dx_dtype=1)
    extra.update({k: v for k, v in change.items() if k in extra})
    a = dict(_norm(**{k: v for k, v in change.items() if k not in extra}), **extra)
    order = ("x", "stats", "cu", "gamma", "beta", "dout", "dx", "dgamma", "dbeta", "ws", "B", "max_len", "M", "C", "G", "ldx", "ldd",
             "ldg", "act", "x_dtype", "dout_dtype", "dx_dtype", "seed", "site", "rate")
    with pytest.raises(hip.HipError, match=text):
        hip.call("fs2_group_norm_bwd", *[a[k] for k in order], 0)


def test_workspace_queries():
    lib = hip.load()
    # a batch that fills the chip with its own work items needs none; one short query against many keys does
    assert lib.fs2_cross_attention_workspace(32, 800, 120, 25600, 2, 2, 128, 1) == 0
    assert lib.fs2_cross_attention_workspace(1, 1, 4000, 1, 2, 2, 128, 1) > 0
    assert lib.fs2_cross_attention_workspace(0, 1, 4000, 1, 2, 2, 128, 1) == 0
    # delta, 16-byte rounded
    assert lib.fs2_cross_attention_bwd_workspace(64, 1, 120, 33, 64, 9, 9, 64, 1) >= 4 * 33 * 9
    assert lib.fs2_cross_attention_mass_workspace(64, 8, 120, 64, 9, 9, 64, 1) == 0
    assert lib.fs2_group_norm_workspace(4, 100, 256, 16) == 0
    assert lib.fs2_group_norm_workspace(4, 100000, 256, 16) > 0
    assert lib.fs2_group_norm_bwd_workspace(4, 100, 256, 16) >= 4 * 2 * 256 * 4
