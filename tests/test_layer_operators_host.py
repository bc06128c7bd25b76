"""Norms, adapters and the loss without a GPU: refusals of the C entries before a device call, the Python layer's
checks, and what the host code launches (a HIP runtime that only logs; operand addresses are never read)."""
import json
import re
import subprocess

import pytest

torch = pytest.importorskip("torch")

import adapter_ref
import loss_ref
from test_workspaces_host import run  # noqa: F401
from veritac_amd import _lib
from veritac_amd._lib import HipGemmError
from veritac_amd.specializations.hip_gemm import adapters, losses, norms, scaled

F32, F16, BF16, I8, I8P = _lib.TYPE_F32, _lib.TYPE_F16, _lib.TYPE_BF16, _lib.TYPE_I8, _lib.TYPE_I8_PADDED
A = [(1 + i) << 30 for i in range(16)]     # addresses that no check reads


@pytest.fixture(scope="module")
def lib():
    return _lib.load_library()


def norm(lib, X=A[0], ldx=64, R=A[1], ldr=64, t=F32, g=A[2], gt=F32, eps=1e-6, H=A[3], ldh=64, Y=A[4], ldy=64, T=None, M=4, K=64):
    return lib.vt_norm(X, ldx, R, ldr, t, g, gt, eps, H, ldh, Y, ldy, T, M, K, None)


@pytest.mark.parametrize("kw", [
    dict(M=-1), dict(K=-1), dict(M=1 << 24), dict(K=1 << 30), dict(t=I8), dict(gt=F16), dict(t=BF16, gt=F16), dict(eps=-1.0),
    dict(eps=float("nan")), dict(X=None), dict(g=None), dict(Y=None), dict(R=None), dict(H=None), dict(ldx=63), dict(ldr=63),
    dict(ldh=63), dict(ldy=63), dict(ldx=1 << 41), dict(X=A[0] + 2), dict(g=A[2] + 1), dict(Y=A[0]), dict(H=A[0]), dict(H=A[4]),
    dict(Y=A[2]), dict(H=A[1] + 256), dict(H=A[1], ldh=128), dict(T=A[5], ldy=64), dict(T=A[5], ldy=136), dict(T=A[5], ldy=128, Y=A[4] + 8),
    dict(T=A[4], ldy=128), dict(T=A[0], ldy=128)], ids=str)
def test_norm_refuses(lib, kw):
    assert norm(lib, **kw) == _lib.VT_EINVAL and "vt_norm" in _lib.last_error(), kw


def norm_grad(lib, D=A[0], ldd=64, H=A[1], ldh=64, E=A[2], lde=64, t=F32, g=A[3], gt=F32, eps=1e-6, X=A[4], ldx=64, dg=A[5], M=4, K=64):
    return lib.vt_norm_grad(D, ldd, H, ldh, E, lde, t, g, gt, eps, X, ldx, dg, M, K, None)


@pytest.mark.parametrize("kw", [
    dict(M=-1), dict(K=1 << 30), dict(t=0), dict(gt=BF16), dict(eps=-0.5), dict(D=None), dict(H=None), dict(X=None), dict(g=None),
    dict(ldd=63), dict(lde=60), dict(X=A[0]), dict(X=A[2]), dict(dg=A[3]), dict(dg=A[4]), dict(dg=A[5] + 2)], ids=str)
def test_norm_grad_refuses(lib, kw):
    assert norm_grad(lib, **kw) == _lib.VT_EINVAL and "vt_norm_grad" in _lib.last_error(), kw


def loss(lib, X=A[0], t=F32, ldx=64, T=None, M=4, K=64, B=A[1], meta=A[2], N=32, y=A[3], yt=_lib.TARGET_I64, out=A[4], state=A[5],
         red=1, one=A[6], count=A[7]):
    return lib.vt_cross_entropy(X, t, ldx, T, M, K, B, meta, N, y, yt, -100, out, state, red, one, count, None)


@pytest.mark.parametrize("kw", [
    dict(N=0), dict(M=-1), dict(K=131072, ldx=131072), dict(t=7), dict(yt=3), dict(y=None), dict(y=A[3] + 4), dict(out=None), dict(state=None),
    dict(state=A[5] + 4), dict(red=4), dict(one=None), dict(count=None), dict(X=None), dict(B=None), dict(meta=None), dict(ldx=63),
    dict(out=A[0]), dict(state=A[4]), dict(one=A[7]), dict(out=A[3]), dict(t=I8), dict(t=I8P, T=A[8]), dict(count=A[5])], ids=str)
def test_loss_refuses(lib, kw):
    assert loss(lib, **kw) == _lib.VT_EINVAL and "vt_cross_entropy" in _lib.last_error(), kw


def loss_grad(lib, Q=A[0], qt=I8P, ldq=128, T=A[1], M=4, K=64, B=A[2], meta=A[3], N=32, state=A[4], d=A[5], step=1, count=None, X=A[6],
              t=F32, ldx=64):
    return lib.vt_cross_entropy_grad(Q, qt, ldq, T, M, K, B, meta, N, state, d, step, count, X, t, ldx, None)


@pytest.mark.parametrize("kw", [dict(N=0), dict(qt=F32), dict(T=None), dict(state=None), dict(d=None), dict(step=2), dict(X=None), dict(t=I8),
                                dict(ldx=63), dict(ldq=64), dict(X=A[4]), dict(X=A[5]), dict(X=A[0]), dict(count=A[6])], ids=str)
def test_loss_grad_refuses(lib, kw):
    assert loss_grad(lib, **kw) == _lib.VT_EINVAL and "vt_cross_entropy_grad" in _lib.last_error(), kw


def adapted(lib, X=A[0], t=F32, ldx=64, T=None, M=4, K=64, B=A[1], meta=A[2], N=32, P=A[3], R=8, L=2, c=1.0, w=A[4], U=A[5], Y=A[6], yt=F32, ldy=32):
    return lib.vt_adapted_linear(X, t, ldx, T, M, K, B, meta, N, P, R, L, c, w, U, Y, yt, ldy, None)


@pytest.mark.parametrize("kw", [
    dict(R=0), dict(R=129), dict(L=0), dict(L=65536), dict(t=F16), dict(t=F16, yt=BF16, ldy=32), dict(yt=I8), dict(X=None), dict(P=None),
    dict(U=None), dict(P=A[3] + 8), dict(U=A[5] + 4), dict(w=A[4] + 2), dict(U=A[0]), dict(Y=A[5]), dict(Y=A[4]), dict(U=A[3]),
    dict(ldy=31), dict(M=-1), dict(K=-1), dict(N=-1), dict(t=I8)], ids=str)
def test_adapted_refuses(lib, kw):
    assert adapted(lib, **kw) == _lib.VT_EINVAL and "vt_adapted_linear" in _lib.last_error(), kw


def adapted_grad(lib, D=A[0], t=F32, ldd=32, X=A[1], ldx=64, M=4, K=64, B=A[2], meta=A[3], N=32, P=A[4], back=A[5], R=8, L=2, c=1.0, w=A[6],
                 U=A[7], H=A[8], dX=A[9], lddx=64, dd=A[10], du=A[11]):
    return lib.vt_adapted_grad(D, t, ldd, X, ldx, M, K, B, meta, N, P, back, R, L, c, w, U, H, dX, lddx, dd, du, None)


@pytest.mark.parametrize("kw", [
    dict(R=0), dict(L=0), dict(t=I8), dict(D=None), dict(X=None), dict(back=None), dict(U=None), dict(H=None), dict(ldd=31), dict(ldx=63),
    dict(lddx=63), dict(dX=A[0]), dict(dd=A[11]), dict(du=A[1]), dict(H=A[7]), dict(H=A[5]), dict(dX=A[8]), dict(dd=A[10] + 2), dict(M=-1)], ids=str)
def test_adapted_grad_refuses(lib, kw):
    assert adapted_grad(lib, **kw) == _lib.VT_EINVAL and "vt_adapted_grad" in _lib.last_error(), kw


def test_adapter_layouts(lib):
    for k, n, r, count in ((64, 96, 1, 1), (1000, 14336, 16, 3), (4096, 77, 17, 2), (100, 100, 128, 5)):
        rp = 16 if r <= 16 else -(-r // 32) * 32
        assert _lib.adapter_size(k, n, r, count, F16) == 2 * count * rp * (_lib.quant_pitch(k) + -(-n // 64) * 64)
    for bad in ((64, 64, 0, 1), (64, 64, 129, 1), (64, 64, 4, 0), (-1, 64, 4, 1), (131072, 64, 4, 1)):
        with pytest.raises(HipGemmError):
            _lib.adapter_size(*bad, F32)
    assert lib.vt_adapter_pack(A[0], A[1], F32, 64, 64, 4, 1, A[0], None, None) == _lib.VT_EINVAL
    assert lib.vt_adapter_pack(None, A[1], F32, 64, 64, 4, 1, A[2], None, None) == _lib.VT_EINVAL
    assert lib.vt_adapter_pack(A[0], A[1], F32, 64, 64, 4, 1, A[2] + 4, None, None) == _lib.VT_EINVAL
    assert lib.vt_adapter_pack(A[0], A[1], F32, 64, 64, 4, 1, A[2], A[2], None) == _lib.VT_EINVAL


def weight(k=64, n=32, pair=False):
    size, floats = _lib.scaled_size(k, n, pair)
    return scaled.ScaledWeight(torch.zeros(size, dtype=torch.int8), torch.zeros(floats), k, n, pair)


X, G, Y = torch.zeros(3, 64), torch.ones(64), torch.zeros(3, 32)
DOWN, UP, INDEX, TARGET = torch.zeros(2, 4, 64), torch.zeros(2, 32, 4), torch.zeros(3, dtype=torch.int32), torch.zeros(3, dtype=torch.int64)
CALLS = {"norm": lambda x: norms.norm(x, G), "norm_rows": lambda x: norms.norm_rows(x, G),
         "norm_grad": lambda x: norms.norm_grad(x, X, G), "cross_entropy": lambda x: losses.cross_entropy(x, weight(), TARGET),
         "adapted": lambda x: adapters.adapted(x, weight(), (DOWN, UP), INDEX),
         "adapted_grad": lambda x: adapters.adapted_grad(Y if x is X else x[:, :32], X, weight(), (DOWN, UP), INDEX)}


@pytest.mark.parametrize("name", CALLS)
def test_there_is_no_cpu_path(name):
    with pytest.raises(HipGemmError, match="no CPU path|rows are|must be on a gfx950"):
        CALLS[name](X)


@pytest.mark.parametrize("name", CALLS)
def test_forward_mode_is_refused(name):
    import torch.autograd.forward_ad as forward_ad
    with forward_ad.dual_level():
        v = forward_ad.make_dual(torch.zeros(3, 64), torch.ones(3, 64))
        with pytest.raises(HipGemmError, match="forward-mode"):
            CALLS[name](v)


@pytest.mark.parametrize("name,call", [
    ("norm_rows", lambda x: norms.norm_rows(x, G)), ("norm_rows", lambda x: norms.norm_rows(X, G, residual=x)),
    ("norm_rows", lambda x: norms.norm_rows(X, x[0])), ("norm_grad", lambda x: norms.norm_grad(x, X, G)),
    ("norm_grad", lambda x: norms.norm_grad(X, X, G, dh=x)), ("pack_adapters", None),
    ("adapted_grad", lambda x: adapters.adapted_grad(x[:, :32], X, weight(), (DOWN, UP)))],
    ids=["rows", "residual", "gain", "dy", "dh", "down", "adapted_grad"])
def test_gradients_are_not_left_out(name, call):
    v = torch.zeros(3, 64, requires_grad=True)
    if call is None:
        call = lambda x: adapters.pack_adapters(DOWN.clone().requires_grad_(), UP)  # noqa: E731
    with pytest.raises(HipGemmError, match="%s passes no gradient" % name):
        call(v)


CODE = """
lib = _lib.load_library()
B = [(1 + i) << 41 for i in range(20)]

def ok(rc):
    assert rc == 0, (rc, _lib.last_error())

def norm(m, k, t=3, rows=False, res=True, stream=STREAM):
    ok(lib.vt_norm(B[0], k, B[1] if res else None, k, t, B[2], 1, 1e-6, B[3] if res else None, k, B[4], _lib.quant_pitch(k) if rows else k,
                   B[5] if rows else None, m, k, stream))

def norm_grad(m, k, t=3, dg=True, stream=STREAM):
    ok(lib.vt_norm_grad(B[0], k, B[1], k, B[2], k, t, B[3], 1, 1e-6, B[4], k, B[5] if dg else None, m, k, stream))

def loss(m, k, n, t=3, red=1, stream=STREAM):
    ok(lib.vt_cross_entropy(B[0], t, k, B[1], m, k, B[2], B[3], n, B[4], 2, -100, B[5], B[6], red, B[7], B[8], stream))

def loss_grad(m, k, n, t=3, qt=4, stream=STREAM):
    ok(lib.vt_cross_entropy_grad(B[0], qt, k, B[1], m, k, B[2], B[3], n, B[4], B[5], 1, None, B[6], t, k, stream))

def adapted(m, k, n, r, l, t=3, x=None, stream=STREAM):
    ok(lib.vt_adapted_linear(B[0], t if x is None else x, k, B[1], m, k, B[2], B[3], n, B[4], r, l, 1.0, B[5], B[6], B[7], t, n, stream))

def adapted_grad(m, k, n, r, l, t=3, again=True, stream=STREAM):
    ok(lib.vt_adapted_grad(B[0], t, n, B[1], k, m, k, B[2], B[3], n, B[4] if again else None, B[5], r, l, 1.0, B[6], B[7], B[8], B[9], k,
                           B[10], B[11], stream))

def pack(k, n, r, l, t=3, stream=STREAM):
    ok(lib.vt_adapter_pack(B[0], B[1], t, k, n, r, l, B[2], B[3], stream))
"""


def compiled():
    """The new operators' kernels in the built library, by the stubs that launch them."""
    text = subprocess.run(["nm", _lib.load_library()._name], check=True, capture_output=True, text=True).stdout
    found = set()
    for stub in re.findall(r"\S*__device_stub__\S+", text):
        if re.search("norm_|gain_sum|dequant|out_dma16|LseTile|LossTerms|logit_parts|loss_|adapt|shrink|outer", stub):
            found.add(re.sub(r"(\d+)__device_stub__", lambda m: str(int(m.group(1)) - 15), stub))
    return found


def test_every_kernel_has_a_case(run):
    """The cases that the GPU tests check reach every kernel that is built, of the operators that have more than one."""
    sizes = [(1, 1), (3, 7), (5, 511), (70, 513), (40, 4096), (3, 4097), (7, 8192), (3, 8200), (2, 16384), (4, 16390)]
    seen = run(CODE + """
import json
for t in (1, 2, 3):
    for m, k in %r:
        norm(m, k, t); norm(m, k, t, rows=True); norm_grad(m, k, t)
    ok(lib.vt_dequant_rows(B[0], 64, B[1], B[2], t, 64, 3, 64, STREAM))
    for m, k, n in %r:
        loss(m, k, n, t); loss_grad(m, k, n, t)
    for m, k, n, r, l in %r:
        adapted(m, k, n, r, l, t); adapted(m, k, n, r, l, t, x=4); adapted_grad(m, k, n, r, l, t)
    pack(64, 64, 4, 2, t)
print(json.dumps(sorted({e[3].split(" ")[1] for e in launches()})))
""" % (sizes, loss_ref.CASES, adapter_ref.CASES))
    names = compiled()
    assert len(names) > 100
    assert not names - set(seen), sorted(names - set(seen))


def test_workspaces_stay_bounded(run):
    """However many rows a call has: at most 512 MiB of each kind, 600 where a part is 64 rows."""
    got = run(CODE + """
import json
out = []
for call in (lambda s: loss(1 << 20, 4096, 32000, stream=s), lambda s: loss(200000, 64, 4000000, stream=s), lambda s: loss(64, 64, 4000000, stream=s),
             lambda s: loss(1 << 20, 0, 1000, stream=s), lambda s: loss_grad(1 << 18, 4096, 131072, stream=s), lambda s: loss_grad(5000, 4096, 131072, 1, stream=s),
             lambda s: adapted(1 << 20, 4096, 4096, 16, 9, stream=s), lambda s: adapted_grad(1 << 18, 4096, 14336, 64, 2, 1, stream=s),
             lambda s: adapted_grad(100000, 14336, 4096, 128, 300, stream=s), lambda s: norm_grad(1 << 20, 8192, stream=s),
             lambda s: norm_grad(1 << 20, 100000, stream=s)):
    fake.fake_reset()
    STREAM += 1
    call(STREAM)
    out.append(allocated())
print(json.dumps(out))
""")
    for sizes in got:
        assert max(sizes, default=0) <= 600 << 20, sizes
    assert any(s > 300 << 20 for sizes in got for s in sizes)


@pytest.mark.parametrize("call", ["loss(300, 1000, 5000, stream=STREAM)", "loss(5, 1000, 5000, stream=STREAM)", "loss_grad(300, 1000, 5000, stream=STREAM)",
                                  "adapted(48, 4096, 4096, 16, 4, stream=STREAM)", "adapted_grad(300, 999, 1001, 5, 3, 1, stream=STREAM)",
                                  "norm_grad(300, 4096, stream=STREAM)"])
def test_a_call_keeps_its_workspace_until_its_last_launch(run, call):
    """Two host threads on one stream: between a call's first workspace and the launches that use it none of the
    other's comes. (u's kernel, and the sum of the rows' losses, use none.)"""
    seen, per = run(CODE + """
import json
def calls():
    for _ in range(6):
        %s
calls()
per = len(launches()) // 6
fake.fake_reset()
fake.fake_pause(1000)
ts = [threading.Thread(target=calls) for _ in range(2)]
[t.start() for t in ts]; [t.join() for t in ts]
print(json.dumps([[[e[0], e[3].split(" ")[1]] for e in launches()], per]))
""" % call)
    assert per >= 2 and len(seen) == 12 * per
    alone = re.compile("loss_sum_kernel|shrink_tiles|outer")
    held = [who for who, name in seen if not alone.search(name)]
    kept = len(held) // 12
    # the parts of the adapters' gradients are two holds: dx, and the sums of down's and up's
    assert kept >= 1 and all(len(set(held[i:i + kept])) == 1 for i in range(0, len(held), kept)), held


def test_no_empty_grid(run):
    got = run(CODE + """
import json
for m in (0, 1, 65, 300):
    for k in (0, 5):
        norm(m, k); norm(m, k, rows=True); norm_grad(m, k)
        for n in (1, 70):
            loss(m, k, n); loss_grad(m, k, n)
        for n in (0, 70):
            adapted(m, k, n, 3, 2); adapted_grad(m, k, n, 3, 2); pack(k, n, 3, 2)
print(json.dumps([e[3] for e in launches()]))
""")
    assert got and all(int(e.split(" ")[0]) > 0 for e in got), [e for e in got if int(e.split(" ")[0]) == 0]
