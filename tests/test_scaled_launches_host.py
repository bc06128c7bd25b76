"""What the scaled operators launch, on the CPU: their host code runs against a HIP runtime that only logs
(fake_hip.cpp). Operand addresses are made up and never read."""
import re
import subprocess

import pytest

from scaled_cases import CASES
from veritac_amd import _lib
from test_workspaces_host import run  # noqa: F401

CALLS = """
lib = _lib.load_library()
F32, F16, BF16, I8, I8P = 1, 2, 3, 4, 5
BASE = [(1 + i) << 43 for i in range(6)]

def ok(rc):
    assert rc == 0, (rc, _lib.last_error())

def linear(m, k, n, x=BF16, y=BF16, ldx=None, stream=STREAM):
    ok(lib.vt_scaled_linear(BASE[0], x, k if ldx is None else ldx, BASE[1], m, k, BASE[2], BASE[3], n, BASE[4], y, n, stream))

def gated(m, k, n, x=BF16, y=BF16, ldx=None, act=0, stream=STREAM):
    ok(lib.vt_scaled_gated(BASE[0], x, k if ldx is None else ldx, BASE[1], m, k, BASE[2], BASE[3], n, act, BASE[4], y, n, stream))

def linear_grad(m, k, n, t=BF16, stream=STREAM):
    ok(lib.vt_scaled_linear_grad(BASE[0], t, n, m, k, BASE[2], BASE[3], n, BASE[4], k, stream))

def gated_grad(m, k, n, t=BF16, x=I8, ldx=None, stream=STREAM):
    ok(lib.vt_scaled_gated_grad(BASE[0], t, n, BASE[5], x, k if ldx is None else ldx, BASE[1], m, k, BASE[2], BASE[3], n, 0,
                                BASE[4], k, stream))
"""


@pytest.mark.parametrize("op", ["linear", "gated"])
@pytest.mark.parametrize("kind,ldx", [("I8", 0), ("I8", 1), ("I8", 16), ("I8P", 0), ("I8P", 1), ("I8P", 16), ("F32", 0),
                                      ("BF16", 5)])
def test_empty_sums_need_no_rows(run, op, kind, ldx):
    """K = 0: the bias or zeros, whatever the rows; no launch of an empty grid."""
    seen = run(CALLS + """
import json
%s(5, 0, 40, x=%s, ldx=%d)
print(json.dumps([e[3] for e in launches()]))
""" % (op, kind, ldx))
    assert "finish_kernel" in seen[-1] and len(seen) == (1 if kind.startswith("I8") else 2)
    assert all(int(e.split(" ")[0]) > 0 for e in seen)


def compiled():
    """The operators' kernels in the built library, by the stubs that launch them (packing aside)."""
    text = subprocess.run(["nm", _lib.load_library()._name], check=True, capture_output=True, text=True).stdout
    found = set()
    for stub in re.findall(r"\S*__device_stub__\S+", text):
        if re.search("scaled_skinny|dma16_kernel.*ScaledTile|mfma_kernel.*ScaledTile|grad_dma|grad_sum|quant_rows|pad_rows|"
                     "row_terms|finish_kernel|zero_rows", stub):
            found.add(re.sub(r"(\d+)__device_stub__", lambda m: str(int(m.group(1)) - 15), stub))
    return found


# sizes that need none of the products
SIMPLE = """
linear(300, 100, 70, x=I8)
linear_grad(3, 64, 0)
"""


def test_every_kernel_has_a_case(run):
    """The cases that the GPU tests check reach every kernel that is built, so none stays that no call reaches
    and a change of the rules that choose them cannot leave one untested."""
    seen = run(CALLS + SIMPLE + """
kinds = {"f32": F32, "f16": F16, "bf16": BF16}
for op, m, k, n, t, rows in %r:
    x = I8 if rows == "i8" else kinds[t]
    if op == "linear": linear(m, k, n, x=x, y=kinds[t])
    elif op == "gated": gated(m, k, n, x=x, y=kinds[t])
    elif op == "linear_grad": linear_grad(m, k, n, kinds[t])
    else: gated_grad(m, k, n, kinds[t])
import json
print(json.dumps(sorted({e[3].split(" ")[1] for e in launches()})))
""" % (CASES,))
    names = compiled()
    assert len(names) > 90
    assert not names - set(seen), sorted(names - set(seen))


def test_workspaces_stay_bounded(run):
    """However many rows a call has: at most 512 MiB of int8 rows, of gradient terms and of partial sums each."""
    got = run(CALLS + """
import json
out = []
for call in (lambda s: linear(1 << 20, 4096, 4096, stream=s), lambda s: linear(200000, 100000, 64, x=F32, y=F32, stream=s),
             lambda s: gated(150000, 14336, 40, x=I8, ldx=14337, stream=s), lambda s: linear(1 << 23, 64, 16, stream=s),
             lambda s: linear_grad(1 << 20, 4096, 4096, F32, stream=s), lambda s: linear_grad(70000, 128, 28672, stream=s),
             lambda s: linear_grad(4096, 10000, 256000, stream=s), lambda s: linear_grad(300, 16000, 1500000, F16, stream=s),
             lambda s: gated_grad(8192, 4096, 14336, F32, stream=s), lambda s: gated_grad(1 << 18, 4000, 14336, BF16, stream=s)):
    fake.fake_reset()
    STREAM += 1
    call(STREAM)
    out.append(allocated())
print(json.dumps(out))
""")
    for sizes in got:
        assert sizes and max(sizes) <= 512 << 20, sizes
    assert any(s > 400 << 20 for sizes in got for s in sizes)


def test_rows_in_parts_are_all_there(run):
    """Parts of whole 256-row tiles that add up to the call's rows, at their own addresses."""
    for call, bytes_a_row, rows in (("linear_grad(40000, 64, 8192, F32)", 4 * 8192 + 4, 40000),
                                    ("gated_grad(30001, 64, 8192, BF16)", 4 * 8192 + 4, 30001),
                                    ("linear(100000, 16384, 32)", 16384 + 4, 100000)):
        seen = run(CALLS + """
import json
%s
print(json.dumps([e[3] for e in launches()]))
""" % call)
        first = [int(e.split(" ")[0]) for e in seen if "row_terms" in e or "quant_rows" in e]     # a workgroup a row
        assert sum(first) == rows and len(first) == -(-rows // ((512 << 20) // bytes_a_row // 256 * 256))
        assert all(r % 256 == 0 for r in first[:-1]) and max(first) * bytes_a_row <= 512 << 20


THREADS = ["linear(48, 14336, 4096, stream=STREAM)", "linear(300, 1000, 70, x=I8, stream=STREAM)", "gated(500, 1000, 700, stream=STREAM)",
           "linear_grad(300, 999, 1001, F32, stream=STREAM)", "gated_grad(100, 333, 1203, F16, stream=STREAM)",
           "linear(72, 5376, 3584, stream=STREAM)"]


@pytest.mark.parametrize("call", THREADS)
def test_a_scaled_call_keeps_its_workspace_until_its_last_launch(run, call):
    """Two host threads on one stream: no launch of one comes between the launches of the other's call."""
    seen, per = run(CALLS + """
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
print(json.dumps([[e[0] for e in launches()], per]))
""" % call)
    assert per >= 2 and len(seen) == 12 * per and set(seen) == {"0", "1"}
    assert all(len(set(seen[i:i + per])) == 1 for i in range(0, len(seen), per))
