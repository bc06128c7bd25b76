"""What packing launches, without a GPU (a HIP runtime that only logs)."""
from test_workspaces_host import run  # noqa: F401


def test_packing_linear_weights_is_one_launch(run):
    seen = run("""
lib = _lib.load_library()
B = [(1 + i) << 43 for i in range(8)]
for k, n in ((0, 5), (64, 48), (4096, 131072), (64, 4000000)):
    assert lib.vt_scaled_pack(B[0], None, n, 0, B[1], None, None, k, n, B[2], B[3], STREAM) == 0, _lib.last_error()
print(json.dumps([e[3].split(" ")[1] for e in launches()]))
""")
    assert len(seen) == 4 and all("pack_scaled_kernel" in e for e in seen)
