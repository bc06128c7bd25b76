"""Launches of norms and the loss at the largest sizes that their entries admit, without a GPU (a HIP runtime that only
logs): a launch has less than 2^32 threads, and at most 65535 workgroups along its second side."""
from test_layer_operators_host import CODE
from test_workspaces_host import run  # noqa: F401


def test_row_statistics_of_any_number_of_rows(run):
    """norm_stats_kernel: workgroups of 1024."""
    seen = run(CODE + """
import json
for m in (1, 700, (1 << 22) - 1, 1 << 22, (1 << 24) - 1):
    norm_grad(m, 8200); norm_grad(m, 20000, 1, dg=False)
print(json.dumps([e[3] for e in launches() if "norm_stats" in e[3]]))
""")
    grids = [int(e.split(" ")[0]) for e in seen]
    assert len(grids) == 10 and min(grids) == 1 and all(g * 1024 < 1 << 32 for g in grids), grids
