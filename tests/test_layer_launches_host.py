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


def test_logits_of_any_number_of_rows(run):
    """Rows without values go through their logits whatever their number: logit_parts_kernel's second side."""
    for m, n, parts in ((65535, 5, 1), (65536, 5, 1), (1 << 20, 5000, 2), ((1 << 24) - 1, 1, 1)):
        seen = run(CODE + """
import json
loss(%d, 0, %d)
print(json.dumps([e[3] for e in launches() if "logit_parts" in e[3]]))
""" % (m, n))
        rows = [int(e.split(" ")[0]) // parts for e in seen]
        assert sum(rows) == m and max(rows) <= 65535, rows
