"""Cases of the scaled operators, each named by its operator, rows, inputs, outputs, floating type and kind
of rows (floating, or int8 with scales). Together they launch every kernel that the operators have, which
test_scaled_launches_host.py checks, and the GPU tests compare each with its definition.

COVER: sizes found by search, the cheapest that reach a kernel. SLICES: few rows, K in slices, column
groups of every width. SHORT: more than 64 rows over K of at most 128. LAYERS: sizes of real layers."""

COVER = [
    ("linear", 1, 607, 8562, "f16", "i8"), ("linear", 1, 608, 4738, "f32", "float"),
    ("linear", 1, 611, 4150, "bf16", "float"), ("linear", 1, 612, 12980, "bf16", "float"),
    ("linear", 1, 612, 4100, "bf16", "i8"), ("linear", 1, 615, 20, "f32", "float"),
    ("linear", 1, 617, 12356, "f32", "float"), ("linear", 1, 619, 8921, "f32", "float"),
    ("linear", 1, 630, 12578, "f32", "i8"), ("linear", 1, 631, 21, "f16", "float"),
    ("linear", 1, 645, 8365, "bf16", "float"), ("linear", 1, 17867, 20, "f32", "float"),
    ("linear", 14, 1055, 20, "f32", "float"), ("linear", 17, 613, 12665, "f32", "i8"),
    ("linear", 17, 652, 4116, "bf16", "i8"), ("linear", 17, 685, 8197, "bf16", "float"),
    ("linear", 18, 626, 20, "f32", "float"), ("linear", 33, 626, 4311, "f32", "float"),
    ("linear", 33, 641, 8564, "f16", "float"), ("linear", 33, 671, 21, "bf16", "float"),
    ("linear", 34, 629, 12417, "f16", "float"), ("linear", 50, 618, 8945, "f32", "i8"),
    ("linear", 52, 607, 21, "bf16", "float"), ("linear", 52, 636, 4319, "bf16", "i8"),
    ("linear", 58, 622, 12274, "f16", "i8"), ("linear", 65, 151, 22, "f16", "i8"),
    ("linear", 67, 70, 21, "f32", "i8"), ("linear", 199, 773, 18554, "f32", "i8"),
    ("linear", 389, 428, 16272, "f32", "float"), ("linear", 523, 9034, 22, "f32", "float"),
    ("linear", 525, 4177, 22, "f16", "float"), ("linear", 533, 11198, 20, "bf16", "float"),
    ("linear", 611, 4346, 22, "f32", "float"), ("linear", 1413, 412, 10362, "f16", "float"),
    ("linear", 1645, 392, 8993, "f32", "float"), ("linear", 2822, 387, 2493, "bf16", "i8"),
    ("gated", 1, 606, 4138, "f32", "i8"), ("gated", 1, 626, 4590, "bf16", "float"),
    ("gated", 1, 629, 4384, "f32", "float"), ("gated", 1, 646, 20, "bf16", "float"),
    ("gated", 1, 16505, 20, "bf16", "float"), ("gated", 1, 17698, 23, "f16", "float"),
    ("gated", 2, 609, 20, "f32", "float"), ("gated", 4, 4117, 21, "bf16", "float"),
    ("gated", 4, 4149, 20, "f32", "float"), ("gated", 4, 4215, 21, "f16", "float"),
    ("gated", 13, 1037, 21, "f16", "float"), ("gated", 13, 1058, 23, "bf16", "float"),
    ("gated", 17, 627, 4320, "f16", "i8"), ("gated", 17, 685, 20, "bf16", "i8"),
    ("gated", 34, 603, 21, "f16", "float"), ("gated", 35, 631, 4286, "f32", "i8"),
    ("gated", 55, 614, 4223, "f32", "float"), ("gated", 55, 630, 21, "f16", "float"),
    ("gated", 69, 833, 17527, "f32", "float"), ("gated", 70, 77, 20, "f16", "i8"),
    ("gated", 73, 130, 20, "f16", "float"), ("gated", 530, 9968, 22, "f16", "float"),
    ("gated", 558, 4859, 21, "bf16", "float"), ("gated", 659, 395, 5117, "bf16", "float"),
    ("gated", 722, 403, 10263, "f32", "i8"), ("gated", 1194, 387, 6274, "bf16", "float"),
    ("gated", 1938, 396, 1839, "f32", "float"), ("linear_grad", 1, 65, 17343, "f16", "float"),
    ("linear_grad", 1, 65, 16480, "f32", "float"), ("linear_grad", 1, 65, 8788, "f16", "float"),
    ("linear_grad", 1, 65, 4262, "bf16", "float"), ("linear_grad", 1, 65, 1038, "f16", "float"),
    ("linear_grad", 1, 66, 16478, "bf16", "float"), ("linear_grad", 1, 67, 1122, "bf16", "float"),
    ("linear_grad", 1, 68, 1121, "f32", "float"), ("linear_grad", 1, 69, 4097, "f32", "float"),
    ("linear_grad", 1, 70, 20, "f32", "float"), ("linear_grad", 1, 72, 8515, "bf16", "float"),
    ("linear_grad", 1, 73, 21, "bf16", "float"), ("linear_grad", 2, 66, 4161, "f16", "float"),
    ("linear_grad", 2, 67, 8421, "f32", "float"), ("linear_grad", 2, 68, 20, "f16", "float"),
    ("gated_grad", 1, 70, 20, "bf16", "i8"), ("gated_grad", 71, 769, 17616, "f16", "float"),
    ("gated_grad", 128, 2152, 36, "f16", "float"), ("gated_grad", 471, 130, 7554, "f32", "i8"),
    ("gated_grad", 752, 137, 10493, "bf16", "float"), ("gated_grad", 964, 169, 8114, "f16", "float"),
    ("gated_grad", 1931, 132, 1975, "f16", "float"), ("gated_grad", 3295, 1030, 34, "f16", "i8"),
    ("gated_grad", 3538, 149, 2201, "f32", "float"), ("gated_grad", 5113, 2324, 20, "f32", "i8"),
    ("gated_grad", 5469, 138, 668, "bf16", "float"),
]

SLICES = [
    ("linear", 2, 8192, 4096, "bf16", "float"), ("linear", 4, 4096, 4500, "f32", "float"),
    ("linear", 9, 8192, 6200, "f16", "i8"), ("linear", 16, 8192, 4096, "bf16", "float"),
    ("linear", 40, 6000, 5000, "bf16", "float"), ("linear", 64, 8192, 4300, "f32", "float"),
    ("linear", 64, 4100, 9000, "f16", "i8"), ("gated", 3, 5000, 2500, "f32", "float"),
    ("gated", 12, 8192, 2500, "bf16", "float"), ("gated", 50, 8000, 2300, "f16", "float"),
    ("gated", 64, 4096, 4000, "f32", "i8"),
]

SHORT = [
    ("linear", 200, 100, 3000, "bf16", "float"), ("linear", 65, 128, 64, "f32", "float"),
    ("linear", 3000, 64, 70, "f16", "i8"), ("gated", 200, 100, 3000, "f16", "float"),
    ("gated", 900, 127, 65, "f32", "i8"),
]

LAYERS = [
    ("linear", 1, 4096, 14336, "bf16", "float"), ("linear", 1, 4096, 14336, "f32", "float"),
    ("linear", 16, 4096, 11008, "f16", "float"), ("linear", 48, 14336, 4096, "f16", "float"),
    ("linear", 1024, 4096, 4096, "bf16", "float"), ("linear", 400, 4096, 11008, "f32", "i8"),
    ("linear", 2048, 2048, 2048, "f16", "float"), ("linear", 1100, 1024, 3800, "bf16", "float"),
    ("gated", 1, 4096, 14336, "bf16", "float"), ("gated", 32, 4096, 14336, "bf16", "float"),
    ("gated", 16, 2048, 8192, "f32", "float"), ("gated", 1000, 2048, 2816, "bf16", "float"),
    ("gated", 500, 1024, 5500, "f32", "float"), ("linear_grad", 1024, 4096, 4096, "f32", "float"),
    ("linear_grad", 2048, 2048, 2048, "f16", "float"), ("gated_grad", 500, 2048, 2816, "f32", "float"),
    ("gated_grad", 1000, 1024, 2816, "bf16", "i8"), ("gated_grad", 700, 1024, 2300, "f16", "float"),
]

CASES = COVER + SLICES + SHORT + LAYERS
