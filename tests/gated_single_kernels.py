"""Shapes of a gated layer's gradients asked for by themselves, by the kernel that takes them on 256 CUs: (which, kernel, m, n, k), `which` being dx, one
weight's or both weights' gradients. tests/test_gated_single_routes.py holds the names to what dc_hip_gated_linear_backward picks,
tests/test_gpu_gated_single_kernels.py runs them. Names as in tests/linear_kernels.py. No side is whole vectors or tiles; dx's groups of waves stand on both
sides of the border between the two weights' halves of c.
"""
SINGLES = [
    ("dx", "128", 323, 17, 8413), ("dx", "128/split", 131, 1908, 5595), ("dx", "128x2", 2884, 130, 1027), ("dx", "128x2/split", 795, 2186, 614),
    ("dx", "256", 898, 69, 8281), ("dx", "256/split", 133, 4062, 4188), ("dx", "64", 17, 17, 17), ("dx", "64/split", 17, 395, 17),
    ("dx", "64x2", 18, 133, 17), ("dx", "64x2/split", 17, 2586, 17), ("dx", "64x4", 510, 580, 322), ("dx", "64x4/split", 17, 7242, 17),
    ("dw", "128", 23, 7374, 450), ("dw", "128/split", 3610, 5482, 129), ("dw", "128x2", 195, 1538, 1937), ("dw", "128x2/split", 4274, 1359, 321),
    ("dw", "256", 67, 8002, 1156), ("dw", "256/split", 6143, 129, 5660), ("dw", "64", 17, 17, 17), ("dw", "64/split", 770, 17, 17),
    ("dw", "64x2", 199, 17, 17), ("dw", "64x2/split", 5236, 17, 17), ("dw", "64x4", 970, 293, 254), ("dw", "64x4/split", 4999, 291, 385),
    ("dws", "128", 17, 7582, 198), ("dws", "128/split", 3602, 2779, 129), ("dws", "128x2", 195, 1222, 1222), ("dws", "128x2/split", 4332, 292, 773),
    ("dws", "256", 71, 6701, 649), ("dws", "256/split", 8869, 2050, 129), ("dws", "64", 17, 17, 17), ("dws", "64/split", 801, 17, 17),
    ("dws", "64x2", 195, 17, 17), ("dws", "64x2/split", 5302, 17, 18), ("dws", "64x4", 982, 201, 183), ("dws", "64x4/split", 5059, 282, 193),
]
