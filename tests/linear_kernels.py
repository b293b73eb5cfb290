"""Shapes of linear layers by the kernel that takes them on 256 CUs: tests/test_linear_routes.py holds the names to what dc_linear_route.hpp
picks, tests/test_gpu_linear_kernels.py runs them. Sides that no tile divides, three turns and more along the sums where the
kernel is not for few.

A name is a tile's side, x and its groups of waves, and /split where workgroups share the sums (for both gradients in one launch: /a for
dx, /b for dw); few and its blocks of 8 rows of x, fewwide with 64 outputs a workgroup; any, for rows read as they lie.
"""
FORWARD = [
    ("any", 3, 70, 201, "bf16"), ("any", 5, 33, 401, "fp8"),
    ("few1", 5, 70, 200, "bf16"), ("few2", 12, 70, 208, "bf16"), ("few3", 21, 70, 200, "bf16"), ("few4", 30, 35, 200, "bf16"),
    ("few8", 61, 70, 200, "bf16"), ("few8", 300, 300, 1001, "bf16"),
    ("few1", 5, 70, 400, "fp8"), ("few2", 12, 70, 432, "fp8"), ("few3", 21, 70, 400, "fp8"), ("few4", 30, 35, 432, "fp8"),
    ("few8", 61, 70, 400, "fp8"), ("few8", 300, 300, 1001, "fp8"),
    ("fewwide1", 5, 8401, 200, "bf16"), ("fewwide2", 12, 8437, 208, "bf16"), ("fewwide3", 21, 8644, 208, "bf16"),
    ("fewwide4", 30, 8247, 208, "bf16"),
    ("fewwide1", 5, 8485, 400, "fp8"), ("fewwide2", 12, 8713, 448, "fp8"), ("fewwide3", 21, 8769, 448, "fp8"),
    ("fewwide4", 30, 8494, 400, "fp8"),
    ("64", 197, 1059, 202, "bf16"), ("64/split", 130, 1415, 1287, "bf16"), ("64x2", 397, 578, 470, "bf16"),
    ("64x2/split", 745, 400, 2351, "bf16"), ("64x4", 259, 830, 1164, "bf16"), ("128", 2916, 1351, 327, "bf16"),
    ("128/split", 841, 894, 3690, "bf16"), ("128x2", 680, 4691, 840, "bf16"), ("128x2/split", 339, 729, 8945, "bf16"),
    ("256", 2131, 4802, 202, "bf16"),
    ("64", 264, 817, 425, "fp8"), ("64/split", 337, 680, 3089, "fp8"), ("64x2", 391, 603, 907, "fp8"),
    ("64x2/split", 459, 664, 4613, "fp8"), ("64x4", 394, 577, 2335, "fp8"), ("128", 4051, 966, 680, "fp8"),
    ("128/split", 839, 833, 6886, "fp8"), ("128x2", 5178, 593, 1666, "fp8"), ("128x2/split", 1473, 648, 5963, "fp8"),
    ("256", 4185, 2499, 401, "fp8"),
]
LARGE = [("256/split", 6587, 528, 6285, "bf16")]
# both gradients: m, n, k
PAIRS = [
    ("64", 140, 147, 9), ("64/a", 141, 780, 9), ("64/b", 781, 140, 9), ("64/a/b", 193, 774, 11), ("64x2", 196, 140, 8),
    ("64x2/a", 205, 1024, 181), ("64x2/b", 5233, 140, 8), ("64x2/a/b", 1386, 648, 73), ("128", 197, 193, 6159), ("128/a", 322, 2226, 921),
    ("128/b", 2203, 329, 932), ("128/a/b", 2699, 2824, 74), ("256", 403, 401, 8490), ("256/a", 149, 4666, 1808), ("256/b", 4183, 141, 1928),
    ("256/a/b", 7475, 2023, 130),
]
# one gradient: its rows, the length of its sums, its columns
SINGLES = [
    ("64", 130, 258, 72), ("64/split", 33, 2049, 72), ("64x2", 130, 650, 232), ("64x2/split", 65, 5178, 72), ("64x4", 314, 979, 234),
    ("64x4/split", 193, 8629, 265), ("128", 1100, 259, 2721), ("128/split", 5482, 3767, 132), ("128x2", 2333, 202, 1282),
    ("128x2/split", 769, 4363, 592), ("256", 1537, 207, 5026), ("256/split", 140, 8196, 4120),
]
