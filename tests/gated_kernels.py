"""Shapes of gated layers by the kernel that takes them on 256 CUs: tests/test_gated_routes.py holds the names to what dc_hip_gated_linear and its
backward call pick, tests/test_gpu_gated_kernels.py runs them. Names as in tests/linear_kernels.py, a tile's side counting both weights' rows; for the
gradients /a where workgroups share dx's sums, /b where they share the weights'."""
FORWARD = [
    ("few1", 1, 62, 198, "bf16"), ("few2", 10, 64, 195, "bf16"), ("few3", 18, 60, 202, "bf16"), ("few4", 26, 60, 214, "bf16"),
    ("few8", 35, 60, 196, "bf16"), ("few8", 276, 415, 199, "bf16"), ("64", 445, 578, 197, "bf16"), ("64/split", 326, 677, 2372, "bf16"), ("64x2", 612, 405, 450, "bf16"),
    ("64x2/split", 451, 612, 2594, "bf16"), ("64x4", 455, 522, 1188, "bf16"), ("128", 1499, 1341, 387, "bf16"),
    ("128/split", 321, 805, 4671, "bf16"), ("128x2", 851, 1809, 982, "bf16"), ("128x2/split", 398, 896, 3924, "bf16"),
    ("256", 1348, 3742, 193, "bf16"), ("256/split", 138, 5807, 7230, "bf16"),
    ("few1", 3, 60, 397, "fp8"), ("few2", 11, 60, 387, "fp8"), ("few3", 19, 62, 419, "fp8"), ("few4", 29, 63, 392, "fp8"),
    ("few8", 39, 60, 392, "fp8"), ("few8", 212, 541, 398, "fp8"), ("64", 390, 595, 391, "fp8"), ("64/split", 327, 713, 4630, "fp8"), ("64x2", 386, 605, 898, "fp8"),
    ("64x2/split", 326, 747, 5356, "fp8"), ("64x4", 675, 375, 2348, "fp8"), ("128", 1660, 1937, 395, "fp8"),
    ("128/split", 214, 1593, 6659, "fp8"), ("128x2", 783, 2069, 1755, "fp8"), ("128x2/split", 758, 687, 6558, "fp8"),
    ("256", 1767, 2989, 406, "fp8"),
]
FORWARD += [(name, m, n, k, "blocks") for name, m, n, k, dtype in FORWARD if dtype == "fp8"]
# Products with block scales of few rows: 32 outputs to a workgroup, of eight waves and of four (m, n, k)
BLOCKS = [(5, 4109, 400), (12, 4133, 432), (21, 4201, 400), (30, 4150, 432), (7, 8301, 400), (12, 8437, 208), (21, 8644, 1300), (30, 8247, 2211)]
# m, n, k
GRADIENTS = [
    ("64", 33, 62, 200), ("64/a", 1, 410, 8), ("64/b", 812, 4, 8), ("64/a/b", 772, 66, 10), ("64x2", 1, 65, 8), ("64x2/a", 1, 2044, 8),
    ("64x2/b", 5378, 3, 8), ("64x2/a/b", 398, 636, 125), ("128", 199, 74, 7187), ("128/a", 66, 876, 2073), ("128/b", 2195, 139, 1022),
    ("128/a/b", 2739, 1557, 69), ("256", 399, 221, 8727), ("256/a", 129, 2761, 1597), ("256/b", 2564, 69, 2988),
    ("256/a/b", 2137, 4299, 131),
]
