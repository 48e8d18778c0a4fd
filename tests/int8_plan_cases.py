"""Sizes at which products of 8-bit integers take each of their kernels, with
columns that fill the tiles and with ragged ones.  ``test_int8_plans.py``
checks on the CPU that they do; ``test_int8_plans_gpu.py`` runs them."""

FEW, T64, T64X128, T128_DEEP, T128X256, T128, T256 = range(7)

# (rows, columns of a row, columns of the result, shape, shares of K)
PRODUCTS = [
    (1, 300, 77, FEW, 1), (3, 200, 3001, FEW, 1), (9, 130, 2600, FEW, 1), (30, 257, 90, FEW, 1), (64, 400, 128, FEW, 1),
    (65, 300, 128, T64, 1), (200, 1000, 333, T64, 1), (70, 5100, 192, T64, 2), (65, 7600, 77, T64, 3), (100, 10200, 320, T64, 4),
    (130, 20000, 67, T64, 4),
    (200, 130, 8192, T64X128, 1), (300, 90, 5003, T64X128, 1),
    (509, 200, 5003, T128_DEEP, 1), (1000, 400, 4096, T128_DEEP, 1), (513, 65, 6001, T128_DEEP, 1),
    (1100, 300, 5120, T128X256, 1), (1025, 129, 4999, T128X256, 1),
    (4000, 130, 4480, T128, 1), (4097, 100, 4097, T128, 1),
    (2048, 130, 4352, T256, 1), (2047, 385, 4200, T256, 1),
]

# (rows, columns of a row, hidden columns, columns of the result, shape of gate and up, shares of K)
GATED = [
    (1, 300, 70, 50, FEW, 1), (4, 129, 700, 33, FEW, 1), (17, 200, 160, 64, FEW, 1), (33, 385, 90, 77, FEW, 1),
    (65, 300, 64, 48, T64, 1), (150, 1000, 301, 60, T64, 1), (70, 7168, 300, 129, T64, 2), (65, 7600, 128, 40, T64, 3),
    (130, 10200, 97, 40, T64, 4), (40, 14000, 2100, 40, T64, 3),
    (190, 90, 4480, 50, T64X128, 1), (300, 130, 3001, 70, T64X128, 1),
    (600, 130, 3200, 64, T128_DEEP, 1), (513, 200, 3001, 50, T128_DEEP, 1),
    (1100, 90, 3328, 70, T128X256, 1), (1025, 200, 3001, 50, T128X256, 1),
    (1281, 130, 5632, 70, T128, 1), (1281, 200, 5601, 130, T128, 1),
    (2100, 100, 2176, 60, T256, 1), (2049, 257, 2201, 70, T256, 1),
]

# few rows at both sides of the rule between eight and sixteen waves (rows, columns of a row, columns of the result)
WAVES = [(rows, k, n) for rows in (1, 4, 5, 8, 9, 16, 17, 32, 33, 64) for k, n in ((1536, 100), (1537, 100), (2200, 4096), (1600, 4097))]
