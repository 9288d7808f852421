"""Sizes that large calls' kernels take on 256 compute units, with remainders in every
dimension, and what the library plans for them."""

#: (m, n, k), tile of the forward product
LARGE_PRODUCTS = [((1500, 3000, 1000), (256, 128)), ((6541, 560, 552), (256, 128)), ((6971, 1760, 720), (256, 256)),
                  ((2942, 4272, 760), (256, 256))]

#: (m, n, k), part, its tile, whether k is split
LARGE_GRADIENTS = [((6541, 560, 552), "da", (256, 128), False), ((4103, 5416, 152), "da", (256, 128), True),
                   ((4964, 728, 2440), "da", (256, 256), False), ((570, 5776, 656), "db", (256, 128), False),
                   ((4902, 4464, 144), "db", (256, 128), True), ((739, 7608, 1688), "db", (256, 256), False)]

#: batch, heads, key heads, lq, lk, dim, mask: each row has a wave of its own, in the
#: forward pass and in dq
FULL_CHIP = [(40, 8, 8, 130, 130, 64, {}), (34, 24, 8, 150, 150, 80, dict(window=60, sinks=4)),
             (66, 16, 4, 70, 300, 128, dict(window=90, sinks=9)), (290, 1, 1, 257, 257, 40, dict(window=1, sinks=1)),
             (9, 8, 8, 1000, 1000, 96, dict(window=200, sinks=130)), (33, 40, 8, 90, 90, 128, {})]
