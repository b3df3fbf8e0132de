"""Sizes that reach every kernel of the int8 product and of the attention over the 8-bit cache.  The host test checks that they still do, the device
tests run them."""

# kernel, slices of k, rows, columns, k
PRODUCTS = [
    ("rows", 1, 5, 1030, 700), ("rows", 1, 30, 520, 1285), ("rows", 1, 61, 1030, 640),
    ("tile", 1, 129, 1030, 100), ("tile", 1, 384, 5176, 1000), ("tile", 1, 257, 700, 640), ("tile", 1, 200, 515, 2048),
    ("tile", 2, 70, 130, 2500), ("tile", 2, 300, 2048, 4500), ("tile", 4, 100, 2048, 6144), ("tile", 4, 129, 515, 4500), ("tile", 8, 70, 140, 9000),
    ("tile128", 1, 512, 5176, 100), ("tile128", 1, 385, 4900, 200), ("tile128", 1, 385, 4900, 1285), ("tile128", 1, 3000, 1190, 700), ("tile128", 1, 240, 12288, 2048),
    ("big", 1, 2050, 8301, 100), ("big", 1, 2050, 8301, 256), ("big", 1, 2050, 8301, 640), ("big", 1, 2050, 8301, 1285), ("big", 1, 3000, 4096, 1290),
    ("big", 1, 1024, 12288, 700),
]
PRODUCT_PAST_THE_CACHES = (8200, 8301, 700)          # more than 256 MiB of float32: other stores in the big kernel

# sequences, new rows, positions, heads, queries per head, dim -> 16-row blocks (0: the 128-row kernel), waves, parts
ATTENTION = {
    "four_waves": ((3, 1, 120, 2, 2), (1, 4, 1)),
    "eight_waves": ((3, 2, 700, 2, 2), (1, 8, 1)),
    "parts": ((2, 1, 2500, 1, 4), (1, 4, 7)),
    "two_blocks": ((2, 20, 300, 2, 1), (2, 4, 1)),
    "two_blocks_parts": ((2, 20, 1300, 1, 1), (2, 4, 6)),
    "many_rows": ((26, 70, 110, 10, 1), (0, 4, 1)),
}
