"""Sizes of products on 8-bit integers that take every form of the kernels, deep enough that its stages come round:
whole tiles, ragged ones, and an end of 48 or 80 codes."""

# name, groups of waves, stages of a group
FORMS = [("I8_STREAM_16", 8, 2), ("I8_STREAM_32", 8, 2), ("I8_64x128", 1, 3), ("I8_128x128", 1, 2), ("I8_128x256", 1, 2),
         ("I8_256x256", 1, 2), ("I8_32x32", 8, 2), ("I8_32x64", 4, 3), ("I8_64x64_DEEP", 1, 4), ("I8_64x64", 1, 2),
         ("I8_128x256_DEEP", 1, 3)]

# form, gated, tokens, channels, depth
DEEP = [
    ("I8_STREAM_16", 0, 17, 70, 4144), ("I8_STREAM_32", 0, 33, 1400, 4144), ("I8_64x128", 0, 190, 16390, 1040),
    ("I8_128x128", 0, 130, 12290, 560), ("I8_128x256", 0, 130, 16390, 560), ("I8_128x256_DEEP", 0, 210, 16390, 4176),
    ("I8_256x256", 0, 390, 16390, 560), ("I8_32x32", 0, 130, 100, 4144), ("I8_32x64", 0, 33, 4100, 2608),
    ("I8_64x64_DEEP", 0, 66, 6150, 1104), ("I8_64x64", 0, 130, 260, 560),
    ("I8_STREAM_16", 1, 17, 70, 4144), ("I8_STREAM_32", 1, 33, 1400, 4144), ("I8_64x128", 1, 130, 390, 688),
    ("I8_128x128", 1, 130, 6150, 560), ("I8_128x256", 1, 130, 8200, 560), ("I8_128x256_DEEP", 1, 130, 12290, 4176),
    ("I8_256x256", 1, 260, 12290, 560),
]
