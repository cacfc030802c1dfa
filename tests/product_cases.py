"""Calls of the grouped product that reach every kernel of it, for each kind of sums.

A case: weight and output type, the kernel it is for, groups, the rows they have on average, weight rows and k. The depths
end inside a step of 128 bytes."""
F32, F16, BF16, F8 = 0, 1, 30, 256
KINDS = {(F8, F32): 0, (F8, F16): 0, (F8, BF16): 1, (F16, F16): 2, (BF16, F32): 3}   # the sums: exact, FP8 instruction, fp16, bf16
TYPES = list(KINDS)

# kernel -> groups, rows a group on average, weight rows, bytes of k
FEW = {
    "few8": (5, 3, 200, 2096),
    "few16": (6, 8, 200, 1040),
    "stream8_4": (256, 3, 250, 1296),
    "stream16_4": (140, 7, 481, 1680),
}
# deeper ones: 16 rows of 4096 tiles; FP8 and 16-bit have room for different depths
DEEP = {
    "stream8_8": (1024, 3, 49, {8: 5520, 16: 6032}),
    "stream16_8": (1024, 7, 49, {8: 4112, 16: 5776}),
    "few8 past LDS": (1024, 2, 49, {8: 8208, 16: 12048}),
    "few16 past LDS": (1024, 5, 49, {8: 5648, 16: 6032}),
}
MANY = {
    "tile64x32": (3, 21, 200, 3216),
    "tile128x64": (80, 30, 250, 1040),
    "tile256x128": (20, 100, 1790, 1296),
    "tile256x256": (20, 110, 2000, 1296),
    "tile256x160": (10, 210, 1990, 1552),
}


def cases():
    for types in TYPES:
        bits = 8 if types[0] == F8 else 16
        for name, (groups, mean, rows, k_bytes) in {**FEW, **DEEP, **MANY}.items():
            if KINDS[types] == 0 and name in ("tile256x256", "tile256x160"):
                continue                                # no such tiles for exact FP8 sums
            k_bytes = k_bytes[bits] if isinstance(k_bytes, dict) else k_bytes
            yield types, name, groups, mean, rows, k_bytes if bits == 8 else k_bytes // 2
