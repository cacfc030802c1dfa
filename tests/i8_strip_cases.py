"""Grouped integer products whose groups have more token tiles than a strip holds, several row tiles, and a last strip that is not a whole one."""
# kernel -> rows a group, weight rows, k
CASES = {
    "tile64x32": ([0, 310, 290], 200, 400),
    "tile128x64": ([1500, 2700, 20], 600, 144),
    "tile256x128": ([3, 1500, 497] + 17 * [0], 1790, 272),
    "tile256x256": ([5, 2100, 95] + 17 * [0], 2000, 144),
    "tile256x160": ([3000, 1400, 10, 2050], 2000, 144),
}
