"""Calls of the layer for a few tokens that reach every gate_up kernel of it, and the rule by which a call takes one."""
import math

F32, F16, BF16, F8, I8 = 0, 1, 30, 256, 24
KINDS, X_TYPES = (F8, I8, F16, BF16), (F32, F16, BF16)
E, K = 40, 8


def one_byte(kind):
    return kind in (F8, I8)


def most_entries(x_type):
    return 5 if x_type == F32 else 8


def loads(kind, x_type, entries):
    """A step's loads of the activations of so many entries."""
    values = 128 if one_byte(kind) else 64
    pieces = values * (4 if x_type == F32 else 2) // 16
    return -(-entries * pieces // 64)


def row_tiles(tokens, inter):
    """Those that the call is expected to have."""
    return max(1.0, E * (1 - (1 - K / E) ** tokens)) * (-(-inter // 16))


def kernel(kind, x_type, tokens, inter):
    """(loads of activations, waves that share a row tile, row tiles a wave) of a call."""
    tiles = row_tiles(tokens, inter)
    share = 1 if tiles > 1024 else (2 if tiles > 512 else 4)
    return loads(kind, x_type, min(most_entries(x_type), tokens)), share, max(1, min(4, math.ceil(tiles / 2048 - 0.25))) if share == 1 else 1


def cases():
    """(kind, x_type, tokens, hidden, inter): every number of loads with every sharing and one tile a wave, and two to four tiles a wave. Hidden widths and
    depths that end inside a step; a wave of the shared ones may have no step at all; the last workgroup has fewer tiles than the others."""
    for kind in KINDS:
        for x_type in X_TYPES:
            seen = set()
            for tokens, tiles in [(t, n) for t in (2, 4, 7) for n in (300, 800, 1500)] + [(7, 3400), (16, 5500), (16, 8000)]:
                inter = 16 * math.ceil(tiles / row_tiles(tokens, 16))
                found = kernel(kind, x_type, tokens, inter)
                if found in seen:
                    continue
                seen.add(found)
                hidden = (272 if tiles <= 1024 else 144) - (0 if one_byte(kind) else 8)
                yield kind, x_type, tokens, hidden, inter - (0 if one_byte(kind) else 8)
