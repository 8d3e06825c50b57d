"""Problems for which the attention's host side picks each layout of its kernels, and the layout it picks (mia_relpos_plan): a test of a
variant says so when the rule moves away from it."""
import ctypes

import mia_amd

FORWARD, QUERIES, KEYS = range(3)
F32, BF16 = 0, 1


def layout(direction, dtype, B, heads, Lq, Lk, D):
    """-> (columns of a wave, whether the walk is split, heads of a workgroup of the few-query forward)"""
    plan = (ctypes.c_int * 3)()
    mia_amd.lib().mia_relpos_plan(direction, dtype, B, heads, Lq, Lk, D, plan)
    return plan[0], plan[1] > 1, plan[2]


# (dtype, B, heads, Lq, Lk, D, height, width, q_start): {direction: layout}
TWO = {FORWARD: (2, False, 0), QUERIES: (2, False, 0), KEYS: (2, False, 0)}
VARIANTS = {
    # the default head at a training batch, and maps of several tiles with ends inside one
    (BF16, 128, 8, 100, 100, 48, 10, 10, 0): TWO,
    (BF16, 97, 2, 210, 210, 16, 7, 30, 0): {QUERIES: (2, False, 0), KEYS: (2, False, 0)},
    (BF16, 97, 2, 210, 210, 32, 30, 7, 0): {QUERIES: (2, False, 0), KEYS: (2, False, 0)},
    (BF16, 97, 2, 210, 210, 48, 2, 105, 0): TWO,
    (BF16, 97, 2, 210, 210, 64, 1, 210, 0): TWO,
    (BF16, 97, 2, 210, 150, 96, 14, 15, 0): {FORWARD: (2, False, 0)},
    # two columns and a split walk: over the keys, over the queries
    (BF16, 43, 3, 70, 1500, 16, 30, 50, 700): {QUERIES: (2, True, 0)},
    (BF16, 43, 3, 70, 1500, 32, 1, 1500, 1430): {QUERIES: (2, True, 0)},
    (BF16, 43, 3, 70, 1500, 48, 30, 50, 20): {FORWARD: (2, True, 0), QUERIES: (2, True, 0)},
    (BF16, 43, 3, 70, 1500, 64, 3, 500, 1300): {FORWARD: (2, True, 0), QUERIES: (2, True, 0)},
    (BF16, 11, 5, 70, 2000, 96, 40, 50, 100): {FORWARD: (2, True, 0)},
    (BF16, 13, 5, 2000, 70, 16, 40, 50, 0): {KEYS: (2, True, 0)},
    (BF16, 13, 5, 2000, 70, 32, 1, 2000, 0): {KEYS: (2, True, 0)},
    (BF16, 49, 2, 1000, 70, 48, 20, 50, 0): {KEYS: (2, True, 0)},
    (BF16, 49, 2, 1000, 70, 64, 500, 2, 0): {KEYS: (2, True, 0)},
    # one column
    (BF16, 2, 3, 130, 200, 64, 10, 20, 50): {FORWARD: (1, False, 0), QUERIES: (1, False, 0), KEYS: (1, False, 0)},
    (F32, 2, 3, 130, 200, 32, 10, 20, 50): {FORWARD: (1, False, 0), QUERIES: (1, False, 0), KEYS: (1, False, 0)},
    (BF16, 1, 1, 1100, 1100, 24, 22, 50, 0): {FORWARD: (1, True, 0), QUERIES: (1, True, 0), KEYS: (1, True, 0)},
    (F32, 1, 1, 1100, 1100, 24, 22, 50, 0): {FORWARD: (1, True, 0), QUERIES: (1, True, 0), KEYS: (1, True, 0)},
    # at most 16 queries: waves on one head or on neighbouring ones, one range of the keys or several
    (BF16, 3, 2, 16, 300, 64, 1, 320, 300): {FORWARD: (0, False, 1)},
    (F32, 3, 2, 16, 300, 48, 1, 320, 300): {FORWARD: (0, False, 1)},
    (BF16, 2, 8, 16, 4100, 64, 1, 4116, 4100): {FORWARD: (0, True, 1)},
    (F32, 2, 4, 16, 2100, 48, 1, 2116, 2100): {FORWARD: (0, True, 1)},
    (BF16, 5000, 2, 1, 70, 16, 7, 10, 69): {FORWARD: (0, False, 2)},
    (F32, 600, 4, 1, 200, 16, 10, 20, 77): {FORWARD: (0, False, 4)},
    (BF16, 24, 6, 2, 4100, 64, 1, 4102, 4100): {FORWARD: (0, True, 2)},
    (BF16, 18, 8, 2, 4100, 64, 1, 4102, 4100): {FORWARD: (0, True, 4)},
    (F32, 18, 8, 2, 4100, 40, 1, 4102, 4100): {FORWARD: (0, True, 4)},
}
