"""Sizes of the gated linear that between them go by every kernel it has: each
kind of tiles, with tiles that are whole, split along the contraction, or some of
each, in either precision of the slopes, in one launch of both gradients and in
two."""

import bfhip

# (rows, features, hidden), found among random sizes: few of them, and small ones.
HALF = [(9, 9, 11), (9, 9, 211), (23, 9, 731), (55, 9, 309), (135, 2043, 11268), (203, 8633, 1), (273, 11, 9), (324, 5584, 530),
        (405, 3550, 1674), (581, 1583, 3331), (614, 6576, 707), (694, 970, 8321), (786, 2700, 27), (929, 271, 11069),
        (1250, 4736, 832), (1288, 3233, 1161), (1363, 272, 10926), (1380, 1, 8514), (1504, 2471, 1660), (1914, 4439, 489),
        (1947, 10, 9), (2111, 1, 8697), (2761, 66, 2190), (2853, 1, 4676), (5578, 4390, 1), (5627, 5417, 80), (6570, 1, 1865),
        (6584, 1207, 431), (6817, 376, 2380), (8669, 1921, 436), (10288, 3779, 1), (17482, 151, 1000), (17483, 1, 556),
        (17744, 1223, 1), (17878, 137, 1317), (19309, 9, 9)]
SINGLE = [(9, 9, 11), (66, 5817, 292), (170, 9, 10), (174, 407, 8703), (179, 8690, 430), (198, 8367, 473), (203, 11, 70),
          (203, 8633, 1), (298, 226, 6869), (558, 8791, 450), (706, 165, 5490), (715, 5431, 131), (891, 8589, 417),
          (1034, 8384, 576), (1102, 7592, 175), (2659, 3126, 67), (6244, 1, 316), (17277, 174, 104), (19309, 9, 9)]


def paths(dtype, size):
    """Names of the kernels that a call of this size and its gradients go by."""
    plans = {p: bfhip.gated_plan(dtype, *size, p) for p in ("forward", "inputs", "weights")}
    tiles = {p: (q.kind, q.whole > 0, q.split > 0) for p, q in plans.items()}
    two = plans["inputs"].two_parts
    found = {("forward", tiles["forward"])} | {(p, tiles[p], two) for p in ("inputs", "weights")}
    if plans["inputs"].together:
        found.add(("both", tiles["inputs"], tiles["weights"], two))
    return found
