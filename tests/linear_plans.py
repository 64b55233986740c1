"""Sizes that reach every kernel, tile and split that the linear layers' products can take, and how to ask which that is.

A product's plan is (product, pair, rows of a tile, split, more tiles than pairs of SMs); product 0 is the forward one, 1
dX, 2 dW.  SIZES (tokens, k, n) were chosen so that each plan met among 400000 layers of 1 to 8192 tokens and 64 to 16384
features is some size's; test_linear_plans.py fails where the choice has moved away from them.
"""
import ctypes

from chpl_b200 import _lib

SIZES = [
    (1, 64, 64), (1, 656, 1600), (1, 1960, 1944), (2480, 64, 64), (1, 4304, 4232), (17, 976, 2432), (4845, 144, 64),
    (590, 1440, 64), (900, 64, 1112), (631, 64, 1880), (1083, 1672, 64), (18, 4832, 1840), (275, 64, 9648), (276, 9856, 64),
    (1693, 1616, 64), (769, 64, 3672), (1620, 64, 1784), (1347, 64, 2296), (298, 72, 9512), (293, 10520, 72),
    (2620, 1760, 64), (7322, 392, 136), (522, 5512, 136), (394, 3512, 288), (6498, 64, 1000), (65, 3104, 2104),
    (1254, 64, 5440), (193, 408, 5640), (3318, 64, 2272), (1271, 136, 2816), (1181, 3168, 136), (781, 4608, 144),
    (790, 10320, 72), (3534, 1216, 176), (4602, 64, 2568), (5019, 400, 400), (107, 2400, 3504), (769, 256, 4576),
    (426, 4576, 520), (419, 568, 4416), (507, 280, 7656), (1028, 144, 7648), (3267, 152, 2448), (1182, 320, 3256),
    (838, 3752, 408), (2128, 9768, 64), (1034, 7672, 168), (1371, 816, 1208), (240, 2456, 2312), (2262, 64, 9672),
    (130, 3312, 3256), (241, 7088, 824), (792, 6976, 264), (4313, 4784, 72), (2510, 4760, 136), (441, 520, 7320),
    (797, 3272, 672), (187, 3112, 3144), (3984, 656, 720), (1567, 136, 10064), (1563, 9992, 144), (1019, 11232, 200),
    (1586, 136, 11240), (98, 5168, 4800), (171, 3800, 3744), (197, 8832, 1440), (5853, 688, 648), (3257, 12624, 64),
    (585, 560, 8064), (1582, 13512, 136), (4790, 64, 9640), (3277, 72, 12880), (7311, 7112, 64), (2348, 5360, 272),
    (2327, 272, 5840), (218, 5688, 3224), (6573, 2656, 232), (385, 5656, 1904), (222, 3272, 5848), (411, 1840, 5648),
    (234, 4448, 4224), (129, 5768, 6040), (3299, 5424, 264), (3445, 272, 5072), (148, 4056, 8688), (298, 3864, 4544),
    (6544, 64, 14920), (167, 6864, 7352), (196, 6328, 6808), (4952, 6872, 264), (4722, 272, 7104), (211, 5952, 8504),
    (225, 8088, 9232)]

# several tiles for each pair of CTAs, ragged in every dimension, contractions of many k-blocks
LARGE = [(2300, 4104, 4200), (4000, 3080, 4104), (4100, 3080, 6152)]


def plan(product, features, rows, contraction):
    out = (ctypes.c_int64 * 4)()
    _lib.check(_lib.load().chpl_diag_linear_plan(product, features, rows, contraction, out), "chpl_diag_linear_plan")
    return tuple(out)


def plans(T, k, n):
    """The plans of a layer's three products."""
    found = []
    for product, (f, r, c) in enumerate(((n, T, k), (k, T, n), (k, n, T))):
        pair, bn, split, tiles = plan(product, f, r, c)
        found.append((product, pair, bn, split, bool(pair and tiles > 74)))
    return found
