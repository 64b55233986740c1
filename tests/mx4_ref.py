"""Plain FP64 restatement of the 4-bit format and of where its codes and scales lie, and sizes that reach every kernel, tile and
split of its products."""
import ctypes
import math

import torch

from chpl_b200 import _lib

GROUP = 32
LEVELS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def pack(x):
    """(codes, scales) as integers, rows x cols and rows x ceil(cols / 32), by the rule of include/chpl.h, by the distance to
    every level."""
    x = x.double()
    rows, cols = x.shape
    groups = -(-cols // GROUP)
    p = torch.zeros(rows, groups * GROUP, dtype=torch.float64, device=x.device)
    p[:, :cols] = x
    p = p.reshape(rows, groups, GROUP)
    bad = ~torch.isfinite(p).all(2)
    top = torch.where(bad, torch.zeros_like(p[:, :, 0]), p.abs().amax(2))
    e = torch.where(top >= 2.0 ** -126, torch.frexp(top)[1] + 126, torch.zeros_like(top, dtype=torch.int32))
    s = e.clamp(min=7) - 2
    q = torch.ldexp(torch.nan_to_num(p, 0, 0, 0), (127 - s)[:, :, None])
    a = q.abs().clamp(max=6.0)
    best, code = torch.full_like(a, math.inf), torch.zeros_like(a, dtype=torch.int32)
    for i in (0, 2, 4, 6, 1, 3, 5, 7):  # even codes first, which win ties
        d = (a - LEVELS[i]).abs()
        code = torch.where(d < best, i, code)
        best = torch.minimum(best, d)
    code = code + 8 * torch.signbit(q).int()
    code = torch.where(bad[:, :, None], 0, code)
    return code.reshape(rows, -1)[:, :cols], torch.where(bad, 255, s)


def values(code, scales):
    """What they stand for, in FP64."""
    table = torch.tensor(LEVELS + [-v for v in LEVELS], dtype=torch.float64, device=code.device)
    step = torch.ldexp(torch.ones_like(scales, dtype=torch.float64), scales.int() - 127)
    step = torch.where(scales == 255, math.nan, step)
    return table[code.long()] * step.repeat_interleave(GROUP, dim=1)[:, : code.shape[1]]


def unpacked(c):
    """(codes, scales) of an mx4.Mx4 as integers, and what fills its rows' last groups."""
    b = c.codes.int()
    code = torch.stack([b & 15, b >> 4], 2).reshape(b.shape[0], -1)
    rows, groups = b.shape[0], -(-c.cols // GROUP)
    t = torch.arange(rows, device=b.device)[:, None]
    g = torch.arange(-(-c.cols // 256) * 8, device=b.device)[None]
    at = ((t // 128) * (2 * -(-c.cols // 256)) + g // 4) * 512 + (t % 32) * 16 + (t % 128) // 32 * 4 + g % 4
    s = c.scales.int()[at]
    return code[:, : c.cols], s[:, :groups], code[:, c.cols:], s[:, groups:]


def plan(T, n, k):
    """(1 pairs or 0 clusters, rows of a tile, CTAs of a tile) on the current device (148 SMs where there is none)."""
    p = (ctypes.c_int64 * 3)()
    _lib.check(_lib.load().chpl_diag_mx4_plan(n, T, k, p), "chpl_diag_mx4_plan")
    return tuple(p)


# (tokens, n, k): for every plan met among 400000 layers of 1 to 8192 tokens and 32 to 16384 features, the smallest that met it
SIZES = [(1, 32, 32), (1, 4274, 3858), (4, 1969, 2566), (1, 33, 2317), (17, 32, 34), (23, 4233, 4406), (31, 1944, 2844), (18, 33, 2616),
         (36, 33, 32), (34, 4403, 4884), (39, 1962, 3488), (33, 33, 2824), (52, 33, 34), (572, 388, 5038), (193, 419, 3368), (51, 33, 2819),
         (65, 10571, 32), (73, 4854, 7083), (76, 2051, 4125), (66, 905, 5489), (81, 9663, 33), (81, 5034, 9817), (95, 2405, 4891),
         (84, 952, 9623), (97, 9822, 39), (112, 4951, 12554), (104, 2095, 7703), (106, 898, 15929), (4949, 130, 35), (1073, 789, 12668),
         (529, 392, 10905), (144, 11426, 38), (136, 6430, 9007), (140, 3123, 8054), (140, 1542, 8638), (146, 12927, 37), (155, 6947, 11264),
         (147, 3182, 9511), (145, 1579, 9374), (170, 12948, 37), (163, 8979, 9619), (166, 3269, 12462), (161, 1412, 12068), (6767, 258, 41),
         (1250, 903, 16244), (670, 786, 12091), (564, 450, 16075), (194, 9924, 34), (197, 2443, 13828), (215, 10018, 39), (211, 2590, 16147),
         (227, 9496, 56), (392, 6561, 47), (258, 9531, 34), (262, 11650, 35), (7626, 517, 43), (395, 14305, 46)]
# one token and few on all kinds of widths, K over and under a piece, several tiles for each pair of SMs, ragged everywhere
MORE = [(1, 1, 1), (2, 8, 31), (3, 40, 33), (8, 129, 255), (9, 130, 257), (8, 1024, 4096), (16, 300, 512), (128, 128, 256), (129, 256, 1024),
        (300, 515, 1029), (2300, 4104, 1100), (4000, 3080, 520), (4100, 2050, 2304)]
