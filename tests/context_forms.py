"""Which kernels a call of attention over a context in two parts runs, as the library plans it."""
import ctypes
from collections import namedtuple

import floneum_amd as fa

Tiles = namedtuple("Tiles", "fold prefix own shares")  # a job of the tiled launch: rows of all sequences together, the parts it walks, shares of its keys
Few = namedtuple("Few", "prefix shares")               # a job of the launch for few rows
Form = namedtuple("Form", "rows any rows_per_group key_groups tiles columns few slots")
WORDS = 19


def forms(args, compute_units=256):
    """Of each of a call's parts."""
    words = (ctypes.c_int32 * (2 * WORDS))()
    fa.lib()._ZN4fhip13context_formsEPK22fhip_context_attn_argsiPi(ctypes.byref(args), ctypes.c_int(compute_units), words)
    got = []
    for at in (0, WORDS):
        w = list(words[at:at + WORDS])
        if w[0]:
            tiles = [Tiles(*w[5 + 4 * j:9 + 4 * j]) for j in range(w[4])]
            got.append(Form(w[0], w[1], w[2], w[3], tiles, w[13], [Few(*w[14 + 2 * j:16 + 2 * j]) for j in range(2) if w[15 + 2 * j]], w[18]))
    return got


def described(args, compute_units=256):
    """The same without the numbers of shares, a part each: 'any', or the launches: '256x1: all prefix, own' (rows per workgroup x key groups: jobs; all: rows of
    all sequences together; a job's parts joined by +; ' /' behind it: its keys are in shares), '16 columns: prefix /, own'."""
    out = []
    for f in forms(args, compute_units):
        launches = ["any"] if f.any else []
        if f.tiles:
            jobs = [("all " if t.fold else "") + "+".join(["prefix"] * t.prefix + ["own"] * t.own) + (" /" if t.shares > 1 else "") for t in f.tiles]
            launches.append(f"{f.rows_per_group}x{f.key_groups}: " + ", ".join(jobs))
        if f.few:
            launches.append(f"{f.columns} columns: " + ", ".join(("prefix" if x.prefix else "own") + (" /" if x.shares > 1 else "") for x in f.few))
        out.append("; ".join(launches))
    return out


# Calls that between them reach every launch of the plan, and calls whose last rows run apart: B, H, Hkv, Sq, Skv, P, D, window, sinks, whether lengths and positions
# come with the call, and what runs on 256 compute units.  (The plan goes by estimated time: after a change of its constants a call may have to be replaced by one that
# reaches the same form.)
CALLS_16 = [
    (22, 6, 2, 73, 0, 203, 128, 0, 0, True, "128x2: all prefix"),
    (3, 4, 2, 87, 0, 3102, 128, 0, 0, False, "128x2: all prefix /"),
    (31, 6, 2, 33, 165, 1131, 72, 0, 0, False, "128x2: all prefix /, own"),
    (29, 3, 1, 13, 2217, 514, 128, 0, 0, False, "128x2: all prefix /, own /"),
    (35, 32, 8, 3, 110, 3295, 72, 0, 0, True, "128x2: all prefix /; 16 columns: own"),
    (21, 32, 8, 4, 586, 7908, 72, 0, 0, True, "128x2: all prefix /; 16 columns: own /"),
    (24, 32, 8, 12, 30, 1111, 96, 0, 0, False, "128x2: all prefix /; 32 columns: own"),
    (32, 16, 4, 25, 36, 340, 96, 0, 0, False, "128x2: all prefix, own"),
    (20, 16, 4, 5, 2959, 28, 96, 0, 0, False, "128x2: all prefix, own /"),
    (27, 32, 8, 18, 48, 507, 128, 0, 0, True, "128x2: all prefix; 16 columns: own"),
    (36, 32, 8, 25, 73, 636, 96, 0, 0, True, "128x2: all prefix; 32 columns: own"),
    (1, 4, 1, 69, 206, 0, 128, 0, 0, True, "128x2: own"),
    (31, 4, 2, 9, 3155, 0, 96, 0, 0, False, "128x2: own /"),
    (1, 4, 1, 94, 0, 163, 128, 70, 2, False, "128x2: prefix"),
    (1, 8, 1, 178, 0, 2162, 128, 0, 0, False, "128x2: prefix /"),
    (1, 3, 1, 1, 3, 0, 72, 0, 0, True, "16 columns: own"),
    (1, 2, 2, 1, 155, 0, 128, 0, 0, False, "16 columns: own /"),
    (1, 2, 2, 1, 0, 25, 96, 0, 0, False, "16 columns: prefix"),
    (1, 3, 1, 1, 0, 159, 128, 386, 21, False, "16 columns: prefix /"),
    (1, 2, 2, 1, 48, 157, 64, 553, 2, False, "16 columns: prefix /, own"),
    (1, 2, 2, 1, 221, 320, 72, 854, 2, True, "16 columns: prefix /, own /"),
    (1, 3, 1, 1, 3, 27, 64, 101, 1, False, "16 columns: prefix, own"),
    (1, 4, 2, 1, 153, 21, 64, 0, 0, True, "16 columns: prefix, own /"),
    (22, 16, 4, 24, 0, 22, 96, 0, 0, False, "256x1: all prefix"),
    (3, 32, 8, 9, 0, 5124, 96, 0, 0, True, "256x1: all prefix /"),
    (21, 16, 4, 25, 209, 579, 72, 0, 0, False, "256x1: all prefix /, own"),
    (38, 4, 2, 58, 772, 1232, 72, 0, 0, True, "256x1: all prefix /, own /"),
    (30, 16, 4, 18, 64, 4583, 64, 0, 0, False, "256x1: all prefix /; 16 columns: own"),
    (39, 32, 8, 17, 142, 1341, 64, 0, 0, False, "256x1: all prefix /; 32 columns: own"),
    (16, 32, 8, 18, 19, 21, 128, 0, 0, False, "256x1: all prefix, own"),
    (24, 16, 4, 20, 326, 99, 128, 0, 0, False, "256x1: all prefix, own /"),
    (39, 32, 8, 28, 38, 976, 128, 0, 0, False, "256x1: all prefix; 32 columns: own"),
    (1, 8, 1, 43, 45, 0, 64, 67, 8, True, "256x1: own"),
    (1, 4, 1, 65, 374, 0, 72, 0, 0, False, "256x1: own /"),
    (1, 8, 1, 67, 0, 22, 72, 0, 0, False, "256x1: prefix"),
    (1, 8, 1, 41, 0, 314, 128, 0, 0, True, "256x1: prefix /"),
    (1, 8, 1, 36, 49, 55, 72, 0, 0, False, "256x1: prefix+own"),
    (1, 8, 1, 42, 222, 145, 72, 0, 0, False, "256x1: prefix+own /"),
    (37, 32, 8, 5, 6, 0, 96, 0, 0, True, "32 columns: own"),
    (7, 4, 1, 30, 3345, 0, 64, 0, 0, False, "32 columns: own /"),
    (29, 16, 4, 19, 0, 22, 72, 0, 0, True, "32 columns: prefix"),
    (1, 32, 8, 13, 0, 6133, 64, 0, 0, True, "32 columns: prefix /"),
    (13, 4, 2, 79, 94, 143, 72, 0, 0, False, "32 columns: prefix /, own"),
    (32, 6, 2, 6, 651, 1270, 64, 0, 0, False, "32 columns: prefix /, own /"),
    (22, 32, 8, 5, 7, 36, 72, 0, 0, False, "32 columns: prefix, own"),
    (10, 16, 4, 28, 165, 39, 72, 157, 6, False, "32 columns: prefix, own /"),
    (23, 16, 4, 57, 0, 22, 192, 0, 0, True, "128x1: all prefix"),
    (5, 6, 2, 15, 0, 4641, 256, 0, 0, False, "128x1: all prefix /"),
    (2, 8, 1, 33, 53, 103, 192, 0, 0, False, "128x1: all prefix /, own"),
    (2, 4, 1, 67, 79, 117, 192, 0, 0, False, "128x1: all prefix /, own /"),
    (27, 32, 8, 3, 26, 1417, 192, 0, 0, True, "128x1: all prefix /; 16 columns: own"),
    (35, 16, 4, 1, 99, 7799, 192, 0, 0, False, "128x1: all prefix /; 16 columns: own /"),
    (3, 8, 1, 34, 35, 64, 192, 0, 0, True, "128x1: all prefix, own"),
    (2, 8, 1, 38, 61, 28, 192, 0, 0, True, "128x1: all prefix, own /"),
    (28, 32, 8, 23, 25, 124, 192, 0, 0, False, "128x1: all prefix; 16 columns: own"),
    (1, 8, 1, 34, 40, 0, 192, 549, 3, False, "128x1: own"),
    (1, 3, 1, 127, 251, 0, 192, 0, 0, True, "128x1: own /"),
    (1, 4, 1, 93, 0, 22, 192, 0, 0, True, "128x1: prefix"),
    (1, 8, 1, 47, 0, 229, 192, 0, 0, True, "128x1: prefix /"),
    (1, 8, 1, 48, 49, 91, 256, 71, 73, True, "128x1: prefix /, own"),
    (1, 8, 1, 37, 46, 62, 192, 0, 0, False, "128x1: prefix /, own /"),
    (2, 8, 1, 55, 134, 29, 256, 32, 34, True, "128x1: prefix, own"),
    (1, 4, 1, 100, 123, 37, 192, 0, 0, False, "128x1: prefix, own /"),
    (1, 2, 2, 1, 2, 0, 192, 0, 0, True, "16 columns: own"),
    (1, 2, 2, 1, 216, 0, 256, 0, 0, True, "16 columns: own /"),
    (1, 2, 2, 2, 0, 21, 192, 0, 0, False, "16 columns: prefix"),
    (1, 2, 2, 1, 0, 135, 256, 0, 0, True, "16 columns: prefix /"),
    (1, 2, 2, 2, 19, 70, 192, 0, 0, True, "16 columns: prefix /, own"),
    (1, 4, 1, 1, 67, 78, 192, 0, 0, False, "16 columns: prefix /, own /"),
    (1, 2, 2, 1, 16, 23, 256, 0, 0, True, "16 columns: prefix, own"),
    (2, 2, 2, 1, 67, 34, 192, 0, 0, True, "16 columns: prefix, own /"),
    (30, 32, 8, 36, 37, 0, 256, 0, 0, True, "128x1: own | 16 columns: own"),
    (34, 32, 8, 65, 0, 25, 192, 0, 0, False, "128x1: all prefix | 16 columns: prefix"),
    (13, 32, 8, 231, 0, 20, 192, 0, 0, False, "128x1: prefix | 16 columns: prefix"),
    (4, 32, 8, 133, 141, 34, 256, 0, 0, True, "128x1: all prefix, own | 16 columns: prefix, own /"),
    (3, 32, 8, 164, 189, 126, 192, 0, 0, False, "128x1: all prefix, own | 16 columns: prefix /, own /"),
    (12, 32, 8, 37, 51, 339, 192, 458, 4, True, "128x1: prefix, own | 16 columns: prefix /, own"),
    (31, 16, 4, 35, 60, 214, 256, 136, 1, False, "128x1: all prefix, own | 16 columns: prefix /, own"),
    (35, 4, 2, 193, 249, 0, 192, 0, 0, True, "128x1: own | 16 columns: own /"),
    (27, 32, 8, 40, 47, 109, 256, 192, 43, True, "128x1: prefix, own | 16 columns: prefix, own"),
    (9, 16, 4, 232, 0, 213, 256, 0, 0, True, "128x1: prefix | 16 columns: prefix /"),
    (28, 2, 2, 272, 452, 31, 256, 49, 13, False, "128x1: all prefix, own | 16 columns: prefix, own"),
]
CALLS_F32 = [
    (28, 4, 2, 89, 0, 24, 72, 0, 0, True, "128x1: all prefix"),
    (10, 6, 2, 44, 0, 840, 64, 0, 0, True, "128x1: all prefix /"),
    (38, 32, 8, 10, 20, 51, 72, 0, 0, True, "128x1: all prefix /, own"),
    (25, 6, 2, 39, 111, 163, 96, 0, 0, False, "128x1: all prefix /, own /"),
    (24, 32, 8, 7, 12, 810, 72, 0, 0, False, "128x1: all prefix /; 16 columns: own"),
    (8, 4, 1, 34, 68, 4102, 72, 0, 0, True, "128x1: all prefix /; 16 columns: own /"),
    (14, 32, 8, 17, 32, 30, 128, 0, 0, False, "128x1: all prefix, own"),
    (28, 16, 4, 18, 76, 24, 72, 0, 0, False, "128x1: all prefix, own /"),
    (34, 32, 8, 33, 53, 642, 128, 0, 0, False, "128x1: all prefix; 16 columns: own"),
    (1, 8, 1, 35, 37, 0, 128, 274, 1, False, "128x1: own"),
    (1, 4, 1, 71, 84, 0, 72, 0, 0, True, "128x1: own /"),
    (1, 3, 1, 122, 0, 21, 64, 0, 0, True, "128x1: prefix"),
    (1, 8, 1, 34, 0, 144, 72, 0, 0, False, "128x1: prefix /"),
    (1, 8, 1, 33, 45, 70, 128, 34, 6, True, "128x1: prefix+own"),
    (1, 8, 1, 47, 57, 43, 72, 0, 0, True, "128x1: prefix+own /"),
    (28, 32, 8, 20, 0, 104, 128, 0, 0, True, "128x2: all prefix"),
    (23, 4, 2, 3, 0, 7184, 128, 0, 0, True, "128x2: all prefix /"),
    (16, 16, 4, 14, 15, 586, 128, 0, 0, True, "128x2: all prefix /, own"),
    (28, 2, 2, 54, 206, 524, 128, 0, 0, True, "128x2: all prefix /, own /"),
    (19, 32, 8, 2, 11, 3033, 96, 0, 0, True, "128x2: all prefix /; 16 columns: own"),
    (15, 8, 1, 19, 454, 2294, 72, 0, 0, False, "128x2: all prefix /; 16 columns: own /"),
    (19, 32, 8, 18, 159, 212, 128, 362, 69, False, "128x2: all prefix, own"),
    (33, 2, 2, 67, 333, 38, 128, 0, 0, True, "128x2: all prefix, own /"),
    (34, 16, 4, 25, 107, 0, 128, 0, 0, False, "128x2: own"),
    (2, 32, 8, 67, 530, 0, 128, 0, 0, True, "128x2: own /"),
    (29, 8, 1, 65, 0, 105, 128, 551, 14, False, "128x2: prefix"),
    (3, 32, 8, 69, 0, 331, 128, 0, 0, True, "128x2: prefix /"),
    (12, 32, 8, 36, 46, 64, 128, 314, 11, False, "128x2: prefix+own"),
    (23, 4, 1, 37, 449, 93, 128, 0, 0, True, "128x2: prefix+own /"),
    (2, 2, 2, 1, 2, 0, 72, 0, 0, False, "16 columns: own"),
    (1, 2, 2, 1, 72, 0, 128, 0, 0, False, "16 columns: own /"),
    (1, 2, 2, 1, 0, 20, 128, 0, 0, False, "16 columns: prefix"),
    (1, 2, 2, 1, 0, 89, 96, 257, 2, False, "16 columns: prefix /"),
    (1, 2, 2, 1, 18, 95, 64, 603, 2, True, "16 columns: prefix /, own"),
    (1, 2, 2, 2, 142, 65, 64, 0, 0, False, "16 columns: prefix /, own /"),
    (1, 3, 1, 1, 10, 28, 96, 0, 0, False, "16 columns: prefix, own"),
    (1, 2, 2, 1, 93, 52, 64, 659, 40, False, "16 columns: prefix, own /"),
    (31, 4, 2, 108, 0, 42, 64, 0, 0, True, "64x2: all prefix"),
    (22, 8, 1, 4, 0, 2647, 64, 0, 0, True, "64x2: all prefix /"),
    (20, 32, 8, 7, 113, 495, 64, 0, 0, True, "64x2: all prefix /, own"),
    (2, 32, 8, 14, 2838, 487, 64, 0, 0, True, "64x2: all prefix /, own /"),
    (34, 32, 8, 4, 7, 1318, 64, 0, 0, False, "64x2: all prefix /; 16 columns: own"),
    (15, 32, 8, 1, 277, 8225, 96, 0, 0, False, "64x2: all prefix /; 16 columns: own /"),
    (36, 6, 2, 33, 116, 69, 64, 0, 0, False, "64x2: all prefix, own"),
    (30, 16, 4, 14, 434, 78, 64, 0, 0, True, "64x2: all prefix, own /"),
    (1, 8, 1, 42, 54, 0, 64, 0, 0, False, "64x2: own"),
    (2, 6, 2, 149, 303, 0, 64, 0, 0, True, "64x2: own /"),
    (1, 4, 1, 72, 0, 37, 64, 0, 0, True, "64x2: prefix"),
    (3, 2, 2, 262, 0, 355, 64, 0, 0, False, "64x2: prefix /"),
    (1, 8, 1, 49, 52, 30, 64, 0, 0, False, "64x2: prefix+own"),
    (2, 6, 2, 120, 123, 234, 64, 0, 0, True, "64x2: prefix+own /"),
    (20, 6, 2, 57, 0, 24, 192, 109, 8, False, "128x1: all prefix"),
    (35, 4, 2, 11, 0, 679, 192, 0, 0, False, "128x1: all prefix /"),
    (6, 32, 8, 25, 31, 37, 192, 0, 0, False, "128x1: all prefix /, own"),
    (34, 3, 1, 38, 89, 66, 256, 0, 0, False, "128x1: all prefix /, own /"),
    (21, 32, 8, 2, 3, 1881, 192, 0, 0, False, "128x1: all prefix /; 16 columns: own"),
    (6, 32, 8, 3, 520, 4092, 192, 0, 0, True, "128x1: all prefix /; 16 columns: own /"),
    (30, 16, 4, 10, 12, 23, 192, 0, 0, True, "128x1: all prefix, own"),
    (5, 32, 8, 31, 33, 23, 192, 0, 0, False, "128x1: all prefix, own /"),
    (36, 32, 8, 19, 56, 504, 192, 0, 0, True, "128x1: all prefix; 16 columns: own"),
    (3, 8, 1, 40, 47, 0, 192, 0, 0, False, "128x1: own"),
    (1, 8, 1, 39, 41, 0, 192, 0, 0, True, "128x1: own /"),
    (1, 4, 1, 147, 0, 22, 192, 0, 0, True, "128x1: prefix"),
    (1, 4, 1, 68, 0, 34, 256, 0, 0, False, "128x1: prefix /"),
    (13, 32, 8, 9, 11, 31, 256, 836, 8, True, "128x1: prefix+own"),
    (1, 8, 1, 33, 36, 43, 192, 0, 0, True, "128x1: prefix+own /"),
    (1, 2, 2, 2, 3, 0, 192, 0, 0, True, "16 columns: own"),
    (1, 3, 1, 1, 72, 0, 256, 0, 0, False, "16 columns: own /"),
    (2, 2, 2, 1, 0, 29, 192, 293, 1, False, "16 columns: prefix"),
    (1, 2, 2, 1, 0, 86, 192, 0, 0, False, "16 columns: prefix /"),
    (1, 2, 2, 1, 12, 79, 192, 0, 0, True, "16 columns: prefix /, own"),
    (1, 2, 2, 1, 149, 143, 256, 0, 0, False, "16 columns: prefix /, own /"),
    (1, 2, 2, 1, 3, 51, 192, 0, 0, True, "16 columns: prefix, own"),
    (1, 3, 1, 2, 91, 21, 192, 0, 0, True, "16 columns: prefix, own /"),
    (4, 16, 4, 77, 110, 0, 192, 0, 0, False, "16 columns: own | 16 columns: own /"),
    (16, 8, 1, 40, 0, 113, 192, 66, 81, True, "16 columns: prefix | 16 columns: prefix /"),
    (35, 4, 2, 204, 0, 20, 256, 0, 0, False, "128x1: prefix | 16 columns: prefix"),
    (22, 16, 4, 67, 68, 0, 192, 0, 0, True, "128x1: own | 16 columns: own /"),
    (25, 32, 8, 33, 46, 0, 256, 0, 0, False, "128x1: own | 16 columns: own"),
    (9, 32, 8, 236, 0, 97, 72, 0, 0, True, "128x1: prefix | 16 columns: prefix"),
    (38, 4, 2, 201, 0, 65, 256, 0, 0, False, "128x1: prefix | 16 columns: prefix /"),
    (37, 32, 8, 33, 41, 31, 192, 0, 0, False, "128x1: prefix+own | 16 columns: prefix, own"),
    (28, 16, 4, 134, 140, 0, 72, 0, 0, True, "128x1: own | 16 columns: own"),
    (11, 32, 8, 65, 232, 0, 128, 377, 13, False, "128x2: own | 16 columns: own /"),
    (25, 32, 8, 66, 67, 74, 96, 0, 0, True, "128x1: prefix+own | 16 columns: prefix, own"),
]
