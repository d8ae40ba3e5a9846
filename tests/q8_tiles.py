"""Products of 8-bit rows by the tile that csdr_q8_linear takes for them, and its rule (cost_of in
cortexsdr_amd/csrc/q8_linear.hip) over the figures that stand there, so that a change of those shows in the tests
rather than in what they reach."""
import os
import re

import numpy as np

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cortexsdr_amd", "csrc",
                      "q8_linear.hip")

# (rows of w, tokens) of a tile -> products (M, R, C) with the stages of columns they have there: fewer than the tile
# has in flight, as many, one more and many more, so that each of its loops runs not at all, once and again; all with
# rests of rows (also of four neighbouring ones), of tokens and of columns
CASES = {
    (16, 16): [(9, 17, 16, 1), (9, 18, 664, 2), (9, 17, 1105, 3), (9, 19, 1726, 4), (9, 17, 2168, 5),
               (33, 250, 5001, 10)],
    (32, 32): [(17, 4110, 296, 2), (18, 4171, 545, 3), (17, 4161, 819, 4), (17, 2066, 1033, 5), (17, 2110, 1596, 7),
               (17, 2159, 2370, 10)],
    (32, 64): [(8684, 65, 204, 2), (8262, 66, 362, 3), (8495, 67, 408, 4), (8766, 67, 516, 5), (8679, 67, 781, 7),
               (4129, 33, 3147, 25)],
    (64, 64): [(5499, 257, 65, 1), (8672, 170, 168, 2), (5460, 298, 261, 3), (5536, 271, 429, 4), (8221, 163, 598, 5),
               (8587, 161, 1160, 10)],
    (128, 64): [(329, 8419, 14, 1), (201, 6478, 185, 2), (142, 8271, 352, 3), (80, 8717, 492, 4), (65, 8346, 544, 5),
                (66, 8225, 1247, 10)],
    (128, 128): [(8620, 394, 104, 1), (6536, 545, 184, 2), (8361, 414, 332, 3), (8291, 395, 448, 4),
                 (8524, 402, 1084, 9)],
    # (no product of fewer than three stages is cheapest in these)
    (256, 256): [(3901, 4090, 300, 3), (8268, 1433, 453, 4), (2692, 4402, 897, 8)],
}


def tiles():
    """[(rows, tokens, workgroups a CU holds, fixed, alone, each, groups of waves, stages in flight)] as the source
    has them."""
    with open(SOURCE) as f:
        text = f.read()
    costs = text[text.index("constexpr Cost kCosts[] = {"):]
    costs = re.findall(r"\{(\d+), (\d+), (\d+), ([\d.]+)f, ([\d.]+)f, ([\d.]+)f\}", costs[:costs.index("};")])
    shapes = re.findall(r"return launch_tiles<T, (\d+), (\d+), (\d+), \d+, \d+, (\d+)>", text)
    assert len(costs) == len(shapes) == 7
    out = []
    for c, s in zip(costs, shapes):
        assert c[:2] == s[:2]
        out.append((*map(int, c[:3]), *map(float, c[3:]), int(s[2]), int(s[3])))
    return out


def choice(M, R, C, all_tiles):
    """The tile's place, its stages, and by what share the next one costs more."""
    steps, costs = -(-C // 128), []
    for tr, tm, held, fixed, alone, each, _, _ in all_tiles:
        most = -(-(-(-R // tr) * -(-M // tm)) // 256)  # of a CU's workgroups
        rest = most % held
        us = (most // held) * (fixed + steps * held * each)
        costs.append(us + (fixed + steps * max(alone, rest * each) if rest else 0.0))
    best = int(np.argmin(costs))
    return best, -(-steps // all_tiles[best][6]), sorted(costs)[1] / costs[best] - 1
