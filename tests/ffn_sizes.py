"""Sizes of the experts' products that between them launch every kernel and shape
that a call can (cuda_inf_amd/csrc/moe_shape.h)."""
import numpy as np

# rows of an expert, of every filling of a 128-row tile
LADDER = [1, 2, 16, 17, 31, 32, 33, 48, 63, 64, 65, 80, 95, 96, 97, 110, 127]
LONGER = LADDER + [128, 129, 150, 200, 256, 300]

# P pairs of E experts, k to a token; K inputs, N outputs (up: of each of the two)
# (P, k, E, K, N, rows by expert: None: even, "dense": one expert without ids)
UP = [
    # streams: 1, 2 and 4 groups a wave, 16 rows at a time and more
    (8, 4, 8, 896, 256, None),
    (8, 4, 8, 1920, 256, None),
    (8, 4, 8, 4096, 256, None),
    (60, 4, 256, 2048, 128, None),
    (480, 4, 256, 1024, 128, None),
    (12, 1, 1, 1024, 128, "dense"), (30, 1, 1, 896, 128, "dense"), (50, 1, 1, 640, 256, "dense"),
    (12, 1, 1, 2048, 128, "dense"), (30, 1, 1, 1152, 128, "dense"), (64, 1, 1, 1920, 384, "dense"),
    (12, 1, 1, 4096, 128, "dense"), (40, 1, 1, 4096, 128, "dense"), (64, 1, 1, 2176, 128, "dense"),
    (60, 3, 5, 3968, 256, None),
    # tiles of 1, 2 and 3 column tiles a wave, rows found by the workgroup and planned
    (980, 4, 32, 2304, 384, LADDER), (980, 4, 32, 2304, 768, LADDER), (980, 4, 32, 2304, 1152, LADDER),
    (2144, 4, 32, 2304, 384, LONGER), (2144, 4, 32, 2304, 640, LONGER), (2144, 4, 32, 2304, 1152, LONGER),
    (300, 1, 1, 256, 6272, "dense"), (900, 1, 1, 384, 4480, "dense"),
    (1100, 1, 1, 256, 2176, "dense"), (1100, 1, 1, 2176, 3968, "dense"),
    # 45 and 4096 tokens of 4 of 32 experts of 1792
    (180, 4, 32, 2048, 1792, None),
    (16384, 4, 32, 2048, 1792, None),
]
DOWN = [
    # few pairs in one launch
    (4, 4, 32, 1024, 256, None), (8, 4, 8, 896, 128, None), (4, 4, 32, 1792, 2048, None), (8, 2, 2, 2048, 128, None),
    (4, 4, 8, 4096, 256, None), (8, 4, 8, 2304, 128, None), (7, 1, 1, 3968, 128, "dense"),
    # streams: 1, 2 and 4 groups a wave, K in one part and two
    (12, 4, 32, 1024, 256, None), (12, 4, 32, 1792, 256, None), (12, 4, 32, 4096, 256, None),
    (12, 4, 32, 7168, 256, None), (12, 4, 32, 4224, 256, None), (4, 4, 32, 8192, 128, None),
    (300, 4, 256, 2048, 128, None), (16, 1, 1, 7168, 256, "dense"), (1, 1, 1, 7168, 2048, "dense"),
    # tiles, K in one part and several
    (980, 4, 32, 384, 256, LADDER), (980, 4, 32, 2304, 1536, LADDER), (980, 4, 32, 2304, 2304, LADDER),
    (980, 4, 32, 2304, 256, LADDER), (980, 4, 32, 4608, 512, LADDER),
    (2144, 4, 32, 2304, 256, LONGER), (2144, 4, 32, 2304, 1024, LONGER), (2144, 4, 32, 2304, 2048, LONGER),
    (1104, 4, 4, 1024, 128, None), (2144, 4, 32, 1536, 384, LONGER), (1100, 1, 1, 1536, 1408, "dense"),
    (900, 1, 1, 384, 4736, "dense"), (1100, 1, 1, 256, 4224, "dense"), (1100, 1, 1, 2176, 7936, "dense"),
    (700, 1, 1, 7168, 2048, "dense"),
    # 45 and 4096 tokens of 4 of 32 experts of 1792
    (180, 4, 32, 1792, 2048, None),
    (16384, 4, 32, 1792, 2048, None),
]


def pair_ids(P, k, E, rows):
    """ids int32 [P / k, k] (None: dense): rows[e] pairs of expert e in random order,
    what is left of P no expert's."""
    if rows == "dense":
        return None
    rng = np.random.default_rng(P + E)
    if rows is None:
        return np.stack([rng.permutation(E)[:k] if k <= E else rng.integers(0, E, k) for _ in range(P // k)]).astype(np.int32)
    ids = np.full(P, -1, np.int32)
    at = np.repeat(np.arange(len(rows)), rows)
    ids[:len(at)] = rng.permutation(E)[at]
    return rng.permutation(ids).reshape(P // k, k)
