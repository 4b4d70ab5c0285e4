"""Long cases of attention over the paged 8-bit cache, for kv_bounds.marked: new, lens, query heads, kv heads, head_dim,
page, window, sinks, type, max_len."""
import torch

BF, HF = torch.bfloat16, torch.float16

# one token a sequence: the keys are split over workgroups and joined
LONG_DECODE = [
    ([1], [40000], 32, 8, 128, 64, 0, 0, HF, 40000),
    ([1, 1, 1], [9000, 8939, 8878], 8, 1, 64, 16, 4096, 4, BF, 9000),
    ([1] * 40, [3000 - 61 * b for b in range(40)], 4, 4, 128, 64, 0, 0, BF, 3000),
    ([1], [70001], 3, 1, 32, 16, 8192, 20, BF, 70001),
    ([5, 2], [20011, 7000], 8, 2, 128, 32, 0, 0, HF, 20011),
]
# four waves to a workgroup and more than 48 tiles of keys in one run of them: the looked-up pages and scales of 32 tiles
# are overwritten at least once while they are used. A max_len far above the lengths leaves the keys unsplit.
RINGS = [
    ([300], [5000], 8, 2, 64, 16, 0, 0, BF, 1 << 20),
    ([300], [5000], 8, 2, 32, 16, 0, 0, HF, 1 << 20),
    ([300, 77], [5003, 4100], 128, 32, 64, 32, 0, 0, HF, 5003),
    ([300], [5001], 128, 32, 64, 16, 3000, 70, BF, 5001),
    ([300], [4999], 128, 32, 32, 128, 2500, 5, BF, 4999),
    ([60, 61, 9, 60, 62, 63], [5000, 4000, 700, 3300, 4990, 64], 32, 8, 128, 16, 0, 0, BF, 1 << 20),
    ([60, 61, 60, 62, 63, 60], [5000, 4000, 3300, 4990, 3200, 3135], 96, 24, 128, 64, 3000, 70, HF, 5000),
]
