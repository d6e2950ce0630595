"""Which of the kernels of attention over the 4-bit cache a call takes, by the rule on its sizes, and cases for each."""


def path(H, KV, d, n, most, run):
    """("whole", head_dim, 16-row sets, waves): a workgroup per block; ("share", head_dim, sets): shares of all tiles."""
    G = H // KV
    rows = min(max(run, 1), n) * G
    sets = 2 if rows > 16 else 1
    tq = max(1, min(run, 16 * sets // G))
    blocks = -(-n // tq) * KV
    if rows > 32 or most > (3200 if blocks >= 512 else 1024):
        return "share", d, sets
    return "whole", d, sets, 4 if n * KV >= 512 else 8


# heads, KV heads, head_dim, page, tokens of each sequence, rows that the last token of each sees
CASES = [
    (32, 8, 128, 32, [6] * 12, [6 + 83 * i for i in range(12)]),
    (16, 4, 64, 16, [7] * 20, [7 + 53 * i for i in range(20)]),
    (32, 8, 128, 64, [8, 5, 7] * 4, [1021 - 90 * i for i in range(11)] + [8]),
    (8, 2, 64, 32, [5, 8, 3], [1000, 8, 333]),
    (8, 2, 128, 128, [5, 8, 3], [999, 70, 3]),
    (40, 2, 128, 16, [1] * 260, [1 + (61 * i) % 130 for i in range(258)] + [2111, 3199]),
    (20, 1, 64, 64, [1] * 513, [1 + (37 * i) % 90 for i in range(512)] + [3200]),
    (32, 32, 64, 32, [20] * 16 + [3], [20 + 13 * i for i in range(15)] + [1999, 3]),
    (16, 16, 128, 16, [17] * 32 + [4], [17 + 7 * i for i in range(32)] + [1501]),
    (64, 64, 64, 16, [2] * 9, [2 + 47 * i for i in range(8)] + [1700]),
    (32, 32, 128, 64, [16] * 17, [16 + 5 * i for i in range(16)] + [2050]),
    (40, 8, 128, 32, [1] * 5, [1024, 77, 1, 500, 63]),
    (32, 8, 128, 32, [8] * 8, [1100 + 131 * i for i in range(8)]),
]


def path_of(case):
    H, KV, d, page, new, rows = case
    return path(H, KV, d, sum(new), max(rows), max(new))
