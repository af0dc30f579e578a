"""The rules by which kv8.attend picks its kernels, as a mirror of the library's, for tests that name the path they take
(test_kv8_plan.py holds it to the library's workspace sizes)."""
BLK = 64


def plan(kv, blocks, dim, heads, R, T, bt_cols, window=0):
    """(kind, columns of a tile, workgroups of a list or splits of a prompt, workspace bytes) of a call on a cache of `kv` heads and
    pages of `blocks` blocks: kind LISTED, DIRECT or PROMPT."""
    G, positions, mean = heads // kv, bt_cols * blocks * BLK, -(-T // R)
    seen = window + mean if 0 < window < positions - mean else positions
    cols, items = T * G // R, R * kv
    kind = "PROMPT" if cols >= 40 else "DIRECT" if seen <= (8192 if T <= R and items >= 128 else 1024) else "LISTED"
    width = 128 if kind == "PROMPT" else 32 if kind == "LISTED" and items * seen >= 1 << 19 and cols > 16 else 16
    TQ = width // G
    tiles = (T + R * (TQ - 1)) // TQ
    if kind == "PROMPT":
        wgs = -(-mean // TQ) * items
        splits = max(1, min(512 // wgs if wgs < 256 else 1, seen // (4 * BLK)))
        return kind, width, splits, T * heads * splits * (dim + 4) * 4 if splits > 1 else 0
    if kind == "DIRECT":
        return kind, width, 0, 0
    step = 128 if width == 16 else 64
    entries = tiles * kv * (-(-seen // step) + (seen < positions))
    groups = (entries + 1) // 2 if entries <= 1024 else (entries + 3) // 4 if entries < 2048 else 512 if items > 256 else 256
    if groups > 256 and items < 32:
        groups = 256
    return kind, width, groups, groups * (2 * width * (dim + 4) * 4 + 16)


def entries(kind, width, kv, heads, bs, prev, new, window=0):
    """What a list holds for rows of these histories and new tokens: (row, tile, head, step)."""
    assert kind == "LISTED"
    step, TQ, n = 128 if width == 16 else 64, width // (heads // kv), 0
    for p, c in zip(prev, new):
        lo = max(0, p + 1 - window) // BLK * BLK if window else 0
        n += -(-c // TQ) * kv * max(1, -(-(p + c - lo) // step))
    return n
