"""Philox4x32-10 in Python's whole numbers, from the published description (Salmon et al., "Parallel random numbers: as easy as 1, 2, 3", 2011)."""


def philox(counter, key):
    """Four random words of 32 bits for a counter of four words and a key of two."""
    c, k = list(counter), list(key)
    for _ in range(10):
        left, right = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [right >> 32 ^ c[1] ^ k[0], right & 0xffffffff, left >> 32 ^ c[3] ^ k[1], left & 0xffffffff]
        k = [(k[0] + 0x9E3779B9) & 0xffffffff, (k[1] + 0xBB67AE85) & 0xffffffff]
    return c


def words(first, count, seed, offset):
    """Those of dropout's elements [first, first + count)."""
    halves = lambda v: (v & 0xffffffff, v >> 32 & 0xffffffff)  # noqa: E731
    blocks = {b: philox((*halves(b), *halves(offset)), halves(seed)) for b in range(first // 4, (first + count - 1) // 4 + 1)}
    return [blocks[i // 4][i % 4] for i in range(first, first + count)]
