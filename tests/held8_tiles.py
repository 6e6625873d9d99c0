"""Steps over a cache of 8 bits that go through their keys 128 rows at a time, for the tests of
how they are laid out (CPU) and of what comes out (GPU): (heads, KV heads, head_dim, page,
positions of each sequence, new ones of each, positions of a shared prefix)."""

MANY = {
    "a head a KV head, one tile of rows": (128, 128, 64, 16, [970, 40], [70, 3], 0),
    "four heads a KV head, the last tile's rows few": (64, 16, 128, 64, [1601], [101], 0),
    "a padded head": (60, 20, 80, 32, [1703], [97], 0),
    "a prompt from its start": (64, 16, 64, 32, [610, 30], [610, 30], 0),
    "a shared prefix": (208, 13, 128, 64, [1 + 7 * (i % 5) for i in range(10)], [1] * 10, 4111),
    "a shared prefix, a narrow head": (192, 24, 64, 16, [5 + 11 * (i % 5) for i in range(14)], [1 + i % 2 for i in range(14)], 2500),
    "a group of three rows a token over a prefix": (72, 24, 96, 16, [200, 333, 90], [55, 60, 49], 1200),
}

# too few keys for that: 64 rows at a time
HALF = {
    "three prompts": (20, 5, 128, 16, [65, 105, 300], [65] * 3, 0),
    "a prompt behind a prefix": (8, 2, 64, 16, [300], [80], 1000),
}
