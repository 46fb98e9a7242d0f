"""How nf4_matvec's launch cuts its work, computed here as csrc/nf4_matvec.hip does, and the sizes that the GPU test
runs because of it: wavefronts whose run crosses from one tile of 16 rows to the next, blocks in several rounds,
every template."""

import pytest

WAVES, MOST_TILES, BLOCKS = 16, 16, 256


def cut(outs, K):
    """(tiles to a block, blocks, steps of 128 k to a tile, the numbers of tiles that blocks have)."""
    tiles = [-(-n // 16) for n in outs]
    per = 1
    while sum(-(-t // per) for t in tiles) > BLOCKS and per < MOST_TILES:
        per += 1
    sizes = {per if t >= per else t for t in tiles} | {t % per for t in tiles if t % per}
    return per, sum(-(-t // per) for t in tiles), -(-K // 128), sizes


def crosses(tiles, steps):
    """Whether a wavefront of a block walks steps of two tiles or more."""
    total = tiles * steps
    waves = min(total, WAVES)
    runs = [(w * total // waves, (w + 1) * total // waves) for w in range(waves)]
    return any(b > a and a // steps != (b - 1) // steps for a, b in runs)


def template(M, K, per):
    """(8 or 16 rows of x, x in LDS, steps in flight)."""
    mt = 1 if M <= 8 else 2
    row = 2 * (-(-K // 128) * 128 + 8)
    held = 64 + M * row <= ((95 if mt == 1 else 80) if per > 1 else 64) * 1024
    return mt, held, 2 if mt == 2 and not held else 4


# (outputs of each weight, K, rows of x)
CROSSING = [
    ((8960, 8960), 1536, (1, 8, 9, 16)),     # 5 tiles of 12 steps
    ((18944, 18944), 3584, (1, 8, 9, 16)),   # 10 tiles of 28 steps; 16 rows of x past LDS
    ((45056 - 37,), 256, (1, 8, 9, 16)),     # 11 tiles of 2 steps
    ((45056 - 37,), 384, (1, 5, 16)),        # of 3, fewer than are in flight
    ((30000, 15056), 192, (2, 16)),          # of one and a half
    ((12288 - 5,), 8960, (1, 8, 9)),         # 3 tiles of 70 steps, 8 rows of x past LDS
    ((151936 - 48,), 896, (1, 16)),          # 16 tiles to a block, 594 blocks, the last of 5
]


@pytest.mark.parametrize("case", range(len(CROSSING)))
def test_cases_cross_a_border(case):
    outs, K, _ = CROSSING[case]
    _, _, steps, sizes = cut(outs, K)
    assert any(crosses(t, steps) for t in sizes)


def test_what_the_cases_reach():
    made = [(cut(outs, K), M, K) for outs, K, rows in CROSSING for M in rows]
    assert {template(M, K, c[0]) for c, M, K in made} == {(1, True, 4), (1, False, 4), (2, True, 4), (2, False, 2)}
    assert any(c[1] > BLOCKS and c[0] == MOST_TILES for c, _, _ in made)
    assert {c[2] for c, _, _ in made if c[2] < 4} == {2, 3}  # fewer steps to a tile than are in flight


def test_two_tiles_meet_at_a_border():
    """Why sizes of up to 512 tiles do not cross."""
    assert not any(crosses(2, steps) for steps in range(1, 200))
