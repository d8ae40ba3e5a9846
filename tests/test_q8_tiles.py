"""The products that test_q8_tiles_gpu.py runs reach every tile and each of its loops, by the rule as it stands."""
from q8_tiles import CASES, choice, tiles


def test_cases_reach_their_tiles():
    all_tiles = tiles()
    assert [t[:2] for t in all_tiles] == sorted(CASES, reverse=True)
    for tile, cases in CASES.items():
        for M, R, C, stages in cases:
            best, got, margin = choice(M, R, C, all_tiles)
            # (fp32 and fp64 costs are the same to 1e-6)
            assert all_tiles[best][:2] == tile and got == stages and margin > 0.01, (tile, M, R, C)


def test_cases_cover_the_loops():
    for tr, tm, _, _, _, _, groups, flight in tiles():
        cases = CASES[tr, tm]
        stages = {s for _, _, _, s in cases}
        # (two stages in flight: one is fewer; the largest tile has no fewer than three, see below)
        assert {flight - 1, flight, flight + 1} - ({1, 2} if tr == 256 else set()) <= stages
        assert {flight + 2, flight + 3} & stages and max(stages) >= 2 * flight + 2
        for M, R, C, _ in cases:
            assert R % tr and M % tm and C % 128, (M, R, C)
        assert {R % 4 for _, R, _, _ in cases} - {0}
        if groups > 1:  # a last stage without a step for each of its groups
            assert any(-(-C // 128) % groups for _, _, C, _ in cases)


def test_largest_tile_has_three_stages():
    all_tiles = tiles()
    for M in list(range(1, 20000, 331)) + [4096, 8192]:
        for R in list(range(1, 40000, 607)) + [4096, 8192]:
            for steps in (1, 2):
                best, _, _ = choice(M, R, 128 * steps, all_tiles)
                assert all_tiles[best][0] < 256, (M, R, steps)
