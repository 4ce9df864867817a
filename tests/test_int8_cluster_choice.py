"""How a product of 8-bit integers is cut within a partition of the SMs: by the clusters that the driver says run at once there, which the
number of SMs does not tell.  No more tiles than that are ever taken where K is cut over a cluster."""
import ctypes

import pytest

from semi_pd_b200._lib import lib

# clusters of 1 to 8 CTAs, one CTA an SM: 76 SMs beside 72, those, 108 beside 40, those, and the whole B200
FOUND = {76: (76, 38, 21, 15, 12, 9, 6, 6), 72: (72, 36, 18, 18, 9, 9, 9, 9), 108: (108, 54, 30, 23, 20, 13, 10, 10),
         40: (40, 20, 10, 10, 5, 5, 5, 5), 36: (36, 18, 6, 5, 2, 2, 1, 1), 52: (52, 26, 12, 9, 6, 6, 3, 3), 148: (148, 74, 45, 33, 26, 22, 15, 15)}
# clusters of 4, 6 and 8 CTAs, two CTAs an SM, that ran at once there
TWO = {76: (33, 21, 15), 72: (36, 19, 18), 108: (50, 30, 23), 40: (20, 10, 10), 36: (10, 4, 3), 52: (18, 12, 9), 148: (71, 45, 33)}
WEIGHTS = [(4096, 4096), (4096, 14336), (5120, 5120), (6144, 4096), (28672, 4096), (3584, 8192), (8192, 3584), (1024, 8192), (2304, 8192),
           (10240, 2048), (136, 16384)]
TOKENS = (1, 5, 16, 31, 32, 33, 64, 100, 128, 160, 200, 256, 257, 300, 384, 500, 777, 1000)


def plan(m, n, k, sms, found):
    split, per_sm = ctypes.c_int(0), ctypes.c_int(0)
    clusters = (ctypes.c_int * 8)(*found)
    tiles = lib.spd_int8_scaled_mm_tiles(m, n, k, sms, ctypes.addressof(clusters), ctypes.addressof(split), ctypes.addressof(per_sm))
    assert tiles >= 0
    return tiles, split.value, per_sm.value


@pytest.mark.parametrize("sms", FOUND)
@pytest.mark.parametrize("n,k", WEIGHTS)
def test_one_wave(sms, n, k):
    for m in TOKENS:
        tiles, split, per_sm = plan(m, n, k, sms, FOUND[sms])
        if split > 1:
            at_once = FOUND[sms][2 * split - 1] if per_sm == 1 else TWO[sms][split - 2]
            assert tiles * ((n + 255) // 256) <= at_once, (m, tiles, split, per_sm)


def share(sms):
    return tuple(c * sms // 148 for c in FOUND[148])


def test_not_by_the_share_of_the_sms():
    """Where the driver's count is less than the share, that many tiles go another way; where it is more, they are taken."""
    assert share(76)[3] == 16 and share(72)[2] == 21
    for k in (4096, 14336):
        fours = ((1, 2, 1), (1, 4, 2))                          # 16 tiles on four SMs each: as many as the share has
        assert plan(1, 4096, k, 76, share(76)) in fours
        assert plan(1, 4096, k, 76, FOUND[76]) not in fours     # 15 run
    assert plan(16, 5120, 5120, 72, FOUND[72])[1:] != (3, 2)    # 20 tiles of six CTAs, two an SM: 18 run
    assert plan(64, 5120, 5120, 76, FOUND[76]) == (1, 3, 2)     # 21 run
    assert plan(256, 2304, 8192, 76, FOUND[76]) != (4, 2, 2)    # 36 of four CTAs, two an SM: 33 run
    assert plan(1, 2304, 8192, 72, FOUND[72])[1] == 4           # 9 tiles of eight: 9 run, the share is 7


@pytest.mark.parametrize("n,k", WEIGHTS)
def test_a_cut_that_does_not_fit(n, k):
    for m in TOKENS:
        assert plan(m, n, k, 76, (0,) * 8)[1] == 1
        assert plan(m, n, k, 76, (76, 38, 21, 15, 0, 0, 0, 0))[1] <= 2


def test_without_a_device_the_share():
    for m in TOKENS:
        for n, k in WEIGHTS:
            for sms in (148, 76):
                assert plan(m, n, k, sms, (-1,) * 8) == plan(m, n, k, sms, share(sms))


def test_refusals():
    one = ctypes.c_int(0)
    at = ctypes.addressof(one)
    assert lib.spd_int8_scaled_mm_tiles(0, 64, 64, 0, None, at, at) < 0
    assert lib.spd_int8_scaled_mm_tiles(1, 64, 64, 0, None, None, at) < 0
    assert lib.spd_int8_scaled_mm_tiles(1, 64, 131072, 0, None, at, at) < 0
