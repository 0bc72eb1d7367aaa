"""rotary_frequencies beyond its usual lengths.  No GPU."""
import math

import pytest


@pytest.mark.parametrize("length", [1, 2, 4, 6, 7, 40, 190, 250, 4096])
@pytest.mark.parametrize("n,base", [(2, 10000.0), (8, 10000.0), (64, 10000.0), (128, 5e5), (4, 1.5)])
def test_every_pair_is_slowed_by_how_often_it_turns(n, base, length):
    """yarn: pairs of more than beta_fast turns within the trained length keep their frequency, those of fewer than beta_slow have it divided, whatever the length."""
    from af3_kernels_amd.layers import rotary_frequencies
    for fast, slow in ((32.0, 1.0), (8.0, 2.0), (3.0, 0.25)):
        f, scale = rotary_frequencies(n, base, "yarn", 8.0, length, fast, slow)
        assert scale == 0.1 * math.log(8.0) + 1.0
        plain = rotary_frequencies(n, base)[0].tolist()
        for got, p in zip(f.tolist(), plain):
            turns = length * p / (2.0 * math.pi)
            assert p / 8.0 * (1 - 1e-15) <= got <= p * (1 + 1e-15)
            if turns > fast * (1 + 1e-12):
                assert got == p, (turns, got / p)
            if turns < slow * (1 - 1e-12):
                assert got == p / 8.0, (turns, got / p)


@pytest.mark.parametrize("args", [(2, 10000.0), (128, 1e6)])
def test_the_ramp_between_falls(args):
    from af3_kernels_amd.layers import rotary_frequencies
    ratio = [a / b for a, b in zip(rotary_frequencies(*args, "yarn", 4.0, 4096)[0].tolist(), rotary_frequencies(*args)[0].tolist())]
    assert all(x >= y for x, y in zip(ratio, ratio[1:])) and ratio[0] == 1.0
