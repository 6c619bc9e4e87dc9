"""The step's quotients are the correctly rounded ones, shown for every pair of mantissas for which they
could fail to be.

With integers M and D of 24 bits for the mantissas of m and d, and s = 24 where M < D, else 23, the
quotient lies K / (2 D) units of its last place from a border between two results, for an integer
K = M 2^(s+1) - N D with an odd N. The approximate quotient q is off by at most 1.5 units (its rounding,
and a reciprocal off by 2^-24 of itself), and the correction by the exact remainder adds the
reciprocal's error of that, at most 1.5 * 2^-24 units (2^-20 more of it, for a reciprocal that is itself
rounded to the wrong side). A result can be wrong only where |K| / (2 D) is less, so where |K| is at most 3:
for each D, the M that solve K = 1, -1, 2, -2, 3 or -3 modulo D.
"""

import pytest
import torch

import fussim_b200 as fb

pytestmark = pytest.mark.gpu

CHUNK = 1 << 21


def inverse_of_power(n, d):
    """2^-n modulo odd numbers d (below 2^24: products stay below 2^63)."""
    base, out = (d + 1) // 2, torch.ones_like(d)
    while n:
        if n & 1:
            out = out * base % d
        base, n = base * base % d, n >> 1
    return out


def quotients(m, d):
    """m / d of mantissas as the step forms them: moments are halved exactly, the root of a rounded square
    is the number itself, eps adds nothing, and a rate of 1 leaves a parameter of zero at minus the quotient."""
    m, d = m.float() * 2.0 ** -23, d.float() * 2.0 ** -23
    p = torch.zeros_like(m)
    fb.adamw_step_([p], [torch.zeros_like(m)], [m * 2.0], [d * d * 2.0], step=200, lr=1.0, betas=(0.5, 0.5),
                   eps=2.0 ** -60, weight_decay=0.0)
    return -p


def check(m, d):
    want = (m.double() / d.double()).float()  # (53 bits are enough for the quotient's one rounding to 24)
    bad = (quotients(m, d) != want).nonzero().flatten()[:4]
    assert not len(bad), [(int(m[i]), int(d[i])) for i in bad]


@pytest.mark.parametrize("k", [1, -1, 2, -2, 3, -3])
def test_next_to_a_border(k):
    found = 0
    for first in range(1 << 23, 1 << 24, CHUNK):
        d = torch.arange(first, first + CHUNK, device="cuda", dtype=torch.int64)
        for s in (23, 24):
            # for odd d; for even ones everything is divided by two once (k odd has no solution there, and after
            # it d has to be odd)
            for halved in (False, True):
                if halved and k % 2:
                    continue
                e = d[d % 4 == 2] if halved else d[d % 2 == 1]
                mod, rest, power = (e // 2, k // 2, s) if halved else (e, k, s + 1)
                m0 = (rest * inverse_of_power(power, mod)) % mod
                for j in range(4 if halved else 2):
                    m = m0 + j * mod
                    good = (m >= 1 << 23) & (m < 1 << 24) & ((m < e) if s == 24 else (m >= e))
                    if good.any():
                        mm, dd = m[good], e[good]
                        n = (mm * (1 << (s + 1)) - k) // dd
                        assert (mm * (1 << (s + 1)) - n * dd == k).all()
                        check(mm, dd)
                        found += len(mm)
    # an M modulo d is one of 2^23 in d on average: 2^22 ln 2 = 2.907 million in all of the odd d
    assert found > 2_900_000


def test_powers_of_two_by_all_ones():
    """A reciprocal next to a border itself."""
    d = torch.tensor([(1 << 24) - 1, (1 << 24) - 2, (1 << 24) - 3, (1 << 23) + 1, 1 << 23], device="cuda")
    for m in (1 << 23, (1 << 23) + 1, (1 << 24) - 1, (1 << 24) - 2):
        check(torch.full_like(d, m), d)


def test_other_magnitudes():
    """Random mantissas and exponents over the range of the step's short way, and eps that counts."""
    g = torch.Generator(device="cuda").manual_seed(4)
    n = 1 << 22
    for eps in (2.0 ** -60, 1e-8, 1e-3):
        for _ in range(4):
            m = torch.randn(n, device="cuda", generator=g) * torch.exp2(torch.randint(-70, 79, (n,), device="cuda", generator=g).float())
            d = (1 + torch.rand(n, device="cuda", generator=g)) * torch.exp2(torch.randint(-39, 39, (n,), device="cuda", generator=g).float())
            p = torch.zeros_like(m)
            fb.adamw_step_([p], [torch.zeros_like(m)], [m * 2.0], [d * d * 2.0], step=200, lr=1.0, betas=(0.5, 0.5), eps=eps,
                           weight_decay=0.0)
            want = (m.double() / (d.double() + torch.tensor(eps).double()).float().double()).float()
            assert torch.equal(-p, want)
