"""Attention over the packed cache where values are small, and where first
positions hold most of a row's weight: the weights and values of the products
have to keep their bits there.

Every product's operands are f16.  A value (code - 8) scale is a whole number
of 2^-24 and is rounded by 2^-11 of itself at most, whatever its scale.  A
weight is kept times 2^h and so is rounded by 2^-11 of itself, or by 2^-25-h
of the row's largest where it is below 2^-14-h of it.  (32-bit rows keep the
rest of each beside it.)  Results then hold to test_gpu_pack's bounds, and

    2^-25-h sum |v_j|

more; h is 7 at least, where a row's first estimate of its largest is left
standing while the largest grows by up to 2^8.

Where a sequence has more than 16 query rows a key/value head, of 16 bits and at
most 256 wide, keys are rounded to f16 too, and the score of a position that
stands out is off by up to 2^-11 of it: the others' weights, and with them the
result, by that factor.

In the 2-norm f32 rows have the roundings of scores as large as `above`, each
2^-24 of its partials, beside the 4e-6 of test_gpu_pack: 2^-22 `above`."""

import math

import pytest

torch = pytest.importorskip("torch")

from test_gpu_pack import Setup, unpack64  # noqa: E402

KEPT = 7  # the least power of two a weight is kept times


def floor_of(s, window, sinks):
    """2^-25-h times the sum of the magnitudes a row sees, for each row."""
    c, group = s.cache, s.heads // s.kv
    out = torch.zeros(s.total, s.heads, s.size, dtype=torch.float64, device="cuda")
    first = 0
    for slot, n, f in zip(s.slot_list, s.rows, s.fill):
        for h in range(s.kv):
            v = unpack64(c.value_codes[slot, h, :f + n], c.value_scales[slot, h, :f + n]).abs().nan_to_num(0.0)
            for i in range(n):
                p = f + i
                low = max(0, p - window + 1) if window else 0
                total = v[low:p + 1].sum(0) + v[:min(sinks, low)].sum(0)
                out[first + i, h * group:(h + 1) * group] = total * 2.0 ** (-25 - KEPT)
        first += n
    return out


def check(s, window=0, sinks=0, above=0.0, rounded_keys=False):
    got = s.attend(window=window, sinks=sinks).double()
    want, tol = s.want(window, sinks)
    tol = tol + floor_of(s, window, sinks)
    assert torch.isfinite(got).all()
    over = ((got - want).abs() / tol).max().item()
    rel = ((got - want).norm() / want.norm()).item()
    norm = {torch.float32: 4e-6 + 2.0 ** -22 * above, torch.float16: 2.0 ** -11, torch.bfloat16: 2.3e-3}[s.kind]
    if rounded_keys and s.kind != torch.float32:
        norm += math.expm1(2.0 ** -11 * above)
    assert over <= 1.0 and rel <= norm, (over, rel)
    s.cache.status()


# rows a sequence, depth, heads, size: few units and a short cache; one token cut over many blocks; more rows of wide heads
FEW = [(1, 1000, 8, 256), (1, 1000, 3, 96), (1, 20011, 4, 128), (12, 20011, 2, 512), (3, 20011, 7, 320)]
MANY = [(4, 20011, 8, 256), (4, 20011, 8, 64), (40, 17001, 8, 96)]  # more than 16 rows a key/value head: tcgen05


@pytest.mark.gpu
@pytest.mark.parametrize("rows,depth,heads,size", FEW + MANY)
@pytest.mark.parametrize("kind,step", [("f32", 1e-4), ("f32", 2.0 ** -24), ("bf16", 1e-4), ("bf16", 1e-6),
                                       ("bf16", 2.0 ** -24), ("f16", 2.0 ** -8)])
def test_values_of_any_size(igc_lib, kind, step, rows, depth, heads, size):
    s = Setup(igc_lib, kind, [rows], [depth], heads, 1, size, seed=size + rows)
    s.cache.value_scales.fill_(step)
    check(s)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,depth,heads,size", FEW)
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("above,window", [(10, 0), (14, 0), (14, 900)])
def test_first_positions_that_hold_the_weight(igc_lib, kind, above, window, rows, depth, heads, size):
    """Four first positions stand `above` the others in score, and their values
    are zeros: the result is what the others leave."""
    s = Setup(igc_lib, kind, [rows], [depth], heads, 1, size, seed=size + rows + above)
    stand_out(s, above)
    check(s, window=window, sinks=4 if window else 0, above=above)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,heads,size", [(40, 8, 256), (40, 8, 64), (24, 16, 128), (20, 7, 160)])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("above", [10, 14])
def test_first_positions_that_hold_the_weight_of_many_rows(igc_lib, kind, above, rows, heads, size):
    """More units than blocks, so that most see the first positions and the
    window behind them together."""
    s = Setup(igc_lib, kind, [rows] * 60, [1400 + 7 * i for i in range(60)], heads, 1, size, seed=size + above)
    stand_out(s, above)
    check(s, window=900, sinks=4, above=above, rounded_keys=True)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,depth,heads,size", FEW + MANY)
def test_first_positions_far_above_in_32_bits(igc_lib, rows, depth, heads, size):
    s = Setup(igc_lib, "f32", [rows], [depth], heads, 1, size, seed=size + rows)
    stand_out(s, 20)
    check(s, above=20)


def stand_out(s, above):
    """Columns 0 to 31 of every query are 1, and of the keys 7 scale in the
    first four positions and 0 in the others."""
    c = s.cache
    s.q[:, :, :32] = 1.0
    s.q[:, :, 32:] *= 0.3
    for slot in s.slot_list:
        c.key_codes[slot, :, :, :16] = 0x88
        c.key_codes[slot, :, :4, :16] = 0xFF
        c.key_scales[slot, :, :4, 0] = above / (7 * 32 * s.size ** -0.5)
        c.value_codes[slot, :, :4] = 0x88
