"""Sessions whose caches hold 4-bit codes (igc_session_open_packed): the model's
own passes through the packed cache's operators, against the CPU restatement
with the same quantisation.

What a group of 32 values is stored as jumps where its scale (a half, 2^-11
of it apart) or a code comes to a rounding tie, and a jump can move the logits
of its own row by whole units.  The two sides' float rows differ by about 1e-6
of their values, in the order of their sums, so about 1 group in 100 is in
doubt, whichever side is right.  The tokens are therefore drawn by the
restatement alone, each so that none of its row's groups is within 4e-6 of a
tie; the logits then agree to the parity tests' absolute bar of 2e-2."""

import numpy as np
import pytest

from conftest import CACHED, EXPORT, SMALL, TINY

pytestmark = pytest.mark.gpu
ATOL = 2e-2

SHAPES = {"tiny": TINY, "small": SMALL, "cached": CACHED}


class Drawn:
    """The restatement's session, and a second one that draws tokens ahead."""

    def __init__(self, igo, folder, cfg, sinks, seed):
        om = igo.OracleModel(folder, window_limit=cfg["window_limit"])
        self.o = igo.OracleSession(om, threads=8, packed=True, sinks=sinks)
        self.ahead = igo.OracleSession(om, threads=8, packed=True, sinks=sinks)
        self.rng, self.vocab = np.random.default_rng(seed), cfg["vocab"]

    def tokens(self, n):
        """n tokens for the places after the session's fill."""
        a, out = self.ahead, []
        a.hold(self.o.fill)
        while len(out) < n:
            fill = a.fill
            t = int(self.rng.integers(0, self.vocab))
            a.step(t)
            if a.doubts():
                a.hold(fill)
            else:
                out.append(t)
        return np.array(out, np.int32)


def _close(got, want):
    err = float(np.abs(got - want).max())
    assert err <= ATOL, err


@pytest.mark.parametrize("sinks", [0, 3])
@pytest.mark.parametrize("which", ["tiny", "small", "cached"])
def test_passes_against_the_restatement(igc_lib, igo_mod, which, sinks, tiny_dir, small_dir, cached_dir):
    cfg = SHAPES[which]
    folder = {"tiny": tiny_dir, "small": small_dir, "cached": cached_dir}[which]
    d = Drawn(igo_mod, folder, cfg, sinks, 2)
    o = d.o
    m = igc_lib.Model(folder=folder, window_limit=cfg["window_limit"])
    s = igc_lib.Session(m, packed=True, sinks=sinks)
    ids = d.tokens(77)  # past every sliding window, ending inside a tile
    s.prime(ids)
    o.prime(ids)
    for k in (1, 4, 9, 16):
        blk = d.tokens(k)
        _close(s.guess(blk), o.guess(blk))
        s.guess_keep(min(k, 5))
        o.guess_keep(min(k, 5))
        assert s.fill == o.fill
        t = d.tokens(1)[0]
        _close(s.step(t)[1], o.step(t))
    s.hold(60)
    o.hold(60)
    blk = d.tokens(6)
    _close(s.guess(blk), o.guess(blk))


@pytest.mark.parametrize("sinks", [0, 4])
def test_chunked_prime_against_the_restatement(igc_lib, igo_mod, cached_dir, sinks):
    """A prompt long enough for the batched-lane prime, its attention over the
    codes in one launch a layer, then a step and a block on top."""
    d = Drawn(igo_mod, cached_dir, CACHED, sinks, 3)
    o = d.o
    m = igc_lib.Model(folder=cached_dir, window_limit=CACHED["window_limit"])
    s = igc_lib.Session(m, packed=True, sinks=sinks)
    ids = d.tokens(300)
    s.prime(ids)
    o.prime(ids)
    t = d.tokens(1)[0]
    _close(s.step(t)[1], o.step(t))
    blk = d.tokens(4)
    _close(s.guess(blk), o.guess(blk))
    assert s.cache_peak(0, 0) > 0 and s.cache_peak(0, 1) > 0


def test_wide_heads_in_blocks_and_steps(igc_lib):
    """512-wide global heads.  A session's block against another's steps: each
    step rewrites the places the block's rows had, and a row in doubt between
    the two would show alone, so rows agree but for one in the block."""
    m = igc_lib.Model(spec=igc_lib.SynthSpec(**EXPORT), window_limit=EXPORT["window_limit"])
    ids = np.random.default_rng(5).integers(0, EXPORT["vocab"], 200).astype(np.int32)
    a, b = igc_lib.Session(m, packed=True, sinks=2), igc_lib.Session(m, packed=True, sinks=2)
    a.prime(ids)
    b.prime(ids)
    blk = np.array([11, 12, 13, 14, 15], np.int32)
    rows = a.guess(blk)
    off = [float(np.abs(b.step(t)[1] - rows[j]).max()) for j, t in enumerate(blk)]
    assert np.isfinite(off).all() and sorted(off)[-2] <= ATOL, off


def test_state_calls_and_refusals(igc_lib, small_dir, tmp_path):
    m = igc_lib.Model(folder=small_dir, window_limit=SMALL["window_limit"])
    s, plain = igc_lib.Session(m, packed=True, sinks=2), igc_lib.Session(m)
    # 0.5625 bytes a value against 4
    assert s.cache_room() * 64 == plain.cache_room() * 9
    ids = np.arange(5, 45, dtype=np.int32)
    s.prime(ids)
    first = s.step(ids[-1])[1]
    s.hold(len(ids) - 1)
    again = s.step(ids[-1])[1]
    assert np.array_equal(first, again)  # wound back, the same rows are written again
    take, made = s.round(np.array([again.argmax(), 1, 2], np.int32))
    assert 0 <= take <= 2 and 0 <= made < m.vocab
    with pytest.raises(igc_lib.IgcError) as e:
        s.save(str(tmp_path / "x.keep"))
    assert e.value.code == igc_lib.FAIL_SUPPORT
    plain.prime(ids)
    plain.save(str(tmp_path / "y.keep"))
    with pytest.raises(igc_lib.IgcError) as e:
        s.load(str(tmp_path / "y.keep"))
    assert e.value.code == igc_lib.FAIL_SUPPORT
    crowd = igc_lib.Crowd(m, 2, 2)
    fill = s.fill
    with pytest.raises(igc_lib.IgcError) as e:
        crowd.round([plain, s], np.zeros((2, 2), np.int32))
    assert e.value.code == igc_lib.FAIL_SUPPORT and s.fill == fill
    s.reset()
    s.prime(ids)
    assert np.array_equal(s.step(ids[-1])[1], first)
    with pytest.raises(igc_lib.IgcError) as e:
        igc_lib.Session(m, packed=True, sinks=-1)
    assert e.value.code == igc_lib.FAIL_ARGUMENT
    with pytest.raises(ValueError):
        igc_lib.Session(m, sinks=2)
