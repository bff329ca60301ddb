"""The packed cache's trouble word: what lists that do not fit set, in every
call, and what a status leaves behind."""

import ctypes

import pytest

torch = pytest.importorskip("torch")

from test_gpu_pack import Setup  # noqa: E402

# six rows; the list, the most rows of a sequence, and the rows that no sequence is run for
BAD = [([0, 2, 4, 7], None, [4, 5]), ([0, 2, 4, 6, 9], None, []), ([0, 6, 2], None, []), ([0, 4, 2, 6], None, []),
       ([0, 1, 5, 6], 3, [1, 2, 3, 4]), ([-1, 2, 4, 6], None, [0, 1]), ([0, 6, 6, 8], None, []),
       ([0] + [6] * 400 + [7], None, [])]


@pytest.mark.gpu
@pytest.mark.parametrize("starts,most,left", BAD)
def test_lists_that_do_not_fit_are_told_by_every_call(igc_lib, starts, most, left):
    n = len(starts) - 1
    s = Setup(igc_lib, "bf16", [2, 2, 2], [10, 30, 20], 8, 1, 64, seed=1)
    at = dict(starts=torch.tensor(starts, dtype=torch.int32, device="cuda"), rows_most=most,
              slots=s.slots[torch.arange(n, device="cuda") % 3].contiguous())
    fill = (torch.arange(n, dtype=torch.int32, device="cuda") % 3) * 10 + 5
    scales = s.cache.key_scales.clone()
    s.cache.write(s.k, s.v, fill, **at)
    with pytest.raises(igc_lib.IgcError) as e:
        s.cache.status()
    assert e.value.code == igc_lib.FAIL_STATE
    s.cache.status()
    out = torch.full_like(s.k, 5.0), torch.full_like(s.k, 5.0)
    s.cache.read(fill, 6, torch.bfloat16, out=out, **at)
    with pytest.raises(igc_lib.IgcError):
        s.cache.status()
    assert (out[0][left] == 5.0).all() and (out[1][left] == 5.0).all()
    s.cache.attend(s.q, fill, scale=0.125, **at)
    with pytest.raises(igc_lib.IgcError):
        s.cache.status()
    if len(left) == 4:  # of the sequence with too many rows nothing was written
        slot = s.slot_list[1]
        assert torch.equal(s.cache.key_scales[slot].view(torch.int16), scales[slot].view(torch.int16))


@pytest.mark.gpu
def test_a_status_has_cleared_the_word_when_it_returns(igc_lib):
    """Its clearing does not reach into calls that come after it on other
    streams: nothing of it is left on its stream."""
    s = Setup(igc_lib, "bf16", [1], [10], 8, 1, 64, seed=2)
    lib, stream = igc_lib._lib(), torch.cuda.current_stream()
    for _ in range(300):
        s.cache._trouble.fill_(1)
        code = lib.igc_pack_status(s.cache._p, stream.cuda_stream)
        idle = stream.query()
        assert code == igc_lib.FAIL_STATE and idle
        assert lib.igc_pack_status(s.cache._p, stream.cuda_stream) == igc_lib.OKAY


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [4, 600])
def test_starts_back_and_forth_do_not_multiply_the_work(igc_lib, kind, rows):
    """Every second sequence holds all rows: a list of 2^31 tiles and more from
    a call whose sizes allow a few thousand.  None of it is run, and it is told."""
    heads, n = 8, 40000
    cache = igc_lib.PackCache.open(1, heads, 1 << 20, 32)
    dtype = {"f32": torch.float32, "bf16": torch.bfloat16}[kind]
    q = torch.randn(rows, 5 * heads, 32, device="cuda").to(dtype)
    starts = torch.zeros(n + 1, dtype=torch.int32, device="cuda")
    starts[1::2] = rows
    at = dict(starts=starts, slots=torch.zeros(n, dtype=torch.int32, device="cuda"))
    fill = torch.full((n,), (1 << 20) - rows, dtype=torch.int32, device="cuda")
    out = cache.attend(q, fill, out=torch.full_like(q, 5.0), **at)
    with pytest.raises(igc_lib.IgcError) as e:
        cache.status()
    assert e.value.code == igc_lib.FAIL_STATE and (out == 5.0).all()
    out = cache.attend(q, fill[:1], starts=starts[:2].contiguous(), slots=at["slots"][:1], out=out)
    cache.status()
    assert out.abs().max() == 0  # a cleared cache


@pytest.mark.gpu
def test_a_call_of_too_many_tiles_is_refused_as_such(igc_lib):
    """2^24 rows over 2^20 positions of 8 heads: no pointer is followed."""
    pack = igc_lib.IgcPack(4096, 4096, 4096, 4096, 1, 8, 1 << 20, 64, 0, None)
    room = ctypes.c_size_t(5)
    for rows, want in ((1 << 24, igc_lib.FAIL_SUPPORT), (1 << 12, igc_lib.OKAY)):
        r = igc_lib.IgcPackRows(1, rows, 0, None, 4096, None)
        for kind in (1, 2, 3):
            assert igc_lib._lib().igc_pack_attend_room(pack, r, 8, kind, 0, 0, room) == want
