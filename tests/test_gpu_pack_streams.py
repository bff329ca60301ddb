"""A packed cache made on one stream and used on another."""

import pytest

torch = pytest.importorskip("torch")

from test_gpu_pack import Setup  # noqa: E402


@pytest.mark.gpu
def test_a_cache_is_ready_on_every_stream_when_it_is_made(igc_lib):
    """The word that tells of trouble is clear before the first call, whatever
    is queued on the stream the cache was made on, and stays what a call on
    another stream set."""
    s = Setup(igc_lib, "bf16", [1], [10], 8, 1, 64, seed=3)
    c, far = s.cache, s.fills + 1000
    side, busy = torch.cuda.Stream(), torch.empty(1 << 28, device="cuda")
    s.attend()
    torch.cuda.synchronize()
    for _ in range(3):
        for _ in range(30):
            busy.normal_()
        made = igc_lib.PackCache(c.key_codes, c.key_scales, c.value_codes, c.value_scales)
        with torch.cuda.stream(side):
            made.attend(s.q, far, slots=s.slots, scale=0.125)
        torch.cuda.synchronize()
        with pytest.raises(igc_lib.IgcError) as e:
            made.status()
        assert e.value.code == igc_lib.FAIL_STATE
