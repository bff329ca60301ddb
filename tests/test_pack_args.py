"""The packed cache's entries check their arguments before any device call."""

import ctypes

import pytest


def _pack(lib, **kw):
    v = dict(key_codes=4096, key_scales=8192, value_codes=12288, value_scales=16384, slot_count=2, head_count=2,
             position_count=128, head_size=64, device=0, trouble=None)
    v.update(kw)
    return lib.IgcPack(*(v[n] for n, _ in lib.IgcPack._fields_))


def _rows(lib, **kw):
    v = dict(count=2, row_count=4, rows_most=0, start_list=256, fill_list=512, slot_list=768)
    v.update(kw)
    return lib.IgcPackRows(*(v[n] for n, _ in lib.IgcPackRows._fields_))


def _data(lib, **kw):
    v = dict(data=65536, real_type=3, row_stride=128, head_stride=64)
    v.update(kw)
    return lib.IgcPackData(*(v[n] for n, _ in lib.IgcPackData._fields_))


BAD_PACK = [dict(key_codes=None), dict(value_scales=None), dict(key_codes=4104), dict(slot_count=0),
            dict(head_count=0), dict(position_count=100), dict(position_count=0), dict(head_size=48),
            dict(head_size=0), dict(head_size=544), dict(device=-1)]
BAD_ROWS = [dict(count=0), dict(row_count=-1), dict(fill_list=None), dict(rows_most=-1),
            dict(start_list=None, row_count=3), dict(slot_list=None, count=3, row_count=3)]
BAD_DATA = [dict(data=None), dict(real_type=0), dict(real_type=4), dict(data=65537), dict(row_stride=-1),
            dict(head_stride=-64), dict(real_type=1, data=65538)]


@pytest.mark.parametrize("pack,rows,data", [(b, {}, {}) for b in BAD_PACK] + [({}, b, {}) for b in BAD_ROWS] +
                         [({}, {}, b) for b in BAD_DATA])
def test_bad_arguments_are_refused(igc_lib, pack, rows, data):
    lib = igc_lib._lib()
    p, r, d, good = _pack(igc_lib, **pack), _rows(igc_lib, **rows), _data(igc_lib, **data), _data(igc_lib)
    size = ctypes.c_size_t(77)
    assert lib.igc_pack_write(p, r, d, good, None) == igc_lib.FAIL_ARGUMENT
    assert lib.igc_pack_write(p, r, good, d, None) == igc_lib.FAIL_ARGUMENT
    assert lib.igc_pack_read(p, r, d, good, None) == igc_lib.FAIL_ARGUMENT
    assert lib.igc_pack_read(p, r, good, d, None) == igc_lib.FAIL_ARGUMENT
    assert lib.igc_pack_attend(p, r, 8, d, good, 0, 0, 1.0, None, 0, None) == igc_lib.FAIL_ARGUMENT
    assert lib.igc_pack_attend(p, r, 8, good, d, 0, 0, 1.0, None, 0, None) == igc_lib.FAIL_ARGUMENT
    if not data:
        assert lib.igc_pack_attend_room(p, r, 8, 3, 0, 0, size) == igc_lib.FAIL_ARGUMENT and size.value == 77
    if pack:
        assert lib.igc_pack_status(p, None) == igc_lib.FAIL_ARGUMENT


def test_bad_attention_is_refused(igc_lib):
    lib = igc_lib._lib()
    p, r, d = _pack(igc_lib), _rows(igc_lib), _data(igc_lib)
    inf, nan = float("inf"), float("nan")
    for heads, window, sinks, scale, work in ((0, 0, 0, 1.0, None), (3, 0, 0, 1.0, None), (1, 0, 0, 1.0, None),
                                              (-2, 0, 0, 1.0, None), (8, -1, 0, 1.0, None), (8, 0, -1, 1.0, None),
                                              (8, 0, 0, inf, None), (8, 0, 0, nan, None), (8, 0, 0, 1.0, 4104)):
        assert lib.igc_pack_attend(p, r, heads, d, d, window, sinks, scale, work, 0, None) == igc_lib.FAIL_ARGUMENT
    size = ctypes.c_size_t()
    assert lib.igc_pack_attend(p, r, 8, d, _data(igc_lib, real_type=2), 0, 0, 1.0, None, 0, None) == \
        igc_lib.FAIL_ARGUMENT
    for heads, kind, window, sinks in ((3, 3, 0, 0), (8, 0, 0, 0), (8, 4, 0, 0), (8, 3, -1, 0), (8, 3, 0, -1)):
        assert lib.igc_pack_attend_room(p, r, heads, kind, window, sinks, size) == igc_lib.FAIL_ARGUMENT
    assert lib.igc_pack_attend_room(p, r, 8, 3, 0, 0, None) == igc_lib.FAIL_ARGUMENT
    for call in (lib.igc_pack_write, lib.igc_pack_read):
        assert call(None, r, d, d, None) == igc_lib.FAIL_ARGUMENT
        assert call(p, None, d, d, None) == igc_lib.FAIL_ARGUMENT
        assert call(p, r, None, d, None) == igc_lib.FAIL_ARGUMENT


def test_keys_and_values_have_one_type(igc_lib):
    lib = igc_lib._lib()
    p, r, d = _pack(igc_lib), _rows(igc_lib), _data(igc_lib)
    for call in (lib.igc_pack_write, lib.igc_pack_read):
        assert call(p, r, d, _data(igc_lib, real_type=2), None) == igc_lib.FAIL_ARGUMENT


def test_no_rows_is_no_call(igc_lib):
    lib = igc_lib._lib()
    p, d = _pack(igc_lib), _data(igc_lib)
    r = _rows(igc_lib, row_count=0)
    size = ctypes.c_size_t(5)
    assert lib.igc_pack_write(p, r, d, d, None) == igc_lib.OKAY
    assert lib.igc_pack_read(p, r, d, d, None) == igc_lib.OKAY
    assert lib.igc_pack_attend_room(p, r, 8, 3, 0, 0, size) == igc_lib.OKAY and size.value == 0
    assert lib.igc_pack_attend(p, r, 8, d, d, 0, 0, 1.0, None, 0, None) == igc_lib.OKAY


def test_a_cache_is_made_of_cuda_tensors(igc_lib):
    torch = pytest.importorskip("torch")
    codes, scales = torch.zeros(1, 1, 64, 32, dtype=torch.uint8), torch.zeros(1, 1, 64, 2, dtype=torch.float16)
    with pytest.raises(ValueError):
        igc_lib.PackCache(codes, scales, codes, scales)
    with pytest.raises(ValueError):
        igc_lib.PackCache(codes, scales.float(), codes, scales)
    with pytest.raises(ValueError):
        igc_lib.PackCache(codes[0], scales, codes, scales)


def test_packed_session_refuses_bad_arguments(igc_lib):
    lib, out = igc_lib._lib(), ctypes.c_void_p(1)
    assert lib.igc_session_open_packed(None, 0, ctypes.byref(out)) == igc_lib.FAIL_ARGUMENT
    assert lib.igc_session_open_packed(None, -1, ctypes.byref(out)) == igc_lib.FAIL_ARGUMENT
    assert lib.igc_session_open_packed(None, 0, None) == igc_lib.FAIL_ARGUMENT


def test_arrays_that_are_written_have_places_of_their_own(igc_lib):
    lib = igc_lib._lib()
    p, r, good = _pack(igc_lib), _rows(igc_lib), _data(igc_lib)
    for kw in (dict(row_stride=0), dict(head_stride=0), dict(row_stride=good.head_stride), dict(head_stride=16)):
        bad = _data(igc_lib, **kw)
        assert lib.igc_pack_read(p, r, bad, good, None) == igc_lib.FAIL_ARGUMENT
        assert lib.igc_pack_read(p, r, good, bad, None) == igc_lib.FAIL_ARGUMENT
        assert lib.igc_pack_attend(p, r, 8, good, bad, 0, 0, 1.0, None, 0, None) == igc_lib.FAIL_ARGUMENT


def test_places_are_counted_in_ints(igc_lib):
    lib, r, d = igc_lib._lib(), _rows(igc_lib), _data(igc_lib)
    p = _pack(igc_lib, slot_count=64, position_count=(1 << 24) + 64)
    assert lib.igc_pack_write(p, r, d, d, None) == igc_lib.FAIL_ARGUMENT
