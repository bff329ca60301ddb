"""Attention over the packed cache in the forms that share one list of tiles:
tcgen05 for more than 16 16-bit query rows a key/value head up to 256 wide,
blocks of 32 rows for 32-bit rows and for 512-wide heads.  Every case here has
more units than the device takes as clusters, and asserts the form that its
scratch tells.  Bounds are those of test_gpu_pack (Setup.check)."""

import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_gpu_pack import Setup  # noqa: E402

SEQS = 40
TC = [("f16", 8, 1, 32), ("bf16", 8, 1, 64), ("f16", 8, 2, 96), ("bf16", 21, 3, 128), ("f16", 16, 2, 160),
      ("bf16", 8, 1, 256), ("f16", 8, 1, 256)]
TALL = [("f32", 8, 1, 64), ("f32", 12, 1, 128), ("f32", 8, 1, 256), ("f32", 8, 1, 96), ("f16", 8, 1, 512),
        ("bf16", 8, 1, 416)]


def block_rows(lib, s, window=0, sinks=0):
    """The query rows of a block, by the scratch a call needs: a block leaves at
    most two pieces of rows x (size + 2) floats, and 8 words."""
    room = ctypes.c_size_t()
    rows = lib.IgcPackRows(len(s.rows), s.total, max(s.rows), s.starts.data_ptr(), s.fills.data_ptr(),
                           s.slots.data_ptr())
    kind = {torch.float32: 1, torch.float16: 2, torch.bfloat16: 3}[s.kind]
    assert lib._lib().igc_pack_attend_room(s.cache._p, rows, s.heads, kind, window, sinks, room) == 0
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    found = [rb for rb in (8, 16, 32, 128)
             if room.value % (4 * (8 + 2 * rb * (s.size + 2))) == 0 and
             1 < room.value // (4 * (8 + 2 * rb * (s.size + 2))) <= (1 if rb == 128 else 4) * sms]
    assert len(found) == 1, (room.value, found)
    return found[0]


def ragged(lib, kind, heads, kv, size, seed, padding=True, tail=3):
    """Sequences of 0 to 45 rows at depths about tiles' edges, two of them padding."""
    g = np.random.default_rng(seed)
    rows = [int(x) for x in g.integers(17, 46, SEQS)]
    fill = [int(x) for x in g.choice([0, 1, 19, 47, 63, 64, 90, 127, 128, 200, 257], SEQS)]
    rows[3] = 0
    if padding:
        fill[5], fill[6] = -rows[5], -5
    return Setup(lib, kind, rows, fill, heads, kv, size, seed=seed, extra=1, tail=tail)


def run(lib, s, form, window=0, sinks=0):
    assert block_rows(lib, s, window, sinks) == form
    n = sum(s.rows)
    out = s.attend(window=window, sinks=sinks, rows_most=max(s.rows), out=torch.full_like(s.q, 7.0))
    assert (out[n:] == 7.0).all()  # rows behind the last sequence
    s.check(out, window, sinks)
    return out


SIGHT = [(0, 0), (1, 0), (1, 1), (16, 4), (64, 64), (100, 70), (1000, 5)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind,heads,kv,size", TC)
@pytest.mark.parametrize("window,sinks", SIGHT)
def test_tcgen05_rows_in_sight(igc_lib, kind, heads, kv, size, window, sinks):
    s = ragged(igc_lib, kind, heads, kv, size, seed=size + window)
    run(igc_lib, s, 128, window, sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,heads,kv,size", TALL)
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 1), (100, 70)])
def test_rows_in_sight_of_32_row_blocks(igc_lib, kind, heads, kv, size, window, sinks):
    s = ragged(igc_lib, kind, heads, kv, size, seed=size + window)
    run(igc_lib, s, 16 if kind == "f32" and size > 256 else 32, window, sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,heads,kv,size", TC + TALL[:3])
def test_places_out_of_sight_may_hold_anything(igc_lib, kind, heads, kv, size):
    """Positions that have left every row's window are NaN."""
    s = ragged(igc_lib, kind, heads, kv, size, seed=2, padding=False)
    window, sinks = 33, 2
    for slot, f in zip(s.slot_list, s.fill):
        for scales in (s.cache.key_scales, s.cache.value_scales):
            scales[slot, :, sinks:max(sinks, f - window + 1)] = float("nan")
    run(igc_lib, s, 128 if kind != "f32" else 32, window, sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,heads,kv,size", TC + TALL)
def test_rows_of_other_strides(igc_lib, kind, heads, kv, size):
    """Rows off 16-byte boundaries, heads outermost, and results between others:
    the same bits."""
    s = ragged(igc_lib, kind, heads, kv, size, seed=4)
    n, window, sinks = sum(s.rows), 70, 3
    want = s.attend(window=window, sinks=sinks, rows_most=max(s.rows))[:n]
    s.check(want, window, sinks)
    q = torch.zeros(s.total, heads, size + 3, dtype=s.kind, device="cuda")[:, :, 1:size + 1]
    q.copy_(s.q)
    by_head = s.q.transpose(0, 1).contiguous().transpose(0, 1)
    for rows in (q, by_head):
        out = torch.zeros(s.total, heads + 1, size + 1, dtype=s.kind, device="cuda")
        got = s.attend(q=rows, window=window, sinks=sinks, rows_most=max(s.rows), out=out[:, 1:, 1:])
        assert torch.equal(got[:n], want) and out[:, 0].abs().max() == 0 and out[:, :, 0].abs().max() == 0
        assert got[n:].abs().max() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("kind,heads,kv,size", [t for t in TC if t[0] == "bf16"])
def test_tcgen05_extreme_rows(igc_lib, kind, heads, kv, size):
    """Tiny queries, a row of zeros, a NaN row that stays its own, the largest
    and the smallest scales, and a negative factor."""
    s = ragged(igc_lib, kind, heads, kv, size, seed=6)
    s.q[0] *= 1e-30
    s.q[1] = 0
    s.cache.value_scales[s.slot_list[7], :, 4] = 8188.0
    s.cache.value_scales[s.slot_list[8], :, :] = s.cache.value_scales[s.slot_list[8], :, :] * 2.0 ** -22
    s.check(s.attend(rows_most=max(s.rows)))
    n = sum(s.rows)
    for scale in (-0.05, 0.0):
        got = s.attend(rows_most=max(s.rows), scale=scale)
        want, tol = s.want(scale=abs(scale), q=-s.q)  # the bound's terms are magnitudes
        assert ((got - want).abs() <= tol)[:n].all()
    before = s.attend(rows_most=max(s.rows))
    s.q[2, 1, 5] = float("nan")
    after = s.attend(rows_most=max(s.rows))
    assert torch.isnan(after[2, 1]).all()
    after[2, 1] = before[2, 1]
    assert torch.equal(after[:n], before[:n])


@pytest.mark.gpu
@pytest.mark.parametrize("kind,heads,kv,size", [TC[1], TC[3], TC[5], TALL[2], TALL[4]])
def test_two_streams_and_a_graph(igc_lib, kind, heads, kv, size):
    """The same bits eager, on two streams at once, and captured and replayed."""
    s = ragged(igc_lib, kind, heads, kv, size, seed=7)
    n = sum(s.rows)
    call = lambda: s.attend(rows_most=max(s.rows))[:n]  # noqa: E731
    want = call()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for st in streams:
            with torch.cuda.stream(st):
                got.append(call())
        torch.cuda.synchronize()
        assert torch.equal(got[0], want) and torch.equal(got[1], want)
    graphs, outs = [], []
    for st in streams:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            outs.append(call())
        graphs.append(g)
    for _ in range(10):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for st, g in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
