"""The packed cache's operators (igc_pack_*, PackCache) on the GPU against
plain 64-bit restatements of their formulas.

Tolerances, set from the arithmetic:

* Codes and scales are IEEE f32 divisions, one f16 rounding and one rint:
  equal to numpy's to the bit.
* A score is a sum of exact products (code x query, f16 or its hi/lo halves)
  per 32-column group, from -8 sum q, times the group's f32 scale: with C
  groups at most C + 8 roundings of partials no larger than
  b = scale * sum |q| * 23 * step, 2^-23 each, so a score is off by at most
  d = b (C + 8) 2^-23 and a weight by a factor e^(+-2d) after the division.
* Where a sequence has more than 16 query rows a key/value head, of 16 bits and
  at most 256 wide, keys are operands rounded to f16: a product is off by at
  most 2^-11 of it, so a score by 2^-11 scale sum |q||k| more, and a weight by
  twice that as a factor.
* 16-bit rows: weights and values are each rounded to f16 (2^-11 of each), the
  result to its type (eps / 2).  f32 rows: hi/lo splits leave out 2^-21.
* In the 2-norm these roundings are independent and uniform: h / sqrt(3) each.
  For f32 rows a score's partials add as a random walk, about
  sqrt(C + 8) 2^-24 of scale * sqrt(size) * 8 step |q| (3.2 here): 8e-7, which
  the bound of 4e-6 holds with room for the weights' and values' 2^-21.
"""

import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

KINDS = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def np_pack(x):
    """(codes [.., size/2], scales) of float32 rows, in numpy's IEEE arithmetic."""
    x = np.asarray(x, np.float32)
    g = x.reshape(*x.shape[:-1], -1, 32)
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        big = np.where(np.isnan(g), np.float32(0), np.abs(g)).max(-1)
        scale = np.minimum(big / np.float32(7), np.float32(8188)).astype(np.float16)
        step = scale.astype(np.float32)[..., None]
        n = np.where((step > 0) & ~np.isnan(g), np.rint(g / np.where(step > 0, step, np.float32(1))), np.float32(0))
    n = (np.clip(n, -8, 7) + 8).astype(np.uint8).reshape(x.shape)
    return n[..., 0::2] | (n[..., 1::2] << 4), scale


def unpack64(codes, scales):
    n = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).double() - 8
    return n * scales.double().repeat_interleave(32, -1)


class Setup:
    """A cache with every place the sequences do not reach left as NaN scales
    and random codes, as memory that nothing was written to may hold."""

    def __init__(self, lib, kind, rows, fill, heads, kv, size, seed=0, extra=0, tail=0, slots=None, shuffle=True):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        self.kind, self.rows, self.fill, self.heads, self.kv, self.size = KINDS[kind], rows, fill, heads, kv, size
        most = max([f + n for f, n in zip(fill, rows)] + [1])
        self.n_slots = (slots or len(rows)) + extra
        self.cache = lib.PackCache.open(self.n_slots, kv, most + extra * 64, size)
        c = self.cache
        for codes, scales in ((c.key_codes, c.key_scales), (c.value_codes, c.value_scales)):
            codes.random_(0, 256, generator=g)
            scales.fill_(float("nan"))
        order = torch.randperm(self.n_slots, generator=g, device="cuda")[:len(rows)] if shuffle else \
            torch.arange(len(rows), device="cuda")
        self.slots = order.to(torch.int32)
        self.slot_list = order.tolist()
        for s, (n, f) in enumerate(zip(rows, fill)):
            end = max(f + n, 0)
            for scales in (c.key_scales, c.value_scales):
                part = scales[self.slot_list[s], :, :end]
                part.copy_(torch.rand(part.shape, generator=g, device="cuda") * 0.5 + 0.1)
        self.total = sum(rows) + tail
        starts = np.concatenate([[0], np.cumsum(rows)])
        self.starts = torch.tensor(starts, dtype=torch.int32, device="cuda")
        self.fills = torch.tensor(fill, dtype=torch.int32, device="cuda")
        self.q = torch.randn(self.total, heads, size, generator=g, device="cuda").to(self.kind)
        self.k = (torch.randn(self.total, kv, size, generator=g, device="cuda") * 2).to(self.kind)
        self.v = torch.randn(self.total, kv, size, generator=g, device="cuda").to(self.kind)

    def attend(self, window=0, sinks=0, scale=None, **kw):
        return self.cache.attend(kw.pop("q", self.q), self.fills, starts=self.starts, slots=self.slots, window=window,
                                 sinks=sinks, scale=self.size ** -0.5 if scale is None else scale, **kw)

    def want(self, window=0, sinks=0, scale=None, q=None):
        """The formula in 64 bits: (result, its bound), for the sequences' rows."""
        scale = self.size ** -0.5 if scale is None else scale
        q = (self.q if q is None else q).double()
        c, group = self.cache, self.heads // self.kv
        out = torch.zeros(self.total, self.heads, self.size, dtype=torch.float64, device="cuda")
        tol = torch.zeros_like(out)
        first = 0
        for s, (n, f) in enumerate(zip(self.rows, self.fill)):
            end = f + n
            for i in range(n if end > 0 else 0):
                p = f + i
                if p < 0 or p >= c.positions:
                    continue
                see = [j for j in range(p + 1) if not window or j > p - window or j < sinks]
                at = torch.tensor(see, device="cuda")
                for h in range(self.kv):
                    k = unpack64(c.key_codes[self.slot_list[s], h, at], c.key_scales[self.slot_list[s], h, at])
                    v = unpack64(c.value_codes[self.slot_list[s], h, at], c.value_scales[self.slot_list[s], h, at])
                    step = c.key_scales[self.slot_list[s], h, at].double().repeat_interleave(32, -1)
                    qs = q[first + i, h * group:(h + 1) * group]
                    w = torch.softmax(qs @ k.T * scale, -1)
                    d = scale * (qs.abs() @ step.T).amax(-1) * 23 * (self.size // 32 + 8) * 2.0 ** -23
                    if max(self.rows) * group > 16 and self.size <= 256 and self.kind != torch.float32:
                        d += scale * (qs.abs() @ k.abs().T).amax(-1) * 2.0 ** -11 / 2
                    mass = w @ v.abs()
                    out[first + i, h * group:(h + 1) * group] = w @ v
                    each = 2.0 ** -10 + 2.0 ** -20 if self.kind != torch.float32 else 2.0 ** -19
                    tol[first + i, h * group:(h + 1) * group] = mass * (each + torch.expm1(4 * d).unsqueeze(-1))
            first += n
        tol += out.abs() * torch.finfo(self.kind).eps / 2 + 1e-30
        if self.kind == torch.float16:
            tol += 2.0 ** -25  # below f16's normal range
        return out, tol

    def check(self, got, window=0, sinks=0, scale=None, q=None):
        n = sum(self.rows)
        want, tol = self.want(window, sinks, scale, q)
        got, want, tol = got[:n].double(), want[:n], tol[:n]
        assert torch.isfinite(got).all()
        over = ((got - want).abs() / tol).max().item() if n else 0.0
        assert over <= 1.0, over
        norm = {torch.float32: 4e-6, torch.float16: 2.0 ** -11, torch.bfloat16: 2.3e-3}[self.kind]
        rel = ((got - want).norm() / want.norm().clamp(min=1e-30)).item()
        assert rel <= norm, rel
        self.cache.status()


# ---- rows written and read back

@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kv,size", [(1, 32), (1, 256), (3, 96), (2, 512), (8, 128)])
def test_written_codes_are_the_formulas_to_the_bit(igc_lib, kind, kv, size):
    s = Setup(igc_lib, kind, [1, 7, 0, 64, 33], [5, 0, 9, 63, 127], kv, kv, size, seed=size + kv, extra=1, tail=3)
    s.k[3] = 0  # groups of zeros
    s.k[5, :, :32] *= 1e-7  # scales below f16's normal range
    before = [t.clone() for t in (s.cache.key_codes, s.cache.key_scales, s.cache.value_codes, s.cache.value_scales)]
    s.cache.write(s.k, s.v, s.fills, starts=s.starts, slots=s.slots)
    s.cache.status()
    for rows, codes, scales, c0, s0 in ((s.k, s.cache.key_codes, s.cache.key_scales, before[0], before[1]),
                                        (s.v, s.cache.value_codes, s.cache.value_scales, before[2], before[3])):
        want_c, want_s = np_pack(rows.float().cpu().numpy())
        c1, s1 = c0.cpu().numpy(), s0.view(torch.uint16).cpu().numpy()
        first = 0
        for i, (n, f) in enumerate(zip(s.rows, s.fill)):
            c1[s.slot_list[i], :, f:f + n] = want_c[first:first + n].transpose(1, 0, 2)
            s1[s.slot_list[i], :, f:f + n] = want_s[first:first + n].view(np.uint16).transpose(1, 0, 2)
            first += n
        assert np.array_equal(codes.cpu().numpy(), c1)  # and every other place as it was
        assert np.array_equal(scales.view(torch.uint16).cpu().numpy(), s1)
    for dtype in KINDS.values():
        gk, gv = s.cache.read(s.fills, s.total, dtype, starts=s.starts, slots=s.slots)
        for got, rows in ((gk, s.k), (gv, s.v)):
            codes, scales = np_pack(rows.float().cpu().numpy())
            want = unpack64(torch.from_numpy(codes), torch.from_numpy(scales))[:sum(s.rows)]
            # a code of at most 4 bits times an f16 of 11 is exact in f32: one rounding to the type
            assert torch.equal(got[:sum(s.rows)].cpu(), want.float().to(dtype))


@pytest.mark.gpu
def test_write_saturates_and_keeps_the_cache_finite(igc_lib):
    c = igc_lib.PackCache.open(1, 1, 64, 64)
    x = torch.zeros(4, 1, 64, device="cuda")
    x[0, 0, 0], x[0, 0, 1], x[0, 0, 2] = float("inf"), -float("inf"), 5.0
    x[1, 0, 3], x[1, 0, 4] = float("nan"), 2.0
    x[2, 0, 5] = 3e38
    x[3, 0, :] = float("nan")
    fill = torch.zeros(1, dtype=torch.int32, device="cuda")
    c.write(x, x, fill)
    k, v = c.read(fill, 4, torch.float32)
    assert torch.equal(k, v) and torch.isfinite(k).all()
    assert k[0, 0, 0] == 7 * 8188 and k[0, 0, 1] == -8 * 8188 and k[0, 0, 2] == 0
    step = torch.tensor(2.0 / 7).half().float()
    assert k[1, 0, 3] == 0 and k[1, 0, 4] == 7 * step and k[2, 0, 5] == 7 * 8188
    assert torch.equal(k[3], torch.zeros_like(k[3])) and torch.isfinite(c.key_scales).all()
    want_c, want_s = np_pack(x.cpu().numpy())
    assert np.array_equal(c.key_codes[0, :, :4].cpu().numpy().transpose(1, 0, 2), want_c)


@pytest.mark.gpu
def test_rows_of_any_stride_and_alignment(igc_lib):
    s = Setup(igc_lib, "bf16", [5, 9], [3, 60], 4, 2, 96, seed=4)
    s.cache.write(s.k, s.v, s.fills, starts=s.starts, slots=s.slots)
    want = [t.clone() for t in (s.cache.key_codes, s.cache.value_scales)]
    out = s.attend()
    # a fused row of q|k|v, one value off any 16-byte boundary
    fused = torch.zeros(14, 1 + 8 * 96 + 6, dtype=s.kind, device="cuda")
    q, k, v = (fused[:, 1 + a * 96:1 + b * 96].unflatten(1, (-1, 96)) for a, b in ((0, 4), (4, 6), (6, 8)))
    q.copy_(s.q), k.copy_(s.k), v.copy_(s.v)
    s.cache.key_codes.zero_(), s.cache.value_scales.zero_()
    for i, (n, f) in enumerate(zip(s.rows, s.fill)):  # what lay before the rows
        s.cache.key_codes[s.slot_list[i], :, :f] = want[0][s.slot_list[i], :, :f]
        s.cache.value_scales[s.slot_list[i], :, :f] = want[1][s.slot_list[i], :, :f]
    s.cache.write(k, v, s.fills, starts=s.starts, slots=s.slots)
    for i, (n, f) in enumerate(zip(s.rows, s.fill)):
        assert torch.equal(s.cache.key_codes[s.slot_list[i], :, :f + n], want[0][s.slot_list[i], :, :f + n])
        assert torch.equal(s.cache.value_scales[s.slot_list[i], :, :f + n], want[1][s.slot_list[i], :, :f + n])
    room = torch.zeros(14, 2, 4, 97, dtype=s.kind, device="cuda")
    got = s.attend(q=q, out=room[:, 1, :, 1:])
    assert torch.equal(got, out) and room[:, 0].abs().sum() == 0 and room[:, 1, :, 0].abs().sum() == 0
    gk, _ = s.cache.read(s.fills, 14, s.kind, starts=s.starts, slots=s.slots,
                         out=(room[:, 0, :2, 1:], room[:, 1, 2:, 1:]))
    plain, _ = s.cache.read(s.fills, 14, s.kind, starts=s.starts, slots=s.slots)
    assert torch.equal(gk, plain)


# ---- attention

SHAPES = [  # heads, kv, size
    (8, 1, 256), (2, 1, 64), (8, 1, 32), (5, 5, 96), (14, 2, 128), (16, 1, 160), (6, 3, 320), (8, 1, 512)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv,size", SHAPES)
def test_single_tokens_at_odd_depths(igc_lib, kind, heads, kv, size):
    s = Setup(igc_lib, kind, [1] * 7, [0, 1, 62, 63, 64, 130, 301], heads, kv, size, seed=size, extra=1)
    s.check(s.attend())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv,size", SHAPES)
def test_ragged_blocks_and_empty_sequences(igc_lib, kind, heads, kv, size):
    s = Setup(igc_lib, kind, [4, 0, 1, 9, 3], [60, 7, 0, 64, 200], heads, kv, size, seed=size + 1, extra=1, tail=2)
    out = torch.full_like(s.q, 7.0)
    s.check(s.attend(out=out))
    assert torch.equal(out[17:], torch.full_like(out[17:], 7.0))  # rows behind the last sequence


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv,size", SHAPES)
def test_prompts_and_chunks(igc_lib, kind, heads, kv, size):
    s = Setup(igc_lib, kind, [70, 129], [0, 65], heads, kv, size, seed=size + 2)
    s.check(s.attend())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 0), (16, 4), (64, 64), (65, 3), (100, 70), (1000, 5)])
def test_window_and_first_positions(igc_lib, kind, window, sinks):
    s = Setup(igc_lib, kind, [1, 5, 1, 90], [300, 126, 0, 170], 8, 1, 256, seed=window + sinks, extra=1)
    s.check(s.attend(window=window, sinks=sinks), window, sinks)
    s = Setup(igc_lib, kind, [2, 1, 2], [300, 190, 64], 4, 2, 64, seed=window + sinks, extra=1)
    s.check(s.attend(window=window, sinks=sinks), window, sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_a_window_does_not_read_what_left_it(igc_lib, kind):
    """Places that no row sees may hold anything: evicted positions are NaN."""
    s = Setup(igc_lib, kind, [1, 3], [400, 333], 8, 1, 128, seed=9)
    for slot, f in zip(s.slot_list, s.fill):
        for scales in (s.cache.key_scales, s.cache.value_scales):
            scales[slot, :, 4:f - 63] = float("nan")  # the first row still sees f - 63
    s.check(s.attend(window=64, sinks=4), 64, 4)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [3, 40])
def test_padded_rows_see_nothing_and_come_out_zero(igc_lib, kind, rows):
    s = Setup(igc_lib, kind, [rows, rows, rows], [-2, -rows, 5], 8, 2, 64, seed=rows)
    codes = s.cache.key_codes.clone()
    s.cache.write(s.k, s.v, s.fills, starts=s.starts, slots=s.slots)
    assert torch.equal(s.cache.key_codes[s.slot_list[1]], codes[s.slot_list[1]])
    out = s.attend(out=torch.full_like(s.q, 3.0))
    assert out[:2].abs().max() == 0 and out[rows:2 * rows].abs().max() == 0
    s.check(out)
    k, v = s.cache.read(s.fills, 3 * rows, s.kind, starts=s.starts, slots=s.slots)
    assert k[:2].abs().max() == 0 and v[rows:2 * rows].abs().max() == 0 and k[2].abs().max() > 0


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_extreme_rows(igc_lib, kind):
    """Large and tiny queries, a row of zeros (the mean of the values), scales
    at the largest, and a NaN row that stays its own."""
    s = Setup(igc_lib, kind, [6, 40], [70, 0], 8, 1, 128, seed=3)
    s.q[0] *= 1e30
    s.q[1] *= 1e-30
    s.q[2] = 0
    s.q[3, :, 1:] = 0
    s.cache.key_scales[s.slot_list[0], :, 3] = 8188.0
    s.cache.value_scales[s.slot_list[0], :, 4] = 8188.0
    s.cache.value_scales[s.slot_list[1], :, 5] = 2.0 ** -24
    got = s.attend(scale=1e-2)
    want, tol = s.want(scale=1e-2)
    rows = [1, 2, 3, 4, 5] + list(range(6, 46))  # row 0's scores are past any rounding: its largest alone counts
    over = ((got.double() - want).abs() / tol)[rows].max().item()
    assert over <= 1.0, over
    assert torch.isfinite(got).all()
    s.q[4, 2, 7] = float("nan")
    bad = s.attend(scale=1e-2)
    assert torch.isnan(bad[4, 2]).all()
    bad[4, 2] = got[4, 2]
    assert torch.equal(bad, got)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,heads,kv,size", [("bf16", 32, 8, 128), ("f32", 8, 1, 256), ("f16", 8, 1, 512)])
def test_long_contexts_split_over_blocks(igc_lib, kind, heads, kv, size):
    s = Setup(igc_lib, kind, [1, 2], [9001, 4097], heads, kv, size, seed=5)
    s.check(s.attend())


@pytest.mark.gpu
def test_uniform_rows_without_lists(igc_lib):
    s = Setup(igc_lib, "bf16", [4, 4, 4], [9, 100, 64], 8, 1, 256, seed=6, shuffle=False)
    want = s.attend()
    assert torch.equal(s.cache.attend(s.q, s.fills, scale=16 ** -1.0), want)
    s.check(want)


@pytest.mark.gpu
def test_sequences_share_a_slot_to_read(igc_lib):
    s = Setup(igc_lib, "bf16", [1], [500], 8, 1, 256, seed=7)
    one = s.attend()
    many = s.cache.attend(s.q.expand(5, -1, -1), torch.full((5,), 500, dtype=torch.int32, device="cuda"),
                          slots=s.slots.expand(5).contiguous(), scale=1.0 / 16)
    assert ((many - one).abs().max() <= 2 * torch.finfo(torch.bfloat16).eps * one.abs().max()).item()


@pytest.mark.gpu
def test_results_repeat_to_the_bit(igc_lib):
    for rows, fill in (([1, 1, 4], [5000, 3, 700]), ([300, 17], [1000, 0])):
        s = Setup(igc_lib, "bf16", rows, fill, 8, 1, 256, seed=8)
        first = s.attend()
        for _ in range(3):
            assert torch.equal(s.attend(), first)


@pytest.mark.gpu
def test_a_step_captured_and_replayed(igc_lib):
    """Write then attend, as a decode step runs them, captured once and replayed
    while the positions advance on the device; two graphs at once."""
    s = Setup(igc_lib, "bf16", [1, 1, 1], [10, 190, 64], 8, 1, 256, seed=10, extra=1)
    s.attend()
    s.cache.write(s.k, s.v, s.fills, slots=s.slots)
    s.cache.key_scales.nan_to_num_(0.25), s.cache.value_scales.nan_to_num_(0.25)
    torch.cuda.synchronize()
    graphs, outs = [], []
    side = torch.cuda.Stream()
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            s.cache.write(s.k, s.v, s.fills, slots=s.slots)
            outs.append(s.cache.attend(s.q, s.fills, slots=s.slots, scale=1.0 / 16))
        graphs.append(g)
    for step in range(4):
        s.k.normal_(), s.v.normal_(), s.q.normal_()
        torch.cuda.synchronize()
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[1])
        s.check(outs[0])
        s.fills += 1
        s.fill = [f + 1 for f in s.fill]


@pytest.mark.gpu
def test_work_follows_the_current_stream(igc_lib):
    s = Setup(igc_lib, "bf16", [1, 1], [2000, 64], 8, 1, 256, seed=11)
    want = s.attend()
    side = torch.cuda.Stream()
    busy = torch.empty(1 << 26, device="cuda")
    for _ in range(3):
        q = torch.zeros_like(s.q)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            for _ in range(20):
                busy.normal_()
            q.copy_(s.q)
            got = s.attend(q=q)
        torch.cuda.synchronize()
        assert torch.equal(got, want)


@pytest.mark.gpu
def test_what_does_not_fit_the_cache_is_told(igc_lib):
    s = Setup(igc_lib, "bf16", [2, 2, 2], [10, 62, 20], 8, 1, 64, seed=12)
    codes = s.cache.key_codes.clone()
    want = s.attend()
    s.fills[1] = s.cache.positions - 1  # its second row stands past the cache
    out = s.attend(out=torch.full_like(s.q, 5.0))
    with pytest.raises(igc_lib.IgcError) as e:
        s.cache.status()
    assert e.value.code == igc_lib.FAIL_STATE
    s.cache.status()  # told once
    assert torch.equal(out[:2], want[:2]) and torch.equal(out[4:], want[4:]) and out[3].abs().max() == 0
    s.fills[1] = 62
    s.slots[2] = 99
    out = s.attend(out=torch.full_like(s.q, 5.0))
    with pytest.raises(igc_lib.IgcError):
        s.cache.status()
    assert torch.equal(out[:4], want[:4]) and out[4:].abs().max() == 0
    s.fills[1] = s.cache.positions
    s.cache.write(s.k[:4], s.v[:4], s.fills[1:].contiguous(), starts=s.starts[:3].contiguous(),
                  slots=s.slots[1:].contiguous())
    with pytest.raises(igc_lib.IgcError):
        s.cache.status()
    assert torch.equal(s.cache.key_codes, codes)  # nothing of it was written
    k, v = s.cache.read(s.fills[1:].contiguous(), 4, torch.float32, starts=s.starts[:3].contiguous(),
                        slots=s.slots[1:].contiguous())
    with pytest.raises(igc_lib.IgcError):
        s.cache.status()
    assert k.abs().max() == 0 and v.abs().max() == 0
    # rows past the arrays, backwards, or more than the call said: not run
    s.slots.copy_(torch.tensor(s.slot_list, dtype=torch.int32))
    s.fills[1] = 62
    for starts, most, left in (([0, 2, 4, 7], None, [4, 5]), ([0, 4, 2, 6], None, []), ([0, 1, 5, 6], 3, [1, 2, 3, 4]),
                               ([-1, 2, 4, 6], None, [0, 1])):
        out = s.cache.attend(s.q, s.fills, starts=torch.tensor(starts, dtype=torch.int32, device="cuda"),
                             slots=s.slots, scale=0.125, rows_most=most, out=torch.full_like(s.q, 5.0))
        with pytest.raises(igc_lib.IgcError):
            s.cache.status()
        assert (out[left] == 5.0).all()  # a sequence that is not run leaves its rows


@pytest.mark.gpu
def test_refusals_leave_everything_alone(igc_lib):
    s = Setup(igc_lib, "bf16", [2, 2], [10, 20], 8, 2, 64, seed=13)
    codes = s.cache.key_codes.clone()
    for bad in (dict(window=-1), dict(sinks=-2), dict(scale=float("nan")), dict(scale=float("inf"))):
        with pytest.raises(igc_lib.IgcError) as e:
            s.attend(**bad)
        assert e.value.code == igc_lib.FAIL_ARGUMENT
    with pytest.raises(igc_lib.IgcError):  # 7 heads do not share 2 evenly
        s.attend(q=s.q[:, :7])
    with pytest.raises(ValueError):
        s.attend(q=s.q[:, :, :32])
    with pytest.raises(ValueError):
        s.attend(q=s.q.double())
    with pytest.raises(ValueError):
        s.attend(q=s.q.cpu())
    with pytest.raises(ValueError):
        s.attend(q=s.q.transpose(1, 2))
    with pytest.raises(igc_lib.IgcError):  # the result is of the queries' type
        s.attend(out=torch.empty(s.q.shape, device="cuda"))
    with pytest.raises(ValueError):
        s.cache.write(s.k, s.v, s.fills.long(), starts=s.starts)
    with pytest.raises(ValueError):
        s.cache.write(s.k, s.v, s.fills, starts=s.starts[:2])
    with pytest.raises(ValueError):
        s.cache.write(s.k, s.v[:3], s.fills, starts=s.starts)
    with pytest.raises(igc_lib.IgcError):  # 3 rows do not split over 2 sequences
        s.cache.write(s.k[:3], s.v[:3], s.fills)
    with pytest.raises(igc_lib.IgcError):  # more sequences than slots, and no list of slots
        s.cache.write(s.k, s.v, torch.zeros(4, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        igc_lib.PackCache.open(1, 1, 64, 48)
    with pytest.raises(ValueError):
        igc_lib.PackCache.open(1, 1, 64, 544)
    c = igc_lib.PackCache.open(1, 1, 64, 64)
    with pytest.raises(ValueError):
        igc_lib.PackCache(c.key_codes[:, :, :32], c.key_scales[:, :, :32], c.value_codes[:, :, :32],
                          c.value_scales[:, :, :32])
    assert torch.equal(s.cache.key_codes, codes)
    s.cache.status()
    assert s.cache.attend(s.q[:0], s.fills, starts=torch.zeros_like(s.starts)).shape == (0, 8, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("heads,kv,size", [(71, 1, 64), (160, 1, 32), (21, 3, 128)])
def test_any_number_of_heads_shares_a_key_head(igc_lib, kind, heads, kv, size):
    s = Setup(igc_lib, kind, [3, 1, 2], [70, 5, 300], heads, kv, size, seed=14)
    s.check(s.attend())
    s.check(s.attend(window=33, sinks=2), window=33, sinks=2)


@pytest.mark.gpu
@pytest.mark.parametrize("fill", [2**31 - 1, 2**30 + 7, -2**31])
def test_the_farthest_positions(igc_lib, fill):
    """Past the cache: zeros, told.  Before it: padding."""
    s = Setup(igc_lib, "bf16", [3, 2], [40, 9], 8, 1, 64, seed=15)
    want, codes = s.attend(), s.cache.key_codes.clone()
    s.fills[0] = fill
    out = s.attend(out=torch.full_like(s.q, 5.0))
    s.cache.write(s.k, s.v, s.fills, starts=s.starts, slots=s.slots)
    k, v = s.cache.read(s.fills, 5, torch.float32, starts=s.starts, slots=s.slots)
    if fill > 0:
        with pytest.raises(igc_lib.IgcError):
            s.cache.status()
    s.cache.status()
    assert out[:3].abs().max() == 0 and k[:3].abs().max() == 0 and v[:3].abs().max() == 0
    assert torch.equal(out[3:], want[3:])
    assert torch.equal(s.cache.key_codes[s.slot_list[0]], codes[s.slot_list[0]])


@pytest.mark.gpu
def test_two_streams_and_two_graphs_at_once(igc_lib):
    """Calls on one cache from two streams, eager and captured, with scratch of
    their own each: 4-row blocks cut between blocks, and a prompt."""
    a = Setup(igc_lib, "bf16", [4] * 6, [900, 17, 350, 2000, 64, 1200], 8, 1, 256, seed=16)
    q2, rows2 = a.q[:10].contiguous(), torch.tensor([0, 10], dtype=torch.int32, device="cuda")
    f2, s2 = torch.tensor([1500], dtype=torch.int32, device="cuda"), a.slots[3:4].contiguous()
    one = lambda: a.attend()  # noqa: E731
    two = lambda: a.cache.attend(q2, f2, starts=rows2, slots=s2, scale=0.0625)  # noqa: E731
    want = one(), two()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for st, call in zip(streams, (one, two)):
            with torch.cuda.stream(st):
                got.append(call())
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graphs, outs = [], []
    for st, call in zip(streams, (one, two)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            outs.append(call())
        graphs.append(g)
    for _ in range(20):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for st, g in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


@pytest.mark.gpu
def test_results_in_an_array_of_other_strides(igc_lib):
    s = Setup(igc_lib, "bf16", [5, 40], [100, 30], 8, 2, 128, seed=17)
    want = s.attend()
    by_head = torch.zeros(8, 45, 128, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    wide = torch.zeros(45, 8, 131, dtype=torch.bfloat16, device="cuda")[:, :, 1:129]
    for out in (by_head, wide):
        assert torch.equal(s.attend(out=out), want)
    with pytest.raises(igc_lib.IgcError) as e:
        s.attend(out=torch.zeros(45, 1, 128, dtype=torch.bfloat16, device="cuda").expand(45, 8, 128))
    assert e.value.code == igc_lib.FAIL_ARGUMENT


@pytest.mark.gpu
@pytest.mark.parametrize("kind,heads,kv,size", [("f32", 4, 2, 64), ("bf16", 8, 2, 128), ("f16", 3, 3, 512),
                                                ("f32", 8, 2, 256), ("bf16", 10, 2, 96)])
def test_many_ragged_sequences(igc_lib, kind, heads, kv, size):
    """More units than run at once: one list of tiles, shared out in runs that
    begin and end anywhere; empty sequences, padding, and rows of 0 to 2."""
    g = np.random.default_rng(18)
    rows = [int(x) for x in g.integers(0, 3, 330)]
    fill = [int(x) for x in np.where(g.random(330) < 0.1, -1, g.integers(0, 400, 330))]
    s = Setup(igc_lib, kind, rows, fill, heads, kv, size, seed=19)
    s.check(s.attend(rows_most=2))
    s.check(s.attend(rows_most=2, window=70, sinks=5), window=70, sinks=5)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,heads,kv,size", [("f32", 8, 1, 256), ("bf16", 8, 2, 128), ("f16", 4, 1, 512)])
@pytest.mark.parametrize("rows,depth", [(1, 4200), (5, 1500), (20, 700), (3, 16200)])
def test_few_units_in_clusters(igc_lib, kind, heads, kv, size, rows, depth):
    s = Setup(igc_lib, kind, [rows, max(1, rows - 2)], [depth, depth // 3], heads, kv, size, seed=20)
    s.check(s.attend(rows_most=rows))
