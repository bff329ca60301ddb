"""A packed cache of more than 2^32 bytes a side: rows written, read back and
attended over at its end, in the forms for one row and for many.

Every place but the last 64 positions is cleared: a key of zeros scores 0 and
a value of zeros adds nothing, so a row sees its last positions beside
`positions - 64` weights of exp(0).  Bounds as in test_gpu_pack: weights and
values (and past 16 rows a key/value head keys) rounded to f16 for 16-bit rows,
and f32's own for 32-bit rows."""

import pytest

torch = pytest.importorskip("torch")

from test_gpu_pack import unpack64  # noqa: E402

POSITIONS, KV, GROUP = 1 << 22, 8, 8


@pytest.mark.gpu
@pytest.mark.parametrize("size", [256, 512])
def test_the_end_of_a_long_cache(igc_lib, size):
    cache = igc_lib.PackCache.open(1, KV, POSITIONS, size)
    assert cache.key_codes.numel() >= 1 << 32
    g = torch.Generator(device="cuda")
    g.manual_seed(size)
    k = torch.randn(64, KV, size, generator=g, device="cuda")
    v = torch.randn(64, KV, size, generator=g, device="cuda")
    at = torch.tensor([POSITIONS - 64], dtype=torch.int32, device="cuda")
    cache.write(k, v, at)
    got_k, got_v = cache.read(at, 64, torch.float32)
    keys = unpack64(cache.key_codes[0, :, -64:], cache.key_scales[0, :, -64:])  # [kv, 64, size]
    values = unpack64(cache.value_codes[0, :, -64:], cache.value_scales[0, :, -64:])
    assert torch.equal(got_k.double(), keys.transpose(0, 1)) and torch.equal(got_v.double(), values.transpose(0, 1))
    # what was written holds the rows to half a step of a group's scale
    step = cache.key_scales[0, :, -64:].double().repeat_interleave(32, -1).transpose(0, 1)
    assert ((got_k.double() - k.double()).abs() <= step * 0.51).all()
    for kind in (torch.float32, torch.bfloat16, torch.float16):
        for rows, window in ((1, 0), (40, 0), (3, 16)):
            scale = 2.0 * size ** -0.5
            q = torch.randn(rows, KV * GROUP, size, generator=g, device="cuda").to(kind)
            fill = torch.tensor([POSITIONS - rows], dtype=torch.int32, device="cuda")
            got = cache.attend(q, fill, window=window, scale=scale).double()
            cache.status()
            qs = q.double().unflatten(1, (KV, GROUP))
            score = torch.einsum("rhgd,hjd->rhgj", qs, keys) * scale
            p = 64 - rows + torch.arange(rows, device="cuda").view(-1, 1, 1, 1)
            j = torch.arange(64, device="cuda")
            see = (j <= p) & ((j > p - window) if window else (j <= p))
            w = torch.exp(score).masked_fill(~see, 0.0)
            total = w.sum(-1, keepdim=True) + (0 if window else POSITIONS - 64)
            w = w / total
            want = torch.einsum("rhgj,hjd->rhgd", w, values).flatten(1, 2)
            mass = torch.einsum("rhgj,hjd->rhgd", w, values.abs()).flatten(1, 2)
            near = cache.key_scales[0, :, -64:].double().repeat_interleave(32, -1)
            off = scale * torch.einsum("rhgd,hjd->rhgj", qs.abs(), near).amax(-1) * 23 * (size // 32 + 8) * 2.0 ** -23
            if rows * GROUP > 16 and size <= 256 and kind != torch.float32:
                off += scale * torch.einsum("rhgd,hjd->rhgj", qs.abs(), keys.abs()).amax(-1) * 2.0 ** -11 / 2
            each = 2.0 ** -10 + 2.0 ** -20 if kind != torch.float32 else 2.0 ** -19
            tol = mass * (each + torch.expm1(4 * off).flatten(1).unsqueeze(-1)) + 1e-30
            tol += want.abs() * torch.finfo(kind).eps / 2
            # weights below 2^-21 of the largest hold to 2^-32 of it, and f16 results below its normal range to 2^-25
            tol += 2.0 ** -32 * values.abs().sum(1).repeat_interleave(GROUP, 0)
            if kind == torch.float16:
                tol += 2.0 ** -25
            # the largest weights' sums: 2^22 additions in 32 bits, a tile at a time
            tol += want.abs() * (2.0 ** -24 * 4096 if not window else 0)
            over = ((got - want).abs() / tol).max().item()
            assert torch.isfinite(got).all() and over <= 1.0, (kind, rows, window, over)
