"""Packed sessions of models whose layers are not alike, and of wide heads."""

import json
import os
import struct

import numpy as np
import pytest

from conftest import SMALL, make_checkpoint
from test_gpu_packed_session import ATOL, Drawn

pytestmark = pytest.mark.gpu


def _doubled(folder, out, layer):
    """A copy of the checkpoint in which `layer` has each key/value head twice."""
    with open(os.path.join(folder, "model.safetensors"), "rb") as f:
        n = struct.unpack("<Q", f.read(8))[0]
        head, data = json.loads(f.read(n)), f.read()
    made, at, parts = {}, 0, []
    for name, t in head.items():
        if name == "__metadata__":
            made[name] = t
            continue
        raw, shape = data[t["data_offsets"][0]:t["data_offsets"][1]], list(t["shape"])
        if f".layers.{layer}.self_attn.k_proj" in name or f".layers.{layer}.self_attn.v_proj" in name:
            raw, shape = raw * 2, [2 * shape[0]] + shape[1:]
        made[name] = {"dtype": t["dtype"], "shape": shape, "data_offsets": [at, at + len(raw)]}
        parts.append(raw)
        at += len(raw)
    text = json.dumps(made).encode()
    text += b" " * (-len(text) % 8)
    os.makedirs(out)
    with open(os.path.join(out, "model.safetensors"), "wb") as f:
        f.write(struct.pack("<Q", len(text)) + text + b"".join(parts))
    for name in ("config.json", "tokenizer.json"):
        with open(os.path.join(folder, name), "rb") as a, open(os.path.join(out, name), "wb") as b:
            b.write(a.read())


def test_layers_of_several_key_head_counts(igc_lib, tmp_path):
    """One global layer with its key/value head twice computes what the layer
    with one does, in units of other shapes: its scratch is its own size."""
    window = 32768
    plain, twice = str(tmp_path / "plain"), str(tmp_path / "twice")
    igc_lib.synth_write(igc_lib.SynthSpec(**dict(SMALL, layers=16, window_limit=window)), plain, 4)
    _doubled(plain, twice, 7)
    ids = np.random.default_rng(6).integers(0, SMALL["vocab"], 50).astype(np.int32)
    rows = []
    for folder in (plain, twice):
        m = igc_lib.Model(folder=folder, window_limit=window)
        s = igc_lib.Session(m, packed=True, sinks=2)
        s.prime(ids[:1])  # nothing cached: what follows is blocks of lanes
        rows.append([s.guess(ids[1:17]).copy()])
        s.guess_keep(16)
        rows[-1].append(s.guess(ids[17:21]).copy())
        s.guess_keep(4)
        rows[-1].append(s.step(ids[21])[1].copy()[None])
    for a, b in zip(*rows):
        assert np.isfinite(a).all() and np.abs(a - b).max() <= 2e-2


def test_wide_heads_against_the_restatement(igc_lib, igo_mod, tmp_path):
    """512-wide heads on every layer, sliding and global: a prompt, blocks and
    steps, every row of them to the parity bar."""
    cfg = dict(SMALL, heads=4, head_dim=512, slide_span=40, window_limit=1024)
    folder = str(tmp_path / "wide")
    make_checkpoint(igc_lib, folder, cfg)
    d = Drawn(igo_mod, folder, cfg, 2, 8)
    m = igc_lib.Model(folder=folder, window_limit=cfg["window_limit"])
    s = igc_lib.Session(m, packed=True, sinks=2)
    ids = d.tokens(140)
    s.prime(ids)
    d.o.prime(ids)
    for k in (1, 5, 16):
        blk = d.tokens(k)
        got, want = s.guess(blk), d.o.guess(blk)
        assert np.abs(got - want).max() <= ATOL
        s.guess_keep(k)
        d.o.guess_keep(k)
        t = d.tokens(1)[0]
        assert np.abs(s.step(t)[1] - d.o.step(t)).max() <= ATOL
