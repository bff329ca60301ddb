"""What is brought to the device is there before a kernel reads it, however
busy the copy engines are: a model or a backend plane loaded while other
streams copy gives the bits of one loaded on an idle device."""

import threading

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


class Pressure:
    """Copies of pinned memory on 16 streams, a few on each at all times."""

    def __enter__(self):
        self.host = [torch.empty(16 << 20, dtype=torch.uint8).pin_memory() for _ in range(4)]
        self.dev = [torch.empty(16 << 20, dtype=torch.uint8, device="cuda") for _ in range(16)]
        self.streams = [torch.cuda.Stream() for _ in range(16)]
        self.stop = threading.Event()
        self.thread = threading.Thread(target=self.run)
        self.thread.start()

    def run(self):
        ends = [None] * 16
        while not self.stop.wait(0.0003):
            for i, stream in enumerate(self.streams):
                if ends[i] is not None and not ends[i].query():
                    continue
                with torch.cuda.stream(stream):
                    for _ in range(3):
                        self.dev[i].copy_(self.host[i % 4], non_blocking=True)
                    ends[i] = torch.cuda.Event()
                    ends[i].record(stream)

    def __exit__(self, *exc):
        self.stop.set()
        self.thread.join()
        torch.cuda.synchronize()


@pytest.mark.parametrize("count", [40, 100])
def test_a_model_loaded_beside_other_copies(igc_lib, count):
    """A prompt in passes of 16 lanes, and in a chunk of many, whose tables of
    caches are brought in with it."""
    spec = igc_lib.SynthSpec(vocab=4096, hidden=768, layers=4, heads=8, kv_heads=1, head_dim=256, inner=3 * 768,
                             ple_dim=128, slide_span=64, share_count=1, global_every=3, window_limit=256,
                             norm_offset=1.0, with_layer_scalar=1, seed=5)
    ids = np.random.default_rng(4).integers(0, 4096, count).astype(np.int32)

    def logits():
        m = igc_lib.Model(spec=spec, window_limit=256)
        s = igc_lib.Session(m)
        s.prime(ids)
        return s.step(ids[-1])[1].copy()

    want = logits()
    with Pressure():
        for _ in range(3):
            assert np.array_equal(logits(), want)


def test_a_plane_brought_in_beside_other_copies(igc_lib):
    rng = np.random.default_rng(6)
    rows, cols = 2048, 1536
    code = rng.integers(0, 256, (rows, cols // 2)).astype(np.uint8)
    scale = rng.uniform(0.5, 2.0, (rows, cols // 32)).astype(np.float16)
    act = rng.normal(0, 1, (1, cols)).astype(np.float32)
    plane = igc_lib.IgcPlane(form=2, row_count=rows, col_count=cols, code_data=code.ctypes.data, row_stride=cols // 2,
                             gain_data=scale.ctypes.data, gain_type=2, bit_count=4, code_bias=8, code_flip=0,
                             group_size=32, group_count=cols // 32)

    def product():
        desk = igc_lib.Desk()
        out = desk.mat_mat(plane, act, 1, rows)
        desk.close()
        return out

    want = product()
    with Pressure():
        for _ in range(10):
            assert np.array_equal(product(), want)
