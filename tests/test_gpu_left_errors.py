"""A call that failed leaves nothing behind: its error is its own, and what follows on the thread runs."""
import ctypes as C

import numpy as np
import pytest

import tatara_b200 as tb
from tatara_b200 import _lib as L

pytestmark = pytest.mark.gpu
FS = tb.FEATURE_SETS["halfka-hm-merged"]


def microbench():
    zero, result = (C.c_int32 * 8)(), L.MicrobenchResult()
    return L.load().tb_ft_microbench(99, zero, zero, 1, 128, 4, 0, 8, 1, 0, C.byref(result))


def forward_bench():
    zero, ms = np.zeros(512, np.float32), C.c_float()
    return L.load().tb_ft_forward_bench(99, zero.ctypes.data_as(L.vp), zero.ctypes.data_as(L.vp), zero.ctypes.data_as(L.vp), 1, 128, 4, 1, 1, None, C.byref(ms))


def extract():
    zero = np.zeros(4096, np.uint8).ctypes.data_as(L.vp)
    return L.load().tb_psv_extract(99, FS.index, zero, 1, zero, zero, zero, None, zero, zero)


@pytest.mark.parametrize("failing", [microbench, forward_bench, extract])
def test_the_next_calls_run(failing):
    assert failing() < 0   # no such device
    batch = tb.synthetic_batch(tb.SYNTH_SEED, 64, FS)
    losses = []
    for fail_first in (False, True):
        t = tb.GpuTrainer(64, 256, 16, 32, 9, FS, init=tb.layerstack_default_init(FS, 256, 16, 32, 9))
        for _ in range(2):
            if fail_first:
                assert failing() < 0
            t.train_step(batch, 8.75e-4, 0.0, tb.LossKind.sigmoid())
        losses.append(t.flush_pending_loss())
        t.close()
    assert losses[0] == losses[1]
