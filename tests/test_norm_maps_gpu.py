"""Layer normalisation of maps one position at a time (H * W not a multiple of 4): both sides of every limit of how many channels a thread
holds, with enough positions that all lanes along them are used.  Bounds and reference: test_norm_gpu.py."""
import pytest
import torch
from test_norm_gpu import dev, make, run_both  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(32, 64, 21, 25), (32, 65, 21, 25), (16, 128, 19, 31), (16, 129, 19, 31), (8, 256, 31, 35), (8, 257, 31, 35),
                                   (4, 513, 35, 31), (4, 1025, 17, 17), (2, 2049, 17, 17), (2, 4096, 13, 11), (2, 4097, 13, 11), (2, 8192, 5, 5),
                                   (2, 8193, 5, 5)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_channels_of_a_thread(dev, shape, dtype):  # noqa: F811
    x, w, b, r, dy = make(shape, 1, dtype, torch.float32, dev, seed=sum(shape), residual=True)
    run_both(x, w, b, r, dy, 1, 1e-5, "tanh")
