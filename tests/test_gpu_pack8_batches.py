"""The weight gradient over more batches than one launch has lanes for: 2^32 lanes are 2^23 blocks of 512 or 2^24 of 256."""
import numpy as np
import pytest

from test_gpu_scan import put

pytestmark = pytest.mark.gpu


# a tile a batch, or two: the 128 x 128 tile of 256 lanes, the 256 x 128 tile of 512, f64's 128 x 128 tile of 512
@pytest.mark.parametrize("dtype, b, m, k", [("f32", (1 << 24) + 5, 1, 1), ("f32", (1 << 23) + 5, 1, 129), ("f64", (1 << 23) + 5, 128, 1)])
def test_many_small_batches(dtype, b, m, k):
    """x = 2 everywhere and an upstream gradient of its own for each batch: dst = 2 m up[batch], exactly."""
    from rtensors_amd import hip as H
    be, code, T = H.Hip.new(0), H.DTYPE_BY_NAME[dtype], {"f32": np.float32, "f64": np.float64}[dtype]
    x = be.alloc_uninit(code, b * m * k)
    be.fill_contiguous(x, 2.0, 0, b * m * k)
    codes, exps = be.alloc_pack8(b * m * k)
    be.pack8(x, 0, b * m * k, codes, exps)
    del x
    up = np.repeat((np.arange(b) % 65521 - 30000).astype(T), m)
    dst = be.alloc_uninit(code, b * k)
    be.fill_contiguous(dst, -1.0, 0, b * k)
    be.pack8_matmul_backward(codes, exps, put(be, up), dst, b, m, k, 1)
    got = be.dump(dst).reshape(b, k)
    assert (got == 2 * m * up[::m, None]).all()
    be.sync()
