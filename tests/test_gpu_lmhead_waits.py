"""GPU: the fused LM head when a bounded wait inside it runs out.

A self-checking build (TABBY_CHECKS=1, waits of 2 ms) lets the warp that issues a tile's products
give up behind some that it has just issued. The kernels have to return, every row has to report
TABBY_ETIMEOUT, no CTA may give its tensor memory back before its products are done, and the next
call on the same handle has to be right. No GPU fault is involved: the waits give up.
"""
import ctypes

import numpy as np
import pytest

from tests.conftest import gpu_available

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def checked(tmp_path_factory):
    if not gpu_available():
        pytest.skip("no CUDA device")
    from tabby_b200 import _lib, build

    try:
        build.nvcc()
    except RuntimeError:
        pytest.skip("no nvcc")
    path = str(tmp_path_factory.mktemp("checked") / "libsample.so")
    build.build(out=path, defines=("TABBY_CHECKS=1", "TABBY_WAIT_NS=2000000ull"))
    lib = _lib._load(path, _lib.SIGNATURES)
    lib.tabby_debug_lmhead.argtypes = [ctypes.c_int32, ctypes.POINTER(ctypes.c_int32)]
    return lib


@pytest.mark.parametrize("rows,vocab,hidden,tile", [
    (4, 151936, 896, 0), (4, 151936, 896, 300), (128, 20000, 512, 70), (64, 49152, 64, 5),
])
def test_an_issuer_that_gives_up(oracle, checked, rows, vocab, hidden, tile):
    import torch

    from tabby_b200._lib import OUTCOME_DTYPE, TABBY_ETIMEOUT, lib

    g = torch.Generator().manual_seed(vocab)
    h = torch.randn(rows, hidden, generator=g).to(torch.bfloat16).cuda()
    w = (torch.randn(vocab, hidden, generator=g) * (3.0 / hidden ** 0.5)).to(torch.bfloat16).cuda()
    p = oracle.make_params(np.full(rows, 0.8), np.full(rows, 0.95), np.full(rows, 40), rows)
    pd = torch.from_numpy(p.view(np.uint8).copy()).cuda()
    ud = torch.from_numpy(np.random.default_rng(1).random(rows)).cuda()
    out = torch.zeros(rows * OUTCOME_DTYPE.itemsize, dtype=torch.uint8, device="cuda")

    def sample(L, handle):
        out.zero_()
        assert L.tabby_lmhead_sample_async(handle, h.data_ptr(), w.data_ptr(), rows,
                                           pd.data_ptr(), ud.data_ptr(), out.data_ptr(), None,
                                           None, 0, None,
                                           torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        return out.cpu().numpy().view(OUTCOME_DTYPE).copy()

    def debug(give_up):
        n = ctypes.c_int32()
        assert checked.tabby_debug_lmhead(give_up, ctypes.byref(n)) == 0
        return n.value

    plain, handle = ctypes.c_void_p(), ctypes.c_void_p()
    assert lib().tabby_lmhead_create(0, rows, vocab, hidden, ctypes.byref(plain)) == 0
    want = sample(lib(), plain)
    lib().tabby_lmhead_destroy(plain)
    assert (want["status"] == 0).all()
    assert checked.tabby_lmhead_create(0, rows, vocab, hidden, ctypes.byref(handle)) == 0
    debug(-1)
    np.testing.assert_array_equal(sample(checked, handle).view(np.uint8), want.view(np.uint8))
    debug(tile)
    got = sample(checked, handle)
    assert (got["status"] == TABBY_ETIMEOUT).all() and (got["id"] == -1).all()
    assert debug(-1) == 0  # CTAs with products on their way, and no tile given up again
    np.testing.assert_array_equal(sample(checked, handle).view(np.uint8), want.view(np.uint8))
    checked.tabby_lmhead_destroy(handle)
