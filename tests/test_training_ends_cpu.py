"""Argument checks of the training-side operators at the two ends of a decoder. They come before any device call, so they run
without a GPU."""
import ctypes as C

import pytest


def size(bfb, query, *args):
    n = C.c_size_t(12345)
    return getattr(bfb.lib(), query)(*args, C.byref(n)), n.value


def test_linear_cross_entropy_workspace_sizes(bfb):
    q = "bfb_linear_cross_entropy_workspace"
    st, forward = size(bfb, q, bfb.BF16, 16384, 32000, 2048, 0)
    assert st == bfb.OK and 0 < forward <= 16384 * (250 * 8 * 2 + 4) + 1024    # (maximum, sum) pairs, not logits
    st, both = size(bfb, q, bfb.BF16, 16384, 32000, 2048, 1)
    # a piece of dz in the CUDA-core route's fp32 or the tensor-core route's bf16, dx sums, bias sums
    assert st == bfb.OK and forward <= both <= (256 << 20) * 17 // 16 + 16384 * 2048 * 4 + (1 << 20)
    assert size(bfb, q, bfb.F32, 0, 10, 10, 1)[0] == bfb.OK
    for args in ((bfb.FP8_E4M3, 1, 1, 1, 1), (bfb.BF16, -1, 1, 1, 1), (bfb.BF16, 1, 0, 1, 1), (bfb.BF16, 1, 1, 0, 1),
                 (bfb.BF16, 1 << 31, 1, 1, 1), (bfb.BF16, 1, (1 << 24) + 1, 1, 1)):
        assert size(bfb, q, *args) == (bfb.INVALID_ARGUMENT, 0)
    assert bfb.lib().bfb_linear_cross_entropy_workspace(bfb.F32, 1, 1, 1, 1, None) == bfb.INVALID_ARGUMENT


FWD = dict(x=4096, ld_x=8, w=4096, ld_w=8, bias=None, labels=4096, loss=4096, lse=4096, summary=None, dtype=1, tokens=4, vocab=10, dim=8,
           oob=None, ws=4096, ws_bytes=1 << 30, status=None, stream=None)
BWD = dict(x=4096, ld_x=8, w=4096, ld_w=8, bias=None, labels=4096, lse=4096, grad_loss=None, d_scale=None, scale=1.0, dx=4096, ld_dx=8,
           dw=4096, ld_dw=8, db=None, dtype=1, grad_dtype=1, tokens=4, vocab=10, dim=8, ws=4096, ws_bytes=1 << 30, status=None, stream=None)


@pytest.mark.parametrize("change", [dict(x=None), dict(w=None), dict(labels=None), dict(lse=None), dict(ld_x=7), dict(ld_w=7), dict(dtype=2),
                                    dict(dtype=-1), dict(tokens=-1), dict(vocab=0), dict(dim=0), dict(vocab=(1 << 24) + 1),
                                    dict(tokens=1 << 31), dict(ws=None), dict(ws_bytes=16), dict(ws=4100),
                                    dict(loss=None, summary=4096)])
def test_linear_cross_entropy_forward_refuses(bfb, change):
    args = {**FWD, **change}
    assert bfb.lib().bfb_linear_cross_entropy_fwd(*args.values()) == bfb.INVALID_ARGUMENT
    assert b"linear_cross_entropy" in bfb.lib().bfb_last_error()


@pytest.mark.parametrize("change", [dict(x=None), dict(w=None), dict(labels=None), dict(lse=None), dict(ld_x=7), dict(ld_w=7), dict(dtype=2),
                                    dict(grad_dtype=2), dict(tokens=-1), dict(vocab=0), dict(dim=0), dict(ws=None), dict(ws_bytes=16),
                                    dict(ws=4100), dict(ld_dx=7), dict(ld_dw=7)])
def test_linear_cross_entropy_backward_refuses(bfb, change):
    args = {**BWD, **change}
    assert bfb.lib().bfb_linear_cross_entropy_bwd(*args.values()) == bfb.INVALID_ARGUMENT
    assert b"linear_cross_entropy" in bfb.lib().bfb_last_error()


def test_linear_cross_entropy_with_nothing_to_do(bfb):
    args = {**BWD, "dx": None, "dw": None}
    assert bfb.lib().bfb_linear_cross_entropy_bwd(*args.values()) == bfb.OK
    args = {**FWD, "tokens": 0, "x": None, "labels": None, "lse": None, "ws": None, "ws_bytes": 0}
    assert bfb.lib().bfb_linear_cross_entropy_fwd(*args.values()) == bfb.OK
