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


# ---- scaled embedding -------------------------------------------------------------------------------------------

LOOKUP = dict(ids=4096, table=4096, table_dtype=0, out=4096, out_dtype=0, ld_out=8, tokens=4, vocab=10, dim=8, scale=1.0, oob=None, stream=None)
SCATTER = dict(ids=4096, dout=4096, dout_dtype=0, ld_dout=8, dtable=4096, dtable_dtype=0, tokens=4, vocab=10, dim=8, scale=1.0, accumulate=0,
               ws=4096, ws_bytes=1 << 20, stream=None)


@pytest.mark.parametrize("change", [dict(ids=None), dict(table=None), dict(out=None), dict(table_dtype=2), dict(out_dtype=2), dict(ld_out=7),
                                    dict(tokens=-1), dict(vocab=0), dict(dim=0), dict(vocab=(1 << 24) + 1), dict(tokens=1 << 31)])
def test_embed_scaled_refuses(bfb, change):
    assert bfb.lib().bfb_embed_scaled(*{**LOOKUP, **change}.values()) == bfb.INVALID_ARGUMENT
    assert b"embed_scaled" in bfb.lib().bfb_last_error()


@pytest.mark.parametrize("change", [dict(ids=None), dict(dout=None), dict(dtable=None), dict(dout_dtype=2), dict(dtable_dtype=2), dict(ld_dout=7),
                                    dict(tokens=-1), dict(vocab=0), dict(dim=0), dict(ws=None), dict(ws=4104), dict(ws_bytes=100)])
def test_embed_scaled_backward_refuses(bfb, change):
    assert bfb.lib().bfb_embed_scaled_bwd(*{**SCATTER, **change}.values()) == bfb.INVALID_ARGUMENT
    assert b"embed_scaled" in bfb.lib().bfb_last_error()


def test_embed_scaled_sizes_and_nothing_to_do(bfb):
    st, n = size(bfb, "bfb_embed_scaled_bwd_workspace", 65536, 32000, 2048)
    assert st == bfb.OK and 4 * 65536 * 4 <= n <= 4 * 65536 * 4 + 65536 // 8 * 2048 * 8 + 32000
    assert size(bfb, "bfb_embed_scaled_bwd_workspace", 4, 0, 8) == (bfb.INVALID_ARGUMENT, 0)
    assert bfb.lib().bfb_embed_scaled(*{**LOOKUP, "tokens": 0, "ids": None}.values()) == bfb.OK
    assert bfb.lib().bfb_embed_scaled_bwd(*{**SCATTER, "tokens": 0, "ids": None, "dout": None, "ws": None, "accumulate": 1}.values()) == bfb.OK


# ---- distillation -----------------------------------------------------------------------------------------------

DISTILL = dict(z=4096, dtype=0, ld=10, ids=4096, teacher=4096, teacher_dtype=0, k=3, tau=1.0, grad_loss=None, d_scale=None, scale=1.0, loss=4096,
               lse=4096, grad=8192, grad_dtype=0, ld_grad=10, rows=4, vocab=10, oob=None, stream=None)


@pytest.mark.parametrize("change", [dict(z=None), dict(ids=None), dict(teacher=None), dict(dtype=2), dict(teacher_dtype=2), dict(grad_dtype=2),
                                    dict(ld=9), dict(ld_grad=9), dict(k=0), dict(k=1025), dict(tau=0.0), dict(tau=-1.0), dict(tau=1e-7), dict(tau=1e7), dict(tau=float("nan")),
                                    dict(tau=float("inf")), dict(rows=-1), dict(vocab=0), dict(vocab=(1 << 24) + 1, ld=1 << 25, ld_grad=1 << 25),
                                    dict(grad=4096, grad_dtype=1), dict(grad=4096, ld_grad=11)])
def test_distill_refuses(bfb, change):
    assert bfb.lib().bfb_distill_topk(*{**DISTILL, **change}.values()) == bfb.INVALID_ARGUMENT
    assert b"distill_topk" in bfb.lib().bfb_last_error()


def test_distill_with_nothing_to_do(bfb):
    assert bfb.lib().bfb_distill_topk(*{**DISTILL, "rows": 0, "z": None}.values()) == bfb.OK
