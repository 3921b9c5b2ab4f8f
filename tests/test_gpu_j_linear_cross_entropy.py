"""The linear cross entropy (bfb_linear_cross_entropy_fwd / _bwd) through the C ABI against the formulas in 64 bits: the
tensor-core route (bf16 operands on 16-byte rows), the CUDA-core route (fp32, and bf16 rows TMA cannot read), rows that do
not count, classes taken out by a -inf bias, pitches, pieces of the vocabulary, streams and captured graphs.

Bounds are elementwise and follow from the arithmetic. With u = 2^-24 and a dot product of length K in fp32 (products of
bf16 values are exact in it; the tensor core may truncate instead of rounding, hence 2u a step) a logit is off by at most
2 K u sum |x||w| + u |z|, lse by the largest logit error plus a few roundings, and p = exp(z - lse) by the sum of both,
relatively. dz is rounded to bf16 (half a step: 2^-8 relative) on the tensor-core route, and a result once more where
it is bf16."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_BF16 = 2.0 ** -8


def workspace(gpu, torch, dtype, tokens, vocab, dim, backward=1):
    n = C.c_size_t(0)
    gpu.check(gpu.lib().bfb_linear_cross_entropy_workspace(dtype, tokens, vocab, dim, backward, C.byref(n)))
    return torch.full((max(1, n.value),), 0x7F, dtype=torch.uint8, device="cuda"), n.value


def padded(torch, rows, dim, pad, dtype, fill):
    """A [rows, dim] view with `pad` extra columns a row and a row behind the last, filled with a mark."""
    whole = torch.full((rows + 1, dim + pad), fill, dtype=dtype, device="cuda")
    return whole, whole[:rows, :dim]


def forward(gpu, torch, x, w, bias, labels, stream=None, ws=None, want_summary=True, loss=None):
    tokens, dim = x.shape
    vocab = w.shape[0]
    code = gpu.F32 if x.dtype == torch.float32 else gpu.BF16
    ws = ws or workspace(gpu, torch, code, tokens, vocab, dim)
    loss = torch.full((tokens + 3,), 7.0, device="cuda")
    lse = torch.full((tokens + 3,), 7.0, device="cuda")
    summary = torch.full((3,), 7.0, device="cuda")
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    gpu.check(gpu.lib().bfb_linear_cross_entropy_fwd(
        x.data_ptr(), x.stride(0) if tokens > 1 else max(dim, x.stride(0)), w.data_ptr(), max(dim, w.stride(0)),
        None if bias is None else bias.data_ptr(), labels.data_ptr(), loss.data_ptr(), lse.data_ptr(),
        summary.data_ptr() if want_summary else None, code, tokens, vocab, dim, bad.data_ptr(), ws[0].data_ptr(), ws[1],
        status.data_ptr(), stream))
    return dict(loss=loss, lse=lse, summary=summary, bad=bad, status=status, ws=ws)


def backward(gpu, torch, x, w, bias, labels, lse, grad_dtype, grad_loss=None, d_scale=None, scale=1.0, pad=0, stream=None, ws=None,
             want=(True, True, True)):
    tokens, dim = x.shape
    vocab = w.shape[0]
    code = gpu.F32 if x.dtype == torch.float32 else gpu.BF16
    gcode = gpu.F32 if grad_dtype == torch.float32 else gpu.BF16
    ws = ws or workspace(gpu, torch, code, tokens, vocab, dim)
    dx_whole, dx = padded(torch, tokens, dim, pad, grad_dtype, 5.0)
    dw_whole, dw = padded(torch, vocab, dim, pad, grad_dtype, 5.0)
    db = torch.full((vocab + 3,), 5.0, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    gpu.check(gpu.lib().bfb_linear_cross_entropy_bwd(
        x.data_ptr(), max(dim, x.stride(0)), w.data_ptr(), max(dim, w.stride(0)), None if bias is None else bias.data_ptr(),
        labels.data_ptr(), lse.data_ptr(), None if grad_loss is None else grad_loss.data_ptr(),
        None if d_scale is None else d_scale.data_ptr(), scale, dx.data_ptr() if want[0] else None, dim + pad,
        dw.data_ptr() if want[1] else None, dim + pad, db.data_ptr() if want[2] else None, code, gcode, tokens, vocab, dim,
        ws[0].data_ptr(), ws[1], status.data_ptr(), stream))
    return dict(dx=dx, dw=dw, db=db[:vocab], dx_whole=dx_whole, dw_whole=dw_whole, db_whole=db, status=status)


def reference(torch, x, w, bias, labels, row_grad):
    """Values and elementwise error bounds in 64 bits."""
    x64, w64 = x.double(), w.double()
    z = x64 @ w64.t() + (0.0 if bias is None else bias.double())
    dim, vocab = x.shape[1], w.shape[0]
    z_err = 2 * dim * U * (x64.abs() @ w64.abs().t()) + 2 * U * z.abs().nan_to_num(posinf=0.0)
    top = z.max(1).values
    lse = top + torch.exp(z - top[:, None]).sum(1).log()
    counted = (labels >= 0) & (labels < vocab)
    label = labels.clamp(0, vocab - 1).round().long()
    at = z.gather(1, label[:, None])[:, 0]
    # the exponentials' arguments are of the size of the logits: their rounding, 4 u |z| log2(e), and the sum's
    lse_err = z_err.max(1).values + U * (8 * z.abs().nan_to_num(posinf=0.0).max(1).values + 4 * lse.abs() + 64)
    loss = torch.where(counted, lse - at, torch.zeros_like(lse))
    p = torch.exp(z - lse[:, None])
    rel = z_err + lse_err[:, None] + U * (8 * z.abs().nan_to_num(posinf=0.0) + 8 * lse.abs()[:, None] + 16)
    g = torch.where(counted, row_grad.double(), torch.zeros_like(lse))
    dz = p.clone()
    rows = torch.arange(len(lse), device=z.device)
    dz[rows, label] -= 1.0
    dz *= g[:, None]
    dz_err = (p * rel + 4 * U * dz.abs() / g.abs()[:, None].clamp(min=1e-300)) * g.abs()[:, None]
    return dict(z=z, lse=lse, lse_err=lse_err, loss=loss, loss_err=lse_err + z_err.max(1).values, dz=dz, dz_err=dz_err, counted=counted)


def within(got, want, err, out_half):
    got = got.double()
    assert bool(got.isfinite().all())
    excess = (got - want).abs() - (err + out_half * (want.abs() + err) + 1e-37)
    worst = float(excess.max()) if excess.numel() else 0.0
    assert worst <= 0, worst


def gradients_within(torch, got, r, x, w, tensor_cores, grad_dtype):
    half_dz = HALF_BF16 if tensor_cores else 0.0
    out_half = U if grad_dtype == torch.float32 else HALF_BF16
    dz, err = r["dz"], r["dz_err"]
    dz_err = err + half_dz * (dz.abs() + err)
    tokens, vocab = dz.shape
    x64, w64 = x.double(), w.double()
    mass = dz.abs() + dz_err
    within(got["dx"], dz @ w64, dz_err @ w64.abs() + 2 * (vocab + 8) * U * (mass @ w64.abs()), out_half)
    within(got["dw"], dz.t() @ x64, dz_err.t() @ x64.abs() + 2 * (tokens + 8) * U * (mass.t() @ x64.abs()), out_half)
    within(got["db"], dz.sum(0), err.sum(0) + (tokens + 8) * U * (dz.abs() + err).sum(0), U)


def make(torch, tokens, vocab, dim, dtype, with_bias, seed, pad=0, spread=2.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    xw, x = padded(torch, tokens, dim, pad, dtype, 3.0)
    ww, w = padded(torch, vocab, dim, pad, dtype, 3.0)
    x.copy_(torch.randn(tokens, dim, generator=gen, device="cuda"))
    w.copy_(torch.randn(vocab, dim, generator=gen, device="cuda") * (spread / dim ** 0.5))
    bias = torch.randn(vocab, generator=gen, device="cuda") * 0.3 if with_bias else None
    labels = torch.randint(0, vocab, (tokens,), generator=gen, device="cuda").float()
    out = torch.rand(tokens, generator=gen, device="cuda") < 0.15
    return x, w, bias, torch.where(out, torch.full_like(labels, -100.0), labels)


TC_SHAPES = [(1, 1, 8), (1, 300, 64), (2, 127, 16), (7, 257, 64), (33, 128, 72), (128, 256, 64), (129, 1000, 136), (256, 4097, 256),
             (300, 1003, 200), (515, 777, 512), (1030, 2500, 64), (5000, 300, 64),
             (300, 20001, 200)]


@pytest.mark.parametrize("tokens,vocab,dim", TC_SHAPES)
@pytest.mark.parametrize("with_bias,grad", [(False, "bf16"), (True, "f32")])
def test_tensor_core_route(gpu, tokens, vocab, dim, with_bias, grad):
    import torch
    pad = 8 if with_bias else 0
    x, w, bias, labels = make(torch, tokens, vocab, dim, torch.bfloat16, with_bias, tokens + vocab, pad=pad)
    f = forward(gpu, torch, x, w, bias, labels)
    weight = torch.rand(tokens, device="cuda") + 0.5
    r = reference(torch, x, w, bias, labels, weight * (0.25 * f["summary"][2]))
    t = torch.float32 if grad == "f32" else torch.bfloat16
    got = backward(gpu, torch, x, w, bias, labels, f["lse"], t, grad_loss=weight, d_scale=f["summary"][2:], scale=0.25, pad=pad)
    torch.cuda.synchronize()
    assert int(f["status"]) == 0 and int(got["status"]) == 0 and int(f["bad"]) == 0
    within(f["lse"][:tokens], r["lse"], r["lse_err"], U)
    within(f["loss"][:tokens], r["loss"], r["loss_err"], U)
    assert (f["lse"][tokens:] == 7.0).all() and (f["loss"][tokens:] == 7.0).all()
    count = int(r["counted"].sum())
    assert f["summary"][1] == count and abs(float(f["summary"][2]) - (1.0 / count if count else 0.0)) <= U
    within(f["summary"][:1], r["loss"].sum()[None], r["loss_err"].sum()[None], U)
    gradients_within(torch, got, r, x, w, True, t)
    # columns and rows beside the results stay as they were
    assert (got["dx_whole"][tokens:] == 5.0).all() and (got["dx_whole"][:, dim:] == 5.0).all()
    assert (got["dw_whole"][vocab:] == 5.0).all() and (got["dw_whole"][:, dim:] == 5.0).all()
    assert (got["db_whole"][vocab:] == 5.0).all()


@pytest.mark.parametrize("tokens,vocab,dim", [(1, 1, 1), (1, 70, 3), (5, 64, 33), (65, 130, 97), (200, 1003, 31), (301, 515, 129)])
@pytest.mark.parametrize("dtype,grad", [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16"), ("f32", "bf16")])
def test_cuda_core_route(gpu, tokens, vocab, dim, dtype, grad):
    import torch
    td = torch.float32 if dtype == "f32" else torch.bfloat16
    tg = torch.float32 if grad == "f32" else torch.bfloat16
    x, w, bias, labels = make(torch, tokens, vocab, dim, td, True, tokens * 3 + vocab, pad=1)
    f = forward(gpu, torch, x, w, bias, labels)
    r = reference(torch, x, w, bias, labels, torch.full((tokens,), 0.5, device="cuda"))
    got = backward(gpu, torch, x, w, bias, labels, f["lse"], tg, scale=0.5, pad=1)
    torch.cuda.synchronize()
    within(f["lse"][:tokens], r["lse"], r["lse_err"], U)
    within(f["loss"][:tokens], r["loss"], r["loss_err"], U)
    # fp32 products round themselves too: K more roundings of each sum's terms, which 2 K u covers with the additions
    gradients_within(torch, got, r, x, w, False, tg)
    assert (got["dx_whole"][tokens:] == 5.0).all() and (got["dx_whole"][:, dim:] == 5.0).all()
    assert (got["dw_whole"][vocab:] == 5.0).all() and (got["dw_whole"][:, dim:] == 5.0).all()


def test_pieces_of_the_vocabulary_join(gpu):
    """Enough rows that one piece of dz does not hold all columns: dx is summed over the pieces."""
    import torch
    tokens, vocab, dim = 40000, 9001, 16
    x, w, bias, labels = make(torch, tokens, vocab, dim, torch.bfloat16, True, 5)
    f = forward(gpu, torch, x, w, bias, labels)
    got = {t: backward(gpu, torch, x, w, bias, labels, f["lse"], t, d_scale=f["summary"][2:]) for t in (torch.float32, torch.bfloat16)}
    torch.cuda.synchronize()
    row_grad = torch.full((tokens,), float(f["summary"][2]), device="cuda")
    r = reference(torch, x, w, bias, labels, row_grad)
    for t, g in got.items():
        assert int(g["status"]) == 0
        gradients_within(torch, g, r, x, w, True, t)


@pytest.mark.parametrize("dtype,dim", [("bf16", 64), ("bf16", 61), ("f32", 64)])
def test_gradients_that_are_not_asked_for(gpu, dtype, dim):
    import torch
    td = torch.float32 if dtype == "f32" else torch.bfloat16
    x, w, bias, labels = make(torch, 70, 300, dim, td, True, 9)
    f = forward(gpu, torch, x, w, bias, labels)
    whole = backward(gpu, torch, x, w, bias, labels, f["lse"], td)
    for keep in range(3):
        part = backward(gpu, torch, x, w, bias, labels, f["lse"], td, want=tuple(i == keep for i in range(3)))
        torch.cuda.synchronize()
        for i, name in enumerate(("dx", "dw", "db")):
            if i == keep:
                assert torch.equal(part[name], whole[name])
            else:
                assert (part[name] == 5.0).all()


@pytest.mark.parametrize("dtype,dim", [("bf16", 64), ("f32", 60)])
def test_rows_without_a_label_and_bad_labels(gpu, dtype, dim):
    import torch
    td = torch.float32 if dtype == "f32" else torch.bfloat16
    tokens, vocab = 40, 200
    x, w, bias, labels = make(torch, tokens, vocab, dim, td, True, 13)
    # all rows taken out
    out = torch.full((tokens,), -1.0, device="cuda")
    f = forward(gpu, torch, x, w, bias, out)
    g = backward(gpu, torch, x, w, bias, out, f["lse"], td, d_scale=f["summary"][2:])
    torch.cuda.synchronize()
    assert int(f["bad"]) == 0 and (f["loss"][:tokens] == 0).all() and f["summary"].tolist() == [0.0, 0.0, 0.0]
    assert all((g[n] == 0).all() for n in ("dx", "dw", "db"))
    # labels that are no class: beyond the vocabulary, infinite, NaN; -inf counts as one too, -5 does not
    labels[:5] = torch.tensor([float(vocab), float("inf"), float("nan"), float("-inf"), -5.0], device="cuda")
    f = forward(gpu, torch, x, w, bias, labels)
    g = backward(gpu, torch, x, w, bias, labels, f["lse"], td)
    torch.cuda.synchronize()
    assert int(f["bad"]) == 4 and (f["loss"][:5] == 0).all() and (g["dx"][:5] == 0).all()
    assert float(f["summary"][1]) == int(((labels >= 0) & (labels < vocab)).sum())


@pytest.mark.parametrize("dtype,dim", [("bf16", 64), ("f32", 60)])
def test_classes_taken_out_by_the_bias(gpu, dtype, dim):
    """-inf in the bias: whole blocks of the statistics hold nothing, the classes get no probability and no gradient; the lowest
    finite value does the same. A row left without any class is NaN."""
    import torch
    td = torch.float32 if dtype == "f32" else torch.bfloat16
    tokens, vocab = 50, 700
    x, w, bias, labels = make(torch, tokens, vocab, dim, td, True, 17)
    labels = torch.where(labels >= 0, 600.0 + labels % 100, labels)
    bias[:513] = -float("inf")
    bias[520:530] = torch.finfo(torch.float32).min
    f = forward(gpu, torch, x, w, bias, labels)
    g = backward(gpu, torch, x, w, bias, labels, f["lse"], td)
    torch.cuda.synchronize()
    live = torch.ones(vocab, dtype=torch.bool, device="cuda")
    live[:513] = False
    live[520:530] = False
    z = x.double() @ w[live].double().t() + bias[live].double()
    want = torch.logsumexp(z, 1)
    assert float((f["lse"][:tokens].double() - want).abs().max()) <= 2 * dim * U * 40 + 256 * U
    for n in ("dw", "db"):
        assert (g[n][~live] == 0).all() and g[n].isfinite().all()
    assert g["dx"].isfinite().all()
    bias[:] = -float("inf")
    f = forward(gpu, torch, x, w, bias, labels)
    torch.cuda.synchronize()
    counted = labels >= 0
    assert f["loss"][:tokens][counted].isnan().all() and (f["loss"][:tokens][~counted] == 0).all()


@pytest.mark.parametrize("dtype,dim", [("bf16", 128), ("f32", 100)])
def test_large_logits(gpu, dtype, dim):
    """Logits of a few hundred: one class takes the row, nothing overflows."""
    import torch
    td = torch.float32 if dtype == "f32" else torch.bfloat16
    x, w, bias, labels = make(torch, 64, 500, dim, td, False, 23, spread=100.0)
    f = forward(gpu, torch, x, w, bias, labels)
    g = backward(gpu, torch, x, w, bias, labels, f["lse"], torch.float32)
    torch.cuda.synchronize()
    r = reference(torch, x, w, bias, labels, torch.ones(64, device="cuda"))
    within(f["lse"][:64], r["lse"], r["lse_err"], U)
    gradients_within(torch, g, r, x, w, dtype == "bf16", torch.float32)


def test_gradient_is_the_slope_of_the_loss(gpu):
    """Central differences of the fp32 route's own loss along a random direction in x, W and the bias."""
    import torch
    tokens, vocab, dim = 20, 50, 12
    x, w, bias, labels = make(torch, tokens, vocab, dim, torch.float32, True, 29)
    f = forward(gpu, torch, x, w, bias, labels)
    g = backward(gpu, torch, x, w, bias, labels, f["lse"], torch.float32)
    gen = torch.Generator(device="cuda").manual_seed(1)
    dirs = [torch.randn(t.shape, generator=gen, device="cuda") for t in (x, w, bias)]
    want = sum(float((d.double() * g[n].double()).sum()) for d, n in zip(dirs, ("dx", "dw", "db")))
    h = 2.0 ** -8

    def total(sign):
        moved = [(t + sign * h * d).contiguous() for t, d in zip((x, w, bias), dirs)]
        return float(forward(gpu, torch, *moved, labels)["loss"][:tokens].double().sum())
    slope = (total(1.0) - total(-1.0)) / (2 * h)
    # third-order term of the difference and the losses' roundings (20 losses of about 5, 2^-22 each, over 2h)
    assert abs(slope - want) <= 20 * h * h * 200 + 20 * 5 * 2.0 ** -22 / (2 * h)


def test_same_bits_on_every_run_and_in_a_graph(gpu):
    """A captured and replayed step on a stream of its own gives the bits of the plain calls, also for new inputs."""
    import torch
    tokens, vocab, dim = 333, 3001, 192
    x, w, bias, labels = make(torch, tokens, vocab, dim, torch.bfloat16, True, 31)
    x2 = make(torch, tokens, vocab, dim, torch.bfloat16, True, 32)[0]

    def step(stream=None, ws=None):
        f = forward(gpu, torch, x, w, bias, labels, stream=stream, ws=ws)
        g = backward(gpu, torch, x, w, bias, labels, f["lse"], torch.bfloat16, d_scale=f["summary"][2:], stream=stream, ws=f["ws"])
        return [f["loss"], f["lse"], f["summary"], g["dx"], g["dw"], g["db"]]
    first, second = step(), step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        ws = workspace(gpu, torch, gpu.BF16, tokens, vocab, dim)
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            out = step(torch.cuda.current_stream().cuda_stream, ws)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, out))
    x.copy_(x2)
    want = step()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, out))


def test_two_streams_at_once(gpu):
    import torch
    cases = [make(torch, 200 + 50 * i, 2000, 128, torch.bfloat16, False, 40 + i) for i in range(2)]
    want = []
    for x, w, bias, labels in cases:
        f = forward(gpu, torch, x, w, bias, labels)
        want.append((f["loss"], backward(gpu, torch, x, w, bias, labels, f["lse"], torch.float32)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = []
    for (x, w, bias, labels), s in zip(cases, streams):
        with torch.cuda.stream(s):
            f = forward(gpu, torch, x, w, bias, labels, stream=s.cuda_stream)
            got.append((f["loss"], backward(gpu, torch, x, w, bias, labels, f["lse"], torch.float32, stream=s.cuda_stream, ws=f["ws"])))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1]["dx"], b[1]["dx"]) and torch.equal(a[1]["dw"], b[1]["dw"])


def test_no_rows(gpu):
    import torch
    x = torch.zeros(0, 64, dtype=torch.bfloat16, device="cuda")
    w = torch.ones(100, 64, dtype=torch.bfloat16, device="cuda")
    labels = torch.zeros(0, device="cuda")
    f = forward(gpu, torch, x, w, None, labels)
    g = backward(gpu, torch, x, w, None, labels, f["lse"], torch.bfloat16)
    torch.cuda.synchronize()
    assert f["summary"].tolist() == [0.0, 0.0, 0.0] and (g["dw"] == 0).all() and (g["db"] == 0).all()
