"""Distillation from a teacher's top logits (bfb_distill_topk) against the formulas in 64 bits.

The arguments of the exponentials are differences of logits over the temperature, scaled once by log2(e): off by at most 4 u |a| for
an argument a (u = 2^-24), so a probability is off by (8 A + 64) u relatively, where A is the largest |a| that still has a
probability worth counting (104: smaller ones are below 2^-149 and absolute), and loss and lse by sums of such terms. A bf16 result is
rounded once more, half a step: 2^-8."""
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
REL = (8 * 104 + 64) * U


def call(gpu, torch, z, ids, teacher, tau=1.0, weight=None, d_scale=None, scale=1.0, grad_dtype=None, pad=0, into=None, stream=None, want_grad=True):
    rows, vocab = z.shape
    k = ids.shape[1]
    grad_dtype = grad_dtype or z.dtype
    code = lambda t: gpu.F32 if t == torch.float32 else gpu.BF16  # noqa: E731
    loss, lse = torch.full((rows + 2,), 7.0, device="cuda"), torch.full((rows + 2,), 7.0, device="cuda")
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    whole = into if into is not None else torch.full((rows + 1, vocab + pad), 5.0, dtype=grad_dtype, device="cuda")
    gpu.check(gpu.lib().bfb_distill_topk(
        z.data_ptr(), code(z.dtype), max(vocab, z.stride(0)), ids.data_ptr(), teacher.data_ptr(), code(teacher.dtype), k, tau,
        None if weight is None else weight.data_ptr(), None if d_scale is None else d_scale.data_ptr(), scale, loss.data_ptr(), lse.data_ptr(),
        whole.data_ptr() if want_grad else None, code(grad_dtype), max(vocab, whole.stride(0)), rows, vocab, bad.data_ptr(), stream))
    return dict(loss=loss, lse=lse, whole=whole, grad=whole[:rows, :vocab], bad=bad)


def reference(torch, z, ids, teacher, tau, g):
    inf = float("inf")
    vocab = z.shape[1]
    s = z.double() / tau
    lse = torch.logsumexp(s, 1)
    log_p = s - lse[:, None]
    ok = (ids >= 0) & (ids < vocab)
    t = torch.where(ok, teacher.double() / tau, torch.full((), -inf, dtype=torch.float64, device="cuda"))
    counted = (t > -inf).any(1)
    top = torch.where(counted, t.max(1).values, torch.zeros_like(lse))
    e = torch.exp(t - top[:, None])
    q = e / e.sum(1, keepdim=True).clamp(min=1e-300)
    log_q = torch.log(q.clamp(min=1e-300))
    at = torch.where(ok, ids, torch.zeros_like(ids)).nan_to_num(posinf=0.0, neginf=0.0).long()
    gap = torch.where(q > 0, q * (log_q - log_p.gather(1, at)), torch.zeros_like(q))
    loss = torch.where(counted, tau * tau * gap.sum(1), torch.zeros_like(lse))
    grad = torch.exp(log_p).scatter_add(1, at, -q) * torch.where(counted, tau * g.double(), torch.zeros_like(lse))[:, None]
    loss_err = tau * tau * (q * (log_q.abs() + log_p.gather(1, at).abs() + 1)).nan_to_num().sum(1) * REL
    return lse, loss, loss_err, grad, counted


def make(torch, rows, vocab, k, dtype, seed, spread=2.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    z = (torch.randn(rows, vocab, generator=gen, device="cuda") * spread).to(dtype)
    top = torch.topk(z.float() + torch.randn(rows, vocab, generator=gen, device="cuda"), k, dim=1)
    ids = top.indices.float()
    drop = torch.rand(rows, k, generator=gen, device="cuda") < 0.1
    return z, torch.where(drop, torch.full_like(ids, -1.0), ids), top.values.contiguous()


def check(torch, got, z, ids, teacher, tau, g):
    rows, vocab = z.shape
    lse, loss, loss_err, grad, counted = reference(torch, z, ids, teacher, tau, g)
    assert float(((got["lse"][:rows].double() - lse).abs() - (REL + 4 * U * (lse.abs() + z.double().abs().max() / tau))).max()) <= 0
    assert float(((got["loss"][:rows].double() - loss).abs() - (loss_err + 1e-37)).max()) <= 0
    assert (got["loss"][rows:] == 7.0).all() and (got["lse"][rows:] == 7.0).all()
    half = U if got["grad"].dtype == torch.float32 else 2.0 ** -8
    size = (torch.exp(z.double() / tau - lse[:, None]) + grad.abs() / (tau * g.double().abs()[:, None])) * tau * g.double().abs()[:, None]
    err = REL * size + half * grad.abs() + 1e-37
    assert bool(((got["grad"].double() - grad).abs() <= err * (1 + half)).all())
    assert (got["whole"][rows:] == 5.0).all() and (got["whole"][:, vocab:] == 5.0).all()


# one value, one short block, several vectors a thread, clusters of two to eight blocks, wide blocks, rows beyond a cluster's registers
SHAPES = [(1, 1, 1), (3, 2, 2), (5, 31, 4), (40, 256, 8), (7, 1021, 20), (9, 1029, 33), (6, 4099, 64), (4, 8200, 50), (5, 33000, 100), (3, 70001, 10),
          (3, 131077, 1024), (2, 270001, 30), (2, 530011, 7)]


@pytest.mark.parametrize("rows,vocab,k", SHAPES)
@pytest.mark.parametrize("dtype,grad,tau", [("f32", "f32", 1.0), ("bf16", "bf16", 2.0), ("f32", "bf16", 1.5), ("bf16", "f32", 0.7)])
def test_loss_and_gradient(gpu, rows, vocab, k, dtype, grad, tau):
    import torch
    td = torch.float32 if dtype == "f32" else torch.bfloat16
    tg = torch.float32 if grad == "f32" else torch.bfloat16
    z, ids, teacher = make(torch, rows, vocab, k, td, rows + vocab + k)
    weight = torch.rand(rows, device="cuda") + 0.5
    scale = torch.tensor([0.5], device="cuda")
    for pad in (0, 3):   # an odd pitch: rows start anywhere in a 16-byte line
        wide = torch.full((rows, vocab + pad), 3.0, dtype=td, device="cuda")
        wide[:, :vocab] = z
        got = call(gpu, torch, wide[:, :vocab] if pad else z, ids, teacher, tau, weight, scale, 0.25, tg, pad)
        torch.cuda.synchronize()
        assert int(got["bad"]) == 0
        check(torch, got, z, ids, teacher, tau, weight * 0.125)


@pytest.mark.parametrize("offset,pad", [(1, 0), (2, 5), (3, 1)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_gradient_at_another_alignment_and_in_place(gpu, offset, pad, dtype):
    import torch
    td = torch.float32 if dtype == "f32" else torch.bfloat16
    rows, vocab = 4, 2051
    z, ids, teacher = make(torch, rows, vocab, 9, td, 5)
    g = torch.ones(rows, device="cuda")
    base = torch.full(((rows + 1) * (vocab + pad) + 8,), 5.0, dtype=td, device="cuda")
    out = base[offset:offset + (rows + 1) * (vocab + pad)].view(rows + 1, vocab + pad)
    got = call(gpu, torch, z, ids, teacher, into=out)
    torch.cuda.synchronize()
    check(torch, got, z, ids, teacher, 1.0, g)
    mine = torch.full((rows + 1, vocab + pad), 5.0, dtype=td, device="cuda")
    mine[:rows, :vocab] = z
    # the order of the sums goes by where a row starts in a 16-byte line, so bits are compared on the same rows
    apart = call(gpu, torch, mine[:rows, :vocab], ids, teacher)
    got2 = call(gpu, torch, mine[:rows, :vocab], ids, teacher, into=mine)
    torch.cuda.synchronize()
    assert torch.equal(got2["grad"], apart["grad"]) and torch.equal(got2["loss"], apart["loss"])
    check(torch, got2, z, ids, teacher, 1.0, g)


def test_entries_left_out_and_listed_twice(gpu):
    import torch
    inf = float("inf")
    rows, vocab = 6, 300
    z, ids, teacher = make(torch, rows, vocab, 12, torch.float32, 6)
    ids[0] = -1.0                                   # nothing listed: the row does not count
    teacher[1] = -inf                               # nothing with weight
    ids[2, :6] = ids[2, 6:7]                        # an id listed seven times
    ids[2, 6] = max(0.0, float(ids[2, 6]))
    ids[2, :7] = ids[2, 6]
    ids[3, 0], ids[3, 1], ids[3, 2] = float(vocab), float("nan"), inf
    teacher[4, :5] = -inf
    ids[5, 1:] = -5.0                               # a single entry: the sparse cross entropy
    ids[5, 0] = 17.0
    got = call(gpu, torch, z, ids, teacher)
    torch.cuda.synchronize()
    assert int(got["bad"]) == 3
    g = torch.ones(rows, device="cuda")
    clean = ids.nan_to_num(nan=-1.0, posinf=-1.0)
    check(torch, got, z, clean, teacher, 1.0, g)
    assert got["loss"][0] == 0 and got["loss"][1] == 0 and (got["grad"][:2] == 0).all()
    want = torch.nn.functional.cross_entropy(z[5:].double(), torch.tensor([17], device="cuda"))
    assert abs(float(got["loss"][5]) - float(want)) <= 40 * REL


@pytest.mark.parametrize("vocab", [200, 5000, 40000])
def test_masked_and_broken_student_rows(gpu, vocab):
    import torch
    inf = float("inf")
    z, ids, teacher = make(torch, 7, vocab, 10, torch.float32, 7)
    ids = ids.clamp(min=0)
    low = torch.finfo(torch.float32).min
    keep = torch.zeros(7, vocab, dtype=torch.bool, device="cuda").scatter_(1, ids.long(), True)
    z[0] = torch.where(keep[0], z[0], torch.full_like(z[0], -inf))      # all but the entries masked
    z[1] = torch.where(keep[1], z[1], torch.full_like(z[1], low))       # the same by the lowest finite value
    z[2] = -inf                                                        # no distribution
    z[3] = low                                                         # uniform
    z[4, vocab // 2] = float("nan")
    z[5, vocab // 3] = inf
    z[6, ids[6, 0].long()] = -inf                                      # the teacher wants what the student excludes
    got = call(gpu, torch, z, ids, teacher)
    torch.cuda.synchronize()
    rows = [0, 1]
    part = dict(got, loss=torch.cat([got["loss"][:2], got["loss"][7:]]), lse=torch.cat([got["lse"][:2], got["lse"][7:]]), grad=got["grad"][:2],
                whole=torch.cat([got["whole"][:2], got["whole"][7:]]))
    z01 = torch.where(z[rows] < -1e30, torch.full_like(z[rows], -1e30), z[rows])
    lse, loss, loss_err, grad, _ = reference(torch, z01, ids[rows], teacher[rows], 1.0, torch.ones(2, device="cuda"))
    assert float(((part["loss"][:2].double() - loss).abs() - loss_err).max()) <= 0
    assert float((part["grad"].double() - grad).abs().max()) <= REL
    for r in (2, 4, 5):
        assert got["loss"][r].isnan() and got["grad"][r].isnan().all()
    uniform = torch.full((vocab,), 1.0 / vocab, dtype=torch.float64, device="cuda")
    q = torch.softmax(teacher[3].double(), 0)
    assert float((got["grad"][3].double() - uniform.scatter_add(0, ids[3].long(), -q)).abs().max()) <= REL
    assert got["loss"][6] == inf and got["grad"][6].isfinite().all()
    # a row that does not count is zero whatever it holds
    none = torch.full_like(ids, -1.0)
    got = call(gpu, torch, z, none, teacher)
    torch.cuda.synchronize()
    assert (got["loss"][:7] == 0).all() and (got["grad"] == 0).all()


def test_results_that_are_not_asked_for_and_other_streams(gpu):
    import torch
    z, ids, teacher = make(torch, 20, 9000, 30, torch.bfloat16, 8)
    whole = call(gpu, torch, z, ids, teacher.to(torch.bfloat16))
    bare = call(gpu, torch, z, ids, teacher.to(torch.bfloat16), want_grad=False)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = call(gpu, torch, z, ids, teacher.to(torch.bfloat16), stream=torch.cuda.current_stream().cuda_stream)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(bare["loss"], whole["loss"]) and (bare["whole"] == 5.0).all()
    assert all(torch.equal(out[n], whole[n]) for n in ("loss", "lse", "whole"))
    check(torch, whole, z, ids, teacher.to(torch.bfloat16).float(), 1.0, torch.ones(20, device="cuda"))


def test_gradient_is_the_slope_of_the_loss(gpu):
    import torch
    z, ids, teacher = make(torch, 6, 500, 12, torch.float32, 9)
    got = call(gpu, torch, z, ids, teacher, 2.0)
    d = torch.randn(z.shape, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    h = 2.0 ** -7
    up, down = (call(gpu, torch, (z + s * h * d).contiguous(), ids, teacher, 2.0)["loss"][:6].double().sum() for s in (1.0, -1.0))
    torch.cuda.synchronize()
    want = float((got["grad"].double() * d.double()).sum())
    assert abs(float(up - down) / (2 * h) - want) <= 6 * h * h * 20 + 6 * 4 * 10 * 2.0 ** -22 / (2 * h)
